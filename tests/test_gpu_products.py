"""linear / grouped_linear on the GPU against the definition in 64 bits.

Tolerances, per output, from the rounding steps of the documented arithmetic
(u = half a step of a type: bf16 2^-8, fp16 2^-11, f32 2^-24; S = sum |x w| +
|bias|, the sum of the terms' magnitudes; L = 1.2 bounds every activation's
slope: gelu's is at most 1.13):

    sum       a sum of K products in f32 in any order, each step rounded or
              truncated (one f32 step, 2 u32, at most): K 2 u32 S
    weights   INT4 in a 16-bit output: each weight rounded to x's type: u(x) S
    act       f32 evaluation of the activation: 16 u32 (|z| + 1)
    output    one rounding: u(out) |y|, or half the type's smallest step

Where the bounds add up, |gate| multiplies all but the last.
"""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
TAG = {"f32": 0, "f16": 1, "bf16": 2}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def act64(z, act):
    if act == 1:
        return z.clamp(min=0)
    if act == 2:
        return z * torch.special.expit(z)
    if act == 3:
        return z * torch.special.ndtr(z)
    if act == 4:
        return z * torch.special.expit(2 * np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3))
    return z


def payload_of(w, scale_zero_at=None):
    """quantize_int4's layout of a float matrix (cols a multiple of 32)."""
    g = w.reshape(-1, 32)
    s = (g.abs().amax(1) / 7).to(torch.float16)
    if scale_zero_at is not None:
        s[scale_zero_at] = 0
    q = torch.where(s[:, None] > 0, (g / s[:, None].float()).round(), torch.zeros_like(g))
    q = (q.clamp(-8, 7) + 8).to(torch.uint8).reshape(-1, 2)
    return torch.cat([s.view(torch.uint8), q[:, 0] | (q[:, 1] << 4)])


def weight64(data, n, k):
    s = data[: n * k // 16].view(torch.float16).double()
    b = data[n * k // 16: n * k // 16 + n * k // 2]
    q = torch.stack([b & 15, b >> 4], 1).double() - 8
    return (q.reshape(-1, 32) * s[:, None]).reshape(n, k)


def define(x, w, bias, act, gate, res, out_t, int4):
    """(value, tolerance) in 64 bits of one group's rows."""
    k = x.shape[1]
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    S = xd.abs() @ wd.abs().t()
    if bias is not None:
        z, S = z + bias.double(), S + bias.double().abs()
    u32 = 2.0 ** -24
    err = (k + 2) * 2 * u32 * S
    if int4 and out_t != torch.float32:
        err = err + U[x.dtype] * S
    y = act64(z, act)
    err = 1.2 * err + (16 * u32 * (z.abs() + 1) if act else 0)
    if gate is not None:
        y, err = y * gate.double(), err * gate.double().abs() + u32 * (y * gate.double()).abs()
    if res is not None:
        y = y + res.double()
        err = err + u32 * y.abs()
    return y, err + U[out_t] * (y.abs() + err) + TINY[out_t]


def check(got, want, tol, what=""):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:4].tolist(),
                           got[bad][:4].tolist(), want[bad][:4].tolist(), tol[bad][:4].tolist())


def make(dev, seed, m, n, k, e, form, dt, out, bias, gate, res, bias_f32=False):
    g = torch.Generator(device=dev).manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, device=dev, generator=g)

    t = DT[dt]
    d = {"x": rn(m, k).to(t), "w": [], "bias": None, "gate": None, "res": None}
    for i in range(e):
        w = 0.1 * rn(n, k)
        d["w"].append(payload_of(w, scale_zero_at=i % max(n * k // 32, 1) if k else None)
                      if form == "int4" else w.to(t))
    if bias:
        d["bias"] = rn(e, n).to(torch.float32 if bias_f32 else t)
    if gate:
        d["gate"] = rn(m, n).to(t)
    if res:
        d["res"] = rn(m, n).to(DT[out])
    return d


def run_linear(hb, d, n, k, form, act, out, **kw):
    w = hb.Int4Weight(d["w"][0], n, k) if form == "int4" else d["w"][0]
    return hb.linear(d["x"], w, None if d["bias"] is None else d["bias"][0], act, d["gate"],
                     d["res"], TAG[out], **kw)


SHAPES = [(1, 1, 32), (1, 8, 64), (1, 128, 4096), (1, 1000, 1024), (2, 130, 96), (3, 257, 2048),
          (5, 384, 672), (8, 128, 8192), (9, 640, 512), (15, 100, 160), (16, 256, 256), (17, 129, 320),
          (31, 513, 1056), (33, 128, 64), (64, 1024, 1024), (65, 200, 128), (100, 777, 992),
          (127, 128, 448), (128, 128, 128), (129, 384, 512), (200, 1000, 608), (255, 130, 96),
          (256, 256, 1024), (257, 300, 640), (300, 2048, 256), (513, 640, 800), (1000, 1153, 320),
          # enough whole tiles for pairs of CTAs: a second half past the last feature, odd heights
          (300, 19000, 96), (513, 9728, 160), (1030, 4900, 320), (700, 9600, 1056),
          # more tiles than CTAs of a few rows, with one and with several K parts; half tiles
          (3, 40000, 64), (12, 38000, 96), (7, 5000, 1600), (40, 520, 1024), (90, 260, 800)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("form,dt,out", [("int4", "bf16", "bf16"), ("int4", "f16", "f16"),
                                         ("int4", "bf16", "f32"), ("int4", "f16", "f32"),
                                         ("dense", "bf16", "bf16"), ("dense", "f16", "f32"),
                                         ("dense", "bf16", "f16")])
def test_linear_shapes(hb, dev, m, n, k, form, dt, out):
    i = SHAPES.index((m, n, k))
    act, b, g, r = i % 5, i % 2 == 0, i % 3 == 0, i % 4 < 2
    d = make(dev, i, m, n, k, 1, form, dt, out, b, g, r)
    got = run_linear(hb, d, n, k, form, act, out)
    assert got.dtype == DT[out] and got.shape == (m, n)
    w = weight64(d["w"][0], n, k) if form == "int4" else d["w"][0]
    want, tol = define(d["x"], w, None if d["bias"] is None else d["bias"][0], act, d["gate"],
                       d["res"], DT[out], form == "int4")
    check(got, want, tol)
    hb.linear_status()


@pytest.mark.parametrize("m,n,k", [(1, 5, 1), (1, 64, 7), (2, 33, 31), (7, 100, 333), (16, 64, 1001),
                                   (77, 130, 1001), (33, 65, 12), (300, 70, 4), (129, 257, 100)])
@pytest.mark.parametrize("dt,out", [("bf16", "bf16"), ("f16", "f32")])
def test_dense_rows_of_any_length(hb, dev, m, n, k, dt, out):
    d = make(dev, m + n + k, m, n, k, 1, "dense", dt, out, True, False, True)
    got = run_linear(hb, d, n, k, "dense", 3, out)
    want, tol = define(d["x"], d["w"][0], d["bias"][0], 3, None, d["res"], DT[out], False)
    check(got, want, tol)


@pytest.mark.parametrize("act", range(5), ids=ACTS)
@pytest.mark.parametrize("form", ["int4", "dense"])
@pytest.mark.parametrize("m", [1, 6, 40, 160])
def test_epilogue_combinations(hb, dev, act, form, m):
    n, k = 192, 256
    for j in range(8):
        for out in ("bf16", "f32", "f16"):
            d = make(dev, 50 + j, m, n, k, 1, form, "bf16", out, j & 1, j & 2, j & 4, bias_f32=j >= 4)
            got = run_linear(hb, d, n, k, form, act, out)
            w = weight64(d["w"][0], n, k) if form == "int4" else d["w"][0]
            want, tol = define(d["x"], w, None if d["bias"] is None else d["bias"][0], act,
                               d["gate"], d["res"], DT[out], form == "int4")
            check(got, want, tol, (j, out))


@pytest.mark.parametrize("m", [1, 16, 150])
@pytest.mark.parametrize("k,form", [(1024, "dense"), (4096, "dense"), (16384, "dense"),
                                    (1024, "int4"), (4096, "int4"), (16384, "int4")])
def test_f32_output_keeps_its_precision(hb, dev, m, k, form):
    """The 2-norm of an F32 output's error.  A section of 256 products is at most 16 truncated
    steps of 2^-23 of a partial sum, whose norm is at most the section's on independent data;
    sections add up with rounding, and their norms in quadrature: (16 2^-23 sqrt(K / 256) + K /
    256 2^-24) |y|.  Weights that had been rounded to 16 bits would be off by 1e-4 and more."""
    n = 256
    d = make(dev, k, m, n, k, 1, form, "bf16", "f32", False, False, False)
    got = run_linear(hb, d, n, k, form, 0, "f32").double()
    w = weight64(d["w"][0], n, k) if form == "int4" else d["w"][0].double()
    want = d["x"].double() @ w.t()
    rel = float((got - want).norm() / want.norm())
    assert rel <= 16 * 2.0 ** -23 * (k / 256) ** 0.5 + k / 256 * 2.0 ** -24, rel


def sorted_sizes(kind, m, e, seed):
    rng = np.random.default_rng(seed)
    if kind == "even":
        s = [m // e] * e
        s[-1] += m - sum(s)
    elif kind == "one":
        s = [0] * e
        s[e // 2] = m
    else:
        p = rng.random(e) ** 3 * (rng.random(e) > 0.3) + 1e-3
        s = rng.multinomial(m, p / p.sum()).tolist()
    return s


@pytest.mark.parametrize("m,e,n,k", [(1, 1, 32, 32), (1, 8, 256, 512), (8, 8, 1000, 1024),
                                     (8, 64, 64, 96), (40, 3, 384, 2048), (96, 16, 130, 160),
                                     (257, 5, 200, 64), (1000, 7, 257, 320), (1500, 40, 128, 256),
                                     (1500, 3, 7710, 160), (2100, 7, 2400, 320), (30, 9, 5200, 128),
                                     (60, 2, 300, 1024)])
@pytest.mark.parametrize("kind", ["even", "one", "ragged"])
@pytest.mark.parametrize("form,dt,out", [("int4", "bf16", "bf16"), ("int4", "f16", "f32"),
                                         ("dense", "bf16", "f32"), ("dense", "f16", "f16")])
def test_grouped_shapes(hb, dev, m, e, n, k, kind, form, dt, out):
    seed = m + e + n
    head, tail = (seed % 3), (seed % 5)  # rows before the first group and behind the last one
    sizes = sorted_sizes(kind, m, e, seed)
    rows = m + head + tail
    act, g, r = seed % 5, seed % 2 == 0, seed % 3 == 0
    d = make(dev, seed, rows, n, k, e, form, dt, out, True, g, r)
    for t in ("x", "gate", "res"):  # rows of no group are not read
        if d[t] is not None:
            d[t][:head] = float("nan")
            d[t][rows - tail:] = float("nan")
    off = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]) + head, device=dev,
                       dtype=torch.int64 if seed % 2 else torch.int32)
    y = torch.full((rows, n), 7.0, dtype=DT[out], device=dev)
    w = hb.Int4Weight(d["w"], n, k) if form == "int4" else torch.stack(d["w"])
    got = hb.grouped_linear(d["x"], w, off, d["bias"], act, d["gate"], d["res"], out=y)
    assert got is y
    assert (y[:head] == 7).all() and (y[rows - tail:] == 7).all()
    at = head
    for i, s in enumerate(sizes):
        q = slice(at, at + s)
        at += s
        wi = weight64(d["w"][i], n, k) if form == "int4" else d["w"][i]
        want, tol = define(d["x"][q], wi, d["bias"][i], act, d["gate"][q] if g else None,
                           d["res"][q] if r else None, DT[out], form == "int4")
        check(y[q], want, tol, (i, s))
    hb.linear_status()


@pytest.mark.parametrize("form", ["int4", "dense"])
def test_grouped_equals_linear_per_expert(hb, dev, form):
    """One group is linear's own arithmetic (the same sums up to their order)."""
    n, k, m = 256, 512, 48
    d = make(dev, 3, m, n, k, 1, form, "bf16", "bf16", True, True, True)
    a = run_linear(hb, d, n, k, form, 2, "bf16")
    w = hb.Int4Weight(d["w"], n, k) if form == "int4" else torch.stack(d["w"])
    off = torch.tensor([0, m], dtype=torch.int32, device=dev)
    b = hb.grouped_linear(d["x"], w, off, d["bias"], 2, d["gate"], d["res"])
    w1 = weight64(d["w"][0], n, k) if form == "int4" else d["w"][0]
    want, tol = define(d["x"], w1, d["bias"][0], 2, d["gate"], d["res"], torch.bfloat16, form == "int4")
    check(a, want, tol)
    check(b, want, tol)


@pytest.mark.parametrize("form", ["int4", "dense"])
def test_wrong_offsets_stay_in_range(hb, dev, form):
    """Values outside [0, rows] are clamped, descending ones count as the largest before."""
    n, k, m, e = 96, 128, 50, 4
    d = make(dev, 9, m, n, k, e, form, "f16", "f16", False, False, False)
    w = hb.Int4Weight(d["w"], n, k) if form == "int4" else torch.stack(d["w"])
    buf = torch.full((m + 40, n), 7.0, dtype=torch.float16, device=dev)
    y = buf[20: 20 + m]
    off = torch.tensor([-5, 10, 4, 30, 1 << 30], dtype=torch.int32, device=dev)
    hb.grouped_linear(d["x"], w, off, out=y)
    assert (buf[:20] == 7).all() and (buf[20 + m:] == 7).all()
    for i, q in ((0, slice(0, 4)), (2, slice(10, 30)), (3, slice(30, 50))):
        wi = weight64(d["w"][i], n, k) if form == "int4" else d["w"][i]
        # the groups are [0, 10), none, [10, 30) and [30, 50)
        want, tol = define(d["x"][q], wi, None, 0, None, None, torch.float16, form == "int4")
        check(y[q], want, tol, i)
    off = torch.tensor([1 << 40, -(1 << 40), 1 << 62, -1, 7], dtype=torch.int64, device=dev)
    y.fill_(7)
    hb.grouped_linear(d["x"], w, off, out=y)
    assert (buf == 7).all()  # every group begins and ends at row 50


@pytest.mark.parametrize("form,out", [("int4", "bf16"), ("int4", "f32"), ("dense", "bf16"),
                                      ("dense", "f32")])
@pytest.mark.parametrize("m", [4, 70, 300])
def test_nan_and_infinity_stay_in_their_row(hb, dev, form, out, m):
    n, k = 160, 320
    d = make(dev, 5, m, n, k, 1, form, "bf16", out, False, False, False)
    clean = run_linear(hb, d, n, k, form, 0, out)
    d["x"][1, 17] = float("nan")
    d["x"][3, 5] = float("inf")
    got = run_linear(hb, d, n, k, form, 0, out)
    keep = [i for i in range(m) if i not in (1, 3)]
    assert torch.equal(got[keep], clean[keep])
    assert got[1].isnan().all() and not got[3].isfinite().any()


def test_int4_scales_at_the_edges(hb, dev):
    """Scales of zero, the smallest subnormal, the largest value, infinity and NaN."""
    n, k = 128, 64
    g = torch.Generator(device=dev).manual_seed(1)
    nib = torch.randint(0, 256, (n * k // 2,), dtype=torch.uint8, device=dev, generator=g)
    s = torch.full((n * k // 32,), 0.01, dtype=torch.float16, device=dev)
    bits = s.view(torch.int16)
    bits[0:2], bits[2:4], bits[4:6] = 0, 1, 0x03ff
    bits[6:8] = 0x7bff
    bits[8:10] = 0x7c00
    bits[10:12] = 0x7e00
    data = torch.cat([s.view(torch.uint8), nib])
    w = weight64(data, n, k)
    for dt in ("bf16", "f16"):
        for m in (1, 12, 40):
            x = torch.randn(m, k, device=dev, generator=g).to(DT[dt]) * 0.25
            for out in ("f32", dt):
                got = hb.linear(x, hb.Int4Weight(data, n, k), out_dtype=TAG[out])
                fine = [i for i in range(n) if i not in (4, 5)]
                want, tol = define(x, w[fine], None, 0, None, None, DT[out], True)
                if dt == "f16":
                    # 8 x 65504 leaves the type: row 3 may be infinite in fp16.  A subnormal weight is
                    # a multiple of 2^-24, as its scale is, so that nothing more is rounded
                    inf = fine.index(3)
                    tol[:, inf], want[:, inf] = float("inf"), 0
                    sub = got[:, fine].clone()
                    sub[:, inf] = 0
                    check(sub, want, tol, (dt, m, out))
                else:
                    big = want.abs() > torch.finfo(DT[out]).max
                    check(torch.where(big, 0, got[:, fine].double()), torch.where(big, 0, want), tol,
                          (dt, m, out))
                assert not got[:, 4].isfinite().any() and got[:, 5].isnan().all()


@pytest.mark.parametrize("form", ["int4", "dense"])
@pytest.mark.parametrize("m", [3, 48, 140])
def test_strides_and_shared_buffers(hb, dev, form, m):
    n, k = 96, 256
    d = make(dev, 11, m, n, k, 1, form, "f16", "f16", True, True, True)
    w = hb.Int4Weight(d["w"][0], n, k) if form == "int4" else d["w"][0]
    w64 = weight64(d["w"][0], n, k) if form == "int4" else d["w"][0]
    want, tol = define(d["x"], w64, d["bias"][0], 2, d["gate"], d["res"], torch.float16, form == "int4")

    def call(x=d["x"], w=w, gate=d["gate"], res=d["res"], out=None):
        return hb.linear(x, w, d["bias"][0], 2, gate, res, out=out)

    # padded rows (a multiple of 16 bytes and not), a misaligned start
    for pad, start in ((8, 0), (8, 8), (3, 0), (8, 1)):
        xb = torch.full((m, k + pad + start), float("nan"), dtype=torch.float16, device=dev)
        xb[:, start: start + k] = d["x"]
        check(call(x=xb[:, start: start + k]), want, tol, ("x", pad, start))
        if form == "dense":
            wb = torch.full((n, k + pad + start), float("nan"), dtype=torch.float16, device=dev)
            wb[:, start: start + k] = w
            check(call(w=wb[:, start: start + k]), want, tol, ("w", pad, start))
        ob = torch.full((m, n + pad + start), 7.0, dtype=torch.float16, device=dev)
        o = ob[:, start: start + n]
        assert call(out=o) is o
        check(o, want, tol, ("out", pad, start))
        assert (ob[:, :start] == 7).all() and (ob[:, start + n:] == 7).all()
        gb = torch.full((m, n + pad + start), float("nan"), dtype=torch.float16, device=dev)
        gb[:, start: start + n] = d["gate"]
        check(call(gate=gb[:, start: start + n]), want, tol, ("gate", pad, start))
    # broadcast operands
    row = d["res"][:1]
    want1, tol1 = define(d["x"], w64, d["bias"][0], 2, d["gate"], row.expand(m, n), torch.float16,
                         form == "int4")
    check(call(res=row.expand(m, n)), want1, tol1)
    xr = d["x"][:1].expand(m, k)
    want2, tol2 = define(xr, w64, d["bias"][0], 2, d["gate"], d["res"], torch.float16, form == "int4")
    check(call(x=xr), want2, tol2)
    # out in the place of the residual, of the gate, and of both operands at once
    r = d["res"].clone()
    check(call(res=r, out=r), want, tol)
    g = d["gate"].clone()
    check(call(gate=g, out=g), want, tol)
    # x and out side by side in one buffer
    both = torch.zeros(m, k + n, dtype=torch.float16, device=dev)
    both[:, :k] = d["x"]
    check(call(x=both[:, :k], out=both[:, k:]), want, tol)
    assert torch.equal(both[:, :k], d["x"])


@pytest.mark.parametrize("m", [2, 100])
def test_grouped_weight_strides(hb, dev, m):
    """Experts, rows and columns cut out of a larger tensor."""
    e, n, k = 3, 80, 128
    g = torch.Generator(device=dev).manual_seed(2)
    for pad in (8, 3):
        big = torch.randn(e, n + 5, k + pad, device=dev, generator=g).to(torch.bfloat16)
        w = big[:, 2: n + 2, :k]
        x = torch.randn(m, k, device=dev, generator=g).to(torch.bfloat16)
        off = torch.tensor([0, m // 2, m // 2, m], dtype=torch.int32, device=dev)
        y = hb.grouped_linear(x, w, off)
        for i, q in ((0, slice(0, m // 2)), (2, slice(m // 2, m))):
            want, tol = define(x[q], w[i], None, 0, None, None, torch.bfloat16, False)
            check(y[q], want, tol, (pad, i))


def test_empty_sizes(hb, dev):
    w = torch.randn(16, 32, device=dev).to(torch.float16)
    assert hb.linear(torch.zeros(0, 32, dtype=torch.float16, device=dev), w).shape == (0, 16)
    assert hb.linear(torch.zeros(3, 32, dtype=torch.float16, device=dev), w[:0]).shape == (3, 0)
    b = torch.randn(16, device=dev).to(torch.float16)
    y = hb.linear(torch.zeros(3, 0, dtype=torch.float16, device=dev), w[:, :0], b, hb.ACT_RELU)
    assert torch.equal(y, b.clamp(min=0).expand(3, 16))
    off = torch.zeros(5, dtype=torch.int32, device=dev)
    out = torch.full((3, 16), 7.0, dtype=torch.float16, device=dev)
    hb.grouped_linear(torch.zeros(3, 32, dtype=torch.float16, device=dev), w.expand(4, 16, 32), off,
                      out=out)
    assert (out == 7).all()


def test_offsets_past_32_bits(hb, dev):
    """Outputs past element 2^31 and byte 2^32."""
    m, n, k = 70000, 32768, 32
    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(m, k, device=dev, generator=g).to(torch.bfloat16)
    for form in ("dense", "int4"):
        w = torch.randn(n, k, device=dev, generator=g)
        data = payload_of(w) if form == "int4" else w.to(torch.bfloat16)
        y = hb.linear(x, hb.Int4Weight(data, n, k) if form == "int4" else data)
        w64 = weight64(data, n, k) if form == "int4" else data
        for q in (slice(0, 2), slice(65535, 65538), slice(m - 2, m)):
            want, tol = define(x[q], w64, None, 0, None, None, torch.bfloat16, form == "int4")
            check(y[q], want, tol, q)
        del y


def test_many_experts(hb, dev):
    e, n, k, m = 1024, 16, 32, 700
    d = make(dev, 6, m, n, k, e, "int4", "bf16", "bf16", True, False, False)
    sizes = sorted_sizes("ragged", m, e, 1)
    off = torch.tensor([0] + list(np.cumsum(sizes)), dtype=torch.int32, device=dev)
    y = hb.grouped_linear(d["x"], hb.Int4Weight(d["w"], n, k), off, d["bias"])
    which = torch.repeat_interleave(torch.arange(e, device=dev), torch.tensor(sizes, device=dev))
    w = torch.stack([weight64(p, n, k) for p in d["w"]])
    for i in range(m):
        want, tol = define(d["x"][i: i + 1], w[which[i]], d["bias"][which[i]], 0, None, None,
                           torch.bfloat16, True)
        check(y[i: i + 1], want, tol, i)


@pytest.mark.parametrize("form", ["int4", "dense"])
@pytest.mark.parametrize("m", [5, 90])
def test_same_bits_every_time(hb, dev, form, m):
    n, k, e = 512, 2048, 3
    d = make(dev, 8, m, n, k, e, form, "bf16", "bf16", True, True, True)
    w = hb.Int4Weight(d["w"], n, k) if form == "int4" else torch.stack(d["w"])
    off = torch.tensor([0, m // 3, m // 3, m], dtype=torch.int32, device=dev)
    a = hb.grouped_linear(d["x"], w, off, d["bias"], 1, d["gate"], d["res"])
    for _ in range(5):
        assert torch.equal(a, hb.grouped_linear(d["x"], w, off, d["bias"], 1, d["gate"], d["res"]))


@pytest.mark.parametrize("form", ["int4", "dense"])
@pytest.mark.parametrize("m", [4, 64, 200])
def test_captured_and_replayed(hb, dev, form, m):
    """A captured call reads its inputs, the offsets among them, anew in each replay; two graphs
    run at once on two streams do not share anything."""
    n, k, e = 256, 512, 4
    d = make(dev, 12, m, n, k, e, form, "bf16", "bf16", False, False, False)
    w = hb.Int4Weight(d["w"], n, k) if form == "int4" else torch.stack(d["w"])
    w64 = [weight64(p, n, k) if form == "int4" else p for p in d["w"]]
    graphs = []
    for j in range(2):
        x = d["x"].clone()
        off = torch.tensor([0, m, m, m, m], dtype=torch.int32, device=dev)
        hb.grouped_linear(x, w, off)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        s = torch.cuda.Stream(dev)
        with torch.cuda.graph(gr, stream=s):
            y = hb.grouped_linear(x, w, off)
        graphs.append((gr, x, off, y, s))
    for rep in range(3):
        cut = [[0, m // 4, m // 2, m // 2, m], [0, 0, 1, m, m], [0, m, m, m, m]]
        for j, (gr, x, off, y, s) in enumerate(graphs):
            x.copy_(torch.randn(m, k, device=dev).to(torch.bfloat16))
            off.copy_(torch.tensor(cut[(rep + j) % 3], dtype=torch.int32, device=dev))
        torch.cuda.synchronize()
        for gr, x, off, y, s in graphs:
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for gr, x, off, y, s in graphs:
            o = off.tolist()
            for i in range(e):
                q = slice(o[i], o[i + 1])
                want, tol = define(x[q], w64[i], None, 0, None, None, torch.bfloat16, form == "int4")
                check(y[q], want, tol, (rep, i))


@pytest.mark.parametrize("form", ["int4", "dense"])
def test_streams(hb, dev, form):
    """A call on another stream than the tensors' own, and calls on two streams at once."""
    n, k, m = 512, 1024, 32
    d = make(dev, 13, m, n, k, 1, form, "f16", "f16", False, False, True)
    w = hb.Int4Weight(d["w"][0], n, k) if form == "int4" else d["w"][0]
    want = hb.linear(d["x"], w, residual=d["res"])
    torch.cuda.synchronize()
    ss = [torch.cuda.Stream(dev) for _ in range(2)]
    outs = []
    for i in range(20):
        outs.append(hb.linear(d["x"], w, residual=d["res"], stream=ss[i % 2]))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


def test_weight_freed_while_another_stream_reads_it(hb, dev):
    """A weight laid out on one stream, used on another and dropped at once: its memory is not
    handed out again before the product has read it."""
    n, k, m = 4096, 4096, 300
    data = payload_of(0.1 * torch.randn(n, k, device=dev))
    x = torch.randn(m, k, device=dev).to(torch.bfloat16)
    a, b = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    want = hb.linear(x, hb.Int4Weight(data, n, k))
    torch.cuda.synchronize()
    for _ in range(5):
        w = hb.Int4Weight(data, n, k, stream=a)
        size = w.packed.numel()
        with torch.cuda.stream(b):
            for _ in range(20):
                y = hb.linear(x, w)
        del w
        with torch.cuda.stream(a):
            junk = torch.full((size,), 255, dtype=torch.uint8, device=dev)
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        del junk


def test_two_threads(hb, dev):
    """Calls from two threads at once, each on its own stream."""
    import threading

    n, k = 640, 1024
    d = make(dev, 30, 200, n, k, 1, "int4", "bf16", "bf16", False, False, False)
    w = hb.Int4Weight(d["w"][0], n, k)
    want = {m: hb.linear(d["x"][:m], w) for m in (5, 200)}
    torch.cuda.synchronize()
    bad = []

    def work(m):
        s = torch.cuda.Stream(dev)
        with torch.cuda.stream(s):
            for _ in range(50):
                y = hb.linear(d["x"][:m], w)
        s.synchronize()
        if not torch.equal(y, want[m]):
            bad.append(m)

    ts = [threading.Thread(target=work, args=(m,)) for m in (5, 200)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


def test_reader_hands_out_its_int4_weight(hb, dev, orc):
    """A plain INT4 file multiplied from its payload equals the product with its decoded tensor."""
    from oracle import hct as OH

    n, k, m = 300, 512, 24
    rng = np.random.default_rng(3)
    wf = (0.05 * rng.standard_normal((n, k))).astype(np.float32)
    f = OH.write_hct(orc.quantize_int4(wf.reshape(-1)), [n, k])
    r = hb.HctReader(f)
    w = r.int4_weight()
    assert w.shape == (n, k) and w.experts is None
    x = torch.randn(m, k, device=dev).to(torch.bfloat16)
    y = hb.linear(x, w, out_dtype=hb.F32)
    dec = r.decode(hb.F32)
    want, tol = define(x, dec, None, 0, None, None, torch.float32, True)
    check(y, want, tol)
    y2 = hb.linear(x, r.decode(hb.BF16))
    y3 = hb.linear(x, w)
    want, tol = define(x, dec, None, 0, None, None, torch.bfloat16, True)
    check(y2, want, tol)
    check(y3, want, tol)
    spectral = OH.encode_spectral_q4(OH.gen_weight((64, 64), 2))
    with pytest.raises(hb.Unsupported, match="plain INT4"):
        hb.HctReader(spectral).int4_weight()


def test_payloads_on_the_host_and_longer_than_needed(hb, dev):
    n, k = 40, 96
    data = payload_of(torch.randn(n, k, device=dev))
    x = torch.randn(3, k, device=dev).to(torch.float16)
    a = hb.linear(x, hb.Int4Weight(data, n, k))
    long = torch.cat([data, torch.full((7,), 255, dtype=torch.uint8, device=dev)])
    assert torch.equal(a, hb.linear(x, hb.Int4Weight(long, n, k)))
    assert torch.equal(a, hb.linear(x, hb.Int4Weight(data.cpu().numpy().tobytes(), n, k)))
    odd = torch.cat([data[:1], data])[1:]  # an odd byte address
    assert torch.equal(a, hb.linear(x, hb.Int4Weight(odd, n, k)))
    with pytest.raises(hb.CorruptedData):
        hb.Int4Weight(data[:-1], n, k)


def test_mlp_in_a_row(hb, dev):
    """gate, up and down projections of an MLP as they are used: silu(x Wg) * (x Wu), then Wd and
    the residual, INT4 and dense weights mixed."""
    m, h, i = 37, 256, 704
    d1 = make(dev, 20, m, i, h, 2, "int4", "bf16", "bf16", False, False, False)
    wd = (0.1 * torch.randn(h, i, device=dev)).to(torch.bfloat16)
    x = d1["x"]
    wg, wu = (hb.Int4Weight(p, i, h) for p in d1["w"])
    up = hb.linear(x, wu)
    act = hb.linear(x, wg, activation=hb.ACT_SILU, gate=up, out=up)
    y = hb.linear(act, wd, residual=x)
    g64, u64 = (weight64(p, i, h) for p in d1["w"])
    a, ta = define(x, u64, None, 0, None, None, torch.bfloat16, True)
    b, tb = define(x, g64, None, 2, None, None, torch.float32, True)
    tb = tb + 1.2 * U[torch.bfloat16] * (x.double().abs() @ g64.abs().t())
    h64 = a * b
    th = ta * b.abs() + tb * a.abs() + ta * tb
    th = th + U[torch.bfloat16] * (h64.abs() + th)
    check(act, h64, th)
    want, tol = define(act, wd, None, 0, None, x, torch.bfloat16, False)
    check(y, want, tol)


def test_experts_in_a_row(hb, dev):
    """Rows routed to experts, sorted, through two grouped products, and summed back."""
    t, topk, e, h, i = 21, 2, 6, 128, 192
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(t, h, device=dev, generator=g).to(torch.bfloat16)
    ids = torch.rand(t, e, device=dev, generator=g).topk(topk).indices.reshape(-1)
    order = ids.argsort(stable=True)
    off = torch.zeros(e + 1, dtype=torch.int64, device=dev)
    off[1:] = torch.bincount(ids, minlength=e).cumsum(0)
    w1 = [payload_of(0.1 * torch.randn(i, h, device=dev, generator=g)) for _ in range(e)]
    w2 = torch.randn(e, h, i, device=dev, generator=g).mul(0.1).to(torch.bfloat16)
    xs = x[order // topk]
    a = hb.grouped_linear(xs, hb.Int4Weight(w1, i, h), off, activation=hb.ACT_GELU)
    b = hb.grouped_linear(a, w2, off, out_dtype=hb.F32)
    y = torch.zeros(t, h, device=dev).index_add_(0, order // topk, b)
    want = torch.zeros(t, h, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(want)
    for p in range(t * topk):
        ex = int(ids[order[p]])
        v, tv = define(xs[p: p + 1], weight64(w1[ex], i, h), None, 3, None, None, torch.bfloat16, True)
        check(a[p: p + 1], v, tv)
        v, tv = define(a[p: p + 1], w2[ex], None, 0, None, None, torch.float32, False)
        want[order[p] // topk] += v[0]
        tol[order[p] // topk] += tv[0] + 2.0 ** -23 * v[0].abs()
    check(y, want, tol)


def test_python_refusals(hb, dev):
    f16, bf = torch.float16, torch.bfloat16
    x = torch.zeros(4, 64, dtype=f16, device=dev)
    w = torch.zeros(8, 64, dtype=f16, device=dev)
    off = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    q = hb.Int4Weight(payload_of(torch.randn(8, 64, device=dev)), 8, 64)
    qs = hb.Int4Weight([payload_of(torch.randn(8, 64, device=dev))], 8, 64)
    r = torch.zeros(4, 8, dtype=f16, device=dev)

    def no(match, f, *a, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            f(*a, **kw)

    no("2-D", hb.linear, x[0], w)
    no("float16 or bfloat16", hb.linear, x.float(), w.float())
    no("x's type", hb.linear, x, w.to(bf))
    no("features", hb.linear, x, w[:, :32])
    no("features", hb.linear, x[:, :32], q)
    no("contiguous", hb.linear, torch.zeros(64, 4, dtype=f16, device=dev).t(), w)
    no("contiguous", hb.linear, x, torch.zeros(64, 8, dtype=f16, device=dev).t())
    no("out_features, in_features", hb.linear, x, w[None])
    no("out_features, in_features", hb.grouped_linear, x, w, off)
    no("experts needs grouped", hb.linear, x, qs)
    no("needs a weight with experts", hb.grouped_linear, x, q, off)
    no("weight is on", hb.linear, x, w.cpu())
    no("int32 or int64", hb.grouped_linear, x, w[None], off.float())
    no("int32 or int64", hb.grouped_linear, x, w[None], off.cpu())
    no("experts . 1", hb.grouped_linear, x, w[None], off[:1])
    no("out_dtype", hb.linear, x, w, out_dtype=9)
    no("out is of", hb.linear, x, w, out=r, out_dtype=hb.F32)
    no("out must be", hb.linear, x, w, out=r[:3])
    no("bias must be", hb.linear, x, w, torch.zeros(7, dtype=f16, device=dev))
    no("bias must be", hb.linear, x, w, torch.zeros(8, dtype=bf, device=dev))
    no("bias must be", hb.grouped_linear, x, w[None], off, torch.zeros(8, dtype=f16, device=dev))
    no("contiguous", hb.linear, x, w, torch.zeros(16, dtype=f16, device=dev)[::2])
    no("gate must be", hb.linear, x, w, gate=r.float())
    no("gate must be", hb.linear, x, w, gate=r[:2])
    no("residual must be", hb.linear, x, w, residual=r, out_dtype=hb.F32)
    no("contiguous", hb.linear, x, w, residual=torch.zeros(8, 4, dtype=f16, device=dev).t())
    no("invalid", hb.linear, x, w, activation=9, error=hb.DeviceError)
    no("invalid", hb.linear, x, x[:4, :], out=x[:, :4], error=hb.DeviceError)
    no("backward", hb.linear, x.requires_grad_(), w, error=hb.Unsupported)
    with torch.no_grad():
        hb.linear(x, w)
    no("uint8", hb.Int4Weight, torch.zeros(4, 64, device=dev), 4, 64)
    gr, s = torch.cuda.CUDAGraph(), torch.cuda.Stream(dev)
    data = payload_of(torch.randn(8, 64, device=dev))
    torch.cuda.synchronize()
    with torch.cuda.graph(gr, stream=s):
        no("captured", hb.Int4Weight, data, 8, 64, error=hb.Unsupported)
        y = hb.linear(x.detach(), q)
    gr.replay()
    torch.cuda.synchronize()
    assert (y == 0).all()


def test_status_is_clean(hb):
    hb.linear_status()


@pytest.mark.parametrize("shift", [1, 2])
@pytest.mark.parametrize("m,n,k", [(1, 40, 2), (5, 130, 66), (80, 64, 1502), (150, 300, 994), (20, 5000, 1000)])
@pytest.mark.parametrize("dt,out", [("bf16", "bf16"), ("f16", "f32")])
def test_dense_rows_at_any_place(hb, dev, shift, m, n, k, dt, out):
    """Rows that start on 2 or on 4 bytes, even and odd strides between them, NaN around them."""
    for pad in (6, 7):
        d = make(dev, m + n + k, m, n, k, 2, "dense", dt, out, False, False, False)
        x = torch.full((m, k + pad), float("nan"), device=dev, dtype=DT[dt])[:, shift:shift + k]
        w = torch.full((2, n + 1, k + pad), float("nan"), device=dev, dtype=DT[dt])[:, :n, shift:shift + k]
        x.copy_(d["x"])
        w.copy_(torch.stack(d["w"]))
        want, tol = define(x, w[0], None, 0, None, None, DT[out], False)
        check(hb.linear(x, w[0], out_dtype=TAG[out]), want, tol)
        cut = m // 3
        off = torch.tensor([0, cut, m], dtype=torch.int32, device=dev)
        want2, tol2 = define(x, w[1], None, 0, None, None, DT[out], False)
        got = hb.grouped_linear(x, w, off, out_dtype=TAG[out])
        check(got, torch.cat([want[:cut], want2[cut:]]), torch.cat([tol[:cut], tol2[cut:]]))
    hb.linear_status()


COLD = """
import torch, haagenti_b200 as H
dev = torch.device("cuda", 0)
m, n, k, form, out = {case}
x = torch.ones(m, k, device=dev, dtype=torch.bfloat16)
if form == "int4":
    s = torch.full((n * k // 32,), 0.5, dtype=torch.float16, device=dev).view(torch.uint8)
    w = H.Int4Weight(torch.cat([s, torch.full((n * k // 2,), 0x99, dtype=torch.uint8, device=dev)]), n, k)
else:
    w = torch.full((n, k), 0.5, device=dev, dtype=torch.bfloat16)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = H.linear(x, w, out_dtype=out)
graph.replay()
torch.cuda.synchronize()
assert (y == 0.5 * k).all()
H.linear_status()
"""


@pytest.mark.parametrize("case", [(1, 256, 1024, "int4", None), (40, 256, 1024, "int4", 0),
                                  (40, 256, 1024, "dense", None), (3, 256, 130, "dense", None),
                                  (4096, 2560, 256, "dense", None)])
def test_first_call_of_a_process_captured(hb, dev, case):
    """A graph may hold the first product of a process: nothing has been set up before."""
    subprocess.run([sys.executable, "-c", COLD.format(case=case)], check=True, timeout=300,
                   cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


@pytest.mark.parametrize("form,dt,out", [("int4", "bf16", "f32"), ("int4", "f16", "f32"),
                                         ("int4", "bf16", "bf16"), ("int4", "f16", "f16"),
                                         ("dense", "bf16", "f32"), ("dense", "f16", "f16")])
@pytest.mark.parametrize("m,k", [(4, 320), (16, 1024), (40, 320), (40, 4096), (300, 320)])
def test_infinite_inputs_give_what_the_definition_gives(hb, dev, form, dt, out, m, k):
    """Infinity times a weight has the weight's sign, times zero it is NaN, and infinities of both
    signs are NaN, for however many rows; the other rows keep their values."""
    n = 160
    d = make(dev, m + k, m, n, k, 1, form, dt, out, False, False, False)
    x, inf = d["x"], float("inf")
    x[1, 17], x[2, 5] = inf, -inf
    x[3, 40], x[3, 200] = inf, -inf
    got = run_linear(hb, d, n, k, form, 0, out)
    w = weight64(d["w"][0], n, k) if form == "int4" else d["w"][0]
    want, tol = define(x, w, None, 0, None, None, DT[out], form == "int4")
    bad = torch.tensor([1, 2, 3], device=dev)
    a, b = got[bad].double(), want[bad]
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))
    keep = [i for i in range(m) if i not in (1, 2, 3)]
    check(got[keep], want[keep], tol[keep])


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("m", [16, 64])
def test_f32_outputs_hold_every_int4_weight(hb, dev, dt, m):
    """A row of x that is 1 in one place gives that column of the weights, to the last bit, for
    finite scales of every size (8 x 65504 among them) and either sign."""
    n, k = 4096, 64
    g = torch.Generator(device=dev).manual_seed(7)
    nib = torch.randint(0, 256, (n * k // 2,), dtype=torch.uint8, device=dev, generator=g)
    bits = torch.randint(0, 0x7c00, (n * k // 32,), device=dev, generator=g, dtype=torch.int32)
    bits[:64] = torch.arange(64, device=dev)  # zero and the smallest subnormal scales
    bits[64:96] = 0x7bff - torch.arange(32, device=dev)
    bits[96:128] = 0x1bf0 + torch.arange(32, device=dev)  # about 2^-8
    sign = torch.randint(0, 2, (n * k // 32,), device=dev, generator=g, dtype=torch.int32)
    scales = torch.where(sign > 0, bits - 32768, bits).to(torch.int16).view(torch.float16)
    data = torch.cat([scales.view(torch.uint8), nib])
    x = torch.eye(k, device=dev)[:m].to(DT[dt])
    got = hb.linear(x, hb.Int4Weight(data, n, k), out_dtype=hb.F32)
    assert torch.equal(got, weight64(data, n, k).float().t()[:m])
    off = torch.tensor([0, m], dtype=torch.int32, device=dev)
    got = hb.grouped_linear(x, hb.Int4Weight([data], n, k), off, out_dtype=hb.F32)
    assert torch.equal(got, weight64(data, n, k).float().t()[:m])


@pytest.mark.parametrize("m", [1, 12, 16, 17, 40, 150, 300])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_int4_weights_past_the_range_of_f16(hb, dev, m, out):
    """fp16 x and finite scales whose weights pass 65504: exact for F32 outputs and up to 16 rows;
    else such weights are infinite, as their decoded form is."""
    n, k = 160, 320
    g = torch.Generator(device=dev).manual_seed(m)
    s = torch.full((n * k // 32,), 0.01, dtype=torch.float16, device=dev)
    s[::7], s[3] = 9000.0, 65504.0
    nib = torch.randint(0, 256, (n * k // 2,), dtype=torch.uint8, device=dev, generator=g)
    data = torch.cat([s.view(torch.uint8), nib])
    x = (1e-3 * torch.randn(m, k, device=dev, generator=g)).to(torch.float16)
    got = hb.linear(x, hb.Int4Weight(data, n, k), out_dtype=TAG[out])
    w = weight64(data, n, k)
    if out == "f32" or m <= 16:
        want, tol = define(x, w, None, 0, None, None, DT[out], False)
        check(got, want, tol)
    else:
        r = w.to(torch.float16).double()
        want, tol = define(x, r, None, 0, None, None, DT[out], False)
        fine = want.isfinite()
        assert torch.equal(got.isfinite(), fine) and torch.equal(got.isnan(), want.isnan())
        check(torch.where(fine, got.double(), 0), torch.where(fine, want, 0), torch.where(fine, tol, 0))


@pytest.mark.parametrize("form", ["int4", "dense"])
@pytest.mark.parametrize("m", [16, 17, 150])
@pytest.mark.parametrize("k", [1024, 8192])
def test_f32_output_of_f16_keeps_its_precision(hb, dev, form, m, k):
    """test_f32_output_keeps_its_precision with fp16 x.  INT4: the rounded weights' section is 16
    truncated steps, and the remainders', 2^-10 of it at most, another 16.  Weights without their
    remainders would be off by 2e-4."""
    n = 256
    d = make(dev, k + 1, m, n, k, 1, form, "f16", "f32", False, False, False)
    got = run_linear(hb, d, n, k, form, 0, "f32").double()
    w = weight64(d["w"][0], n, k) if form == "int4" else d["w"][0].double()
    want = d["x"].double() @ w.t()
    rel = float((got - want).norm() / want.norm())
    assert rel <= 16 * 2.0 ** -23 * (1 + 2.0 ** -10) * (k / 256) ** 0.5 + k / 256 * 2.0 ** -24, rel


@pytest.mark.parametrize("m", [3, 16, 40, 300])
@pytest.mark.parametrize("form", ["int4", "dense"])
@pytest.mark.parametrize("grouped", [False, True])
def test_no_input_features_through_the_c_abi(hb, dev, m, form, grouped):
    """in_features of 0 is a product of zero, whatever stands for x and the weights."""
    L, n, e = hb._lib, 136, 2 if grouped else 1
    bias = torch.randn(e, n, device=dev).to(torch.bfloat16)
    gate, res = (torch.randn(m, n, device=dev).to(torch.bfloat16) for _ in range(2))
    off = torch.tensor([0, m // 3, m], dtype=torch.int32, device=dev)
    for out_t in ("bf16", "f32"):
        out = torch.full((m, n), 7.0, dtype=DT[out_t], device=dev)
        r = res.to(DT[out_t])
        a = L.LinearArgs(rows=m, out_features=n, in_features=0, d_x=None, ldx=0, d_weight=None, ldw=0,
                         weight_stride=0, d_bias=bias.data_ptr(), d_gate=gate.data_ptr(), ldgate=n,
                         d_residual=r.data_ptr(), ldresidual=n, d_out=out.data_ptr(), ldout=n,
                         d_offsets=off.data_ptr(), experts=e, offsets_bits=32, x_dtype=L.BF16,
                         weight_form=L.WEIGHT_INT4 if form == "int4" else L.WEIGHT_DENSE,
                         bias_dtype=L.BF16, out_dtype=TAG[out_t], activation=L.ACT_RELU, reserved=0)
        f = L.load().hct_b200_grouped_linear if grouped else L.load().hct_b200_linear
        assert f(C.byref(a), torch.cuda.current_stream().cuda_stream) == L.OK
        rows = torch.arange(m, device=dev)
        b = bias[(rows >= m // 3).long()] if grouped else bias
        want = b.double().clamp(min=0) * gate.double() + r.double()
        check(out, want, (U[DT[out_t]] + 2 * 2.0 ** -24) * want.abs() + 2.0 ** -23 * (b * gate).double().abs())
    hb.linear_status()


@pytest.mark.parametrize("name", ["x", "weight", "bias", "gate", "residual"])
def test_dual_tensors_are_refused(hb, dev, name):
    """A product that dropped a tangent in silence would give wrong derivatives."""
    import torch.autograd.forward_ad as forward_ad

    m, n, k = 4, 16, 32
    kw = {"x": torch.randn(m, k, device=dev), "weight": torch.randn(n, k, device=dev),
          "bias": torch.randn(n, device=dev), "gate": torch.randn(m, n, device=dev),
          "residual": torch.randn(m, n, device=dev)}
    kw = {i: t.to(torch.bfloat16) for i, t in kw.items()}
    want = hb.linear(**kw)
    off = torch.tensor([0, m], dtype=torch.int32, device=dev)
    many = dict(kw, weight=kw["weight"][None], bias=kw["bias"][None])
    with forward_ad.dual_level():
        for f, args in ((hb.linear, kw), (hb.grouped_linear, dict(many, offsets=off))):
            dual = dict(args)
            dual[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
            with pytest.raises(hb.Unsupported, match="forward-mode"):
                f(**dual)
            with torch.no_grad(), pytest.raises(hb.Unsupported, match="forward-mode"):
                f(**dual)
            dual[name] = forward_ad.unpack_dual(dual[name]).primal
            assert torch.equal(f(**dual), want)
    assert torch.equal(hb.linear(**kw), want)


def test_int4_weight_on_a_device_by_name(hb, dev):
    """"cuda" without an index is the payload's device, or the current one."""
    n, k = 16, 64
    data = payload_of(torch.randn(n, k, device=dev))
    x = torch.randn(3, k, device=dev).to(torch.float16)
    want = hb.linear(x, hb.Int4Weight(data, n, k))
    host = data.cpu().numpy().tobytes()
    for payload in (data, host):
        for name in (None, "cuda", "cuda:0", 0, torch.device("cuda"), dev):
            w = hb.Int4Weight(payload, n, k, device=name)
            assert w.device == w.packed.device == dev
            assert torch.equal(hb.linear(x, w), want)
            assert hb.Int4Weight([payload, payload], n, k, device=name).shape == (2, n, k)


@pytest.mark.parametrize("form", ["int4", "dense"])
@pytest.mark.parametrize("m,n,k", [(2048, 9728, 512), (300, 19000, 1024), (1030, 4900, 2048)])
def test_pairs_give_the_same_bits_every_time(hb, dev, form, m, n, k):
    """Tiles that two CTAs share, one issuing for both, linear and grouped, weights of their own
    before each call so that a K step taken too early would show."""
    d = [make(dev, 40 + i, m, n, k, 1, form, "bf16", "bf16", False, False, False) for i in range(2)]
    ws = [hb.Int4Weight(i["w"][0], n, k) if form == "int4" else i["w"][0] for i in d]
    x = d[0]["x"]
    rows = torch.tensor([0, 1, m // 2, m - 1], device=dev)
    want = []
    for i, w in enumerate(ws):
        want.append(hb.linear(x, w))
        w64 = weight64(d[i]["w"][0], n, k) if form == "int4" else w
        v, tol = define(x[rows], w64, None, 0, None, None, torch.bfloat16, form == "int4")
        check(want[i][rows], v, tol)
    for i in range(20):
        assert torch.equal(hb.linear(x, ws[i % 2]), want[i % 2])
    both = hb.Int4Weight([i["w"][0] for i in d], n, k) if form == "int4" else torch.stack(ws)
    off = torch.tensor([0, m // 3, m], dtype=torch.int32, device=dev)
    first = hb.grouped_linear(x, both, off)
    for i in range(10):
        assert torch.equal(hb.grouped_linear(x, both, off), first)
    hb.linear_status()


def test_products_among_other_kernels(hb, dev):
    """Products between library products and the library's own decode on one stream, each of whose
    kernels may start while the one before it ends: every result as when it runs alone."""
    from oracle import hct as OH

    m, n, k = 512, 1024, 1024
    d = make(dev, 60, m, n, k, 1, "int4", "bf16", "bf16", False, False, False)
    q, x = hb.Int4Weight(d["w"][0], n, k), d["x"]
    w = weight64(d["w"][0], n, k).to(torch.bfloat16)
    r = hb.HctReader(OH.encode_spectral_q4(OH.gen_weight((256, 512), 2)))
    calls = [lambda: hb.linear(x, q), lambda: x @ w.t(), lambda: hb.linear(x[:40], q),
             lambda: hb.linear(x[:4], q), lambda: r.decode(hb.BF16), lambda: hb.linear(x, w),
             lambda: x[:64] @ w.t(), lambda: hb.linear(x, q, out_dtype=hb.F32)]
    want = []
    for c in calls:
        want.append(c())
        torch.cuda.synchronize()
    for rep in range(10):
        order = np.random.default_rng(rep).permutation(np.repeat(np.arange(len(calls)), 4))
        got = [(i, calls[i]()) for i in order]
        torch.cuda.synchronize()
        for i, y in got:
            assert torch.equal(y, want[i]), i
    hb.linear_status()


def test_status_does_not_end_a_capture(hb, dev):
    """linear_status on a stream that is being captured is refused, and the graph stays good."""
    x, w = torch.ones(4, 64, device=dev, dtype=torch.float16), torch.ones(8, 64, device=dev, dtype=torch.float16)
    hb.linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hb.linear(x, w)
        with pytest.raises(hb.Unsupported):
            hb.linear_status()
        z = hb.linear(x, w, residual=y)
    graph.replay()
    torch.cuda.synchronize()
    assert (y == 64).all() and (z == 128).all()
    hb.linear_status()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("m", [1, 8, 16, 17, 60])
def test_largest_inputs_with_int4_weights(hb, dev, dt, m):
    """x at its type's ends times weights below 1: the products are within range, and so is every
    step on the way to them."""
    n, k = 160, 320
    d = make(dev, 70 + m, m, n, k, 1, "int4", dt, "f32", False, False, False)
    big, row = torch.finfo(DT[dt]).max, torch.arange(m, device=dev)
    d["x"][row, row * 7 % k] = torch.where(row % 2 == 0, big, -big).to(DT[dt])
    w = weight64(d["w"][0], n, k)
    assert w.abs().max() < 1
    for out in ("f32", dt):
        want, tol = define(d["x"], w, None, 0, None, None, DT[out], True)
        fine = want.abs() <= 0.99 * torch.finfo(DT[out]).max
        got = run_linear(hb, d, n, k, "int4", 0, out)
        check(torch.where(fine, got.double(), 0), torch.where(fine, want, 0), tol, out)


@pytest.mark.parametrize("activation", ["silu", None, 1.0, 1 << 40, -(1 << 40)])
def test_activations_are_constants(hb, dev, activation):
    x, w = torch.ones(4, 64, device=dev, dtype=torch.float16), torch.ones(8, 64, device=dev, dtype=torch.float16)
    with pytest.raises(ValueError, match="ACT_ constants"):
        hb.linear(x, w, activation=activation)
    assert (hb.linear(x, w) == 64).all()


@pytest.mark.parametrize("form", ["int4", "dense"])
@pytest.mark.parametrize("m", [12, 50, 400])
def test_descending_offsets_row_by_row(hb, dev, form, m):
    """Every row of a call whose offsets descend, those after a descent among them: a value below
    its predecessors counts as the largest before it."""
    n, k, e = 96, 128, 5
    d = make(dev, 80 + m, m, n, k, e, form, "f16", "f16", True, False, False)
    w = hb.Int4Weight(d["w"], n, k) if form == "int4" else torch.stack(d["w"])
    for offsets in ([-5, m // 3, 1, m // 2, 0, 1 << 30], [2, m // 2, m // 4, m // 4, m - 1, 0],
                    [m // 3, 0, 0, 0, m // 2, m // 4]):
        ends = np.maximum.accumulate(np.clip(offsets, 0, m))
        y = torch.full((m, n), 7.0, dtype=torch.float16, device=dev)
        off = torch.tensor(offsets, dtype=torch.int32, device=dev)
        hb.grouped_linear(d["x"], w, off, d["bias"], out=y)
        assert (y[:ends[0]] == 7).all() and (y[ends[-1]:] == 7).all()
        for i in range(e):
            q = slice(int(ends[i]), int(ends[i + 1]))
            wi = weight64(d["w"][i], n, k) if form == "int4" else d["w"][i]
            want, tol = define(d["x"][q], wi, d["bias"][i], 0, None, None, torch.float16, form == "int4")
            check(y[q], want, tol, (offsets, i))


@pytest.mark.parametrize("m", [20, 300])
def test_experts_interleaved_or_shared(hb, dev, m):
    """Expert weights whose rows lie between one another's, and one matrix for every expert."""
    n, k, e = 96, 128, 4
    g = torch.Generator(device=dev).manual_seed(m)
    x = torch.randn(m, k, device=dev, generator=g).to(torch.bfloat16)
    rows = torch.randn(n, e, k, device=dev, generator=g).to(torch.bfloat16)
    off = torch.tensor([0, m // 4, m // 4, m // 2, m], dtype=torch.int64, device=dev)
    for w in (rows.transpose(0, 1), rows[:, 0].expand(e, n, k), rows[:, 1].contiguous().expand(e, n, k)):
        y = hb.grouped_linear(x, w, off)
        for i in range(e):
            q = slice(int(off[i]), int(off[i + 1]))
            want, tol = define(x[q], w[i], None, 0, None, None, torch.bfloat16, False)
            check(y[q], want, tol, i)
