"""linear / grouped_linear without a GPU: the packed INT4 layout's size, the C
ABI's struct, and every refusal that is decided before anything is launched."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from haagenti_b200 import _lib as L

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # stands for device pointers: nothing here reaches a launch


def args(**kw):
    a = L.LinearArgs()
    base = dict(rows=4, out_features=8, in_features=64, d_x=P, ldx=64, d_weight=2 * P, ldw=64,
                weight_stride=512, d_out=3 * P, ldout=8, d_offsets=4 * P, experts=2,
                offsets_bits=32, x_dtype=L.BF16, weight_form=L.WEIGHT_DENSE, bias_dtype=L.BF16,
                out_dtype=L.BF16, activation=L.ACT_NONE, reserved=0)
    base.update(kw)
    for k, v in base.items():
        setattr(a, k, v)
    return a


def test_struct_layout_matches_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no C compiler")
    names = [f for f, _ in L.LinearArgs._fields_]
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "hct_b200.h"\nint main(void){'
                   'printf("%zu", sizeof(hct_b200_linear_args));'
                   + "".join(f'printf(" %zu", offsetof(hct_b200_linear_args, {n}));' for n in names)
                   + "return 0;}")
    exe = tmp_path / "sz"
    subprocess.run([cc, "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [C.sizeof(L.LinearArgs)] + [getattr(L.LinearArgs, n).offset for n in names]


def test_constants_match_header():
    text = open(os.path.join(REPO, "include", "hct_b200.h")).read()
    for n in ("NONE", "RELU", "SILU", "GELU", "GELU_TANH"):
        assert f"HCT_B200_ACT_{n} = {getattr(L, 'ACT_' + n)}" in text
    for n in ("DENSE", "INT4"):
        assert f"HCT_B200_WEIGHT_{n} = {getattr(L, 'WEIGHT_' + n)}" in text


@pytest.mark.parametrize("rows,cols,want", [
    (1, 32, 4608), (128, 64, 4608), (129, 64, 2 * 4608), (128, 96, 2 * 4608),
    (4096, 4096, 32 * 64 * 4608), (0, 32, 0), (1, 0, 0), (1, 31, 0), (1, 48, 0),
    (1 << 31, 32, 0), (1, 1 << 31, 0)])
def test_int4_weight_bytes(rows, cols, want):
    assert L.load().hct_b200_int4_weight_bytes(rows, cols) == want


def test_int4_weight_pack_refusals():
    f = L.load().hct_b200_int4_weight_pack
    assert f(P, 4 * 64 * 9 // 16 - 1, 4, 64, P, None) == L.SIZE_MISMATCH
    assert f(P, 4 * 64 * 9 // 16, 4, 63, P, None) == L.INVALID_ARGUMENT
    assert f(None, 1 << 20, 4, 64, P, None) == L.INVALID_ARGUMENT
    assert f(P, 1 << 20, 4, 64, None, None) == L.INVALID_ARGUMENT
    assert f(P, 1 << 20, 4, 64, P + 16, None) == L.INVALID_ARGUMENT


BAD = [
    dict(x_dtype=L.F32), dict(x_dtype=7), dict(out_dtype=3), dict(out_dtype=-1),
    dict(weight_form=2), dict(activation=5), dict(activation=-1), dict(reserved=1),
    dict(d_bias=5 * P, bias_dtype=L.F16), dict(rows=1 << 31), dict(out_features=1 << 31),
    dict(in_features=1 << 31), dict(d_out=None), dict(d_x=None), dict(d_weight=None),
    dict(d_x=P + 1), dict(d_out=3 * P + 1), dict(out_dtype=L.F32, d_out=3 * P + 2),
    dict(d_gate=5 * P + 1, ldgate=8), dict(d_residual=5 * P + 1, ldresidual=8),
    dict(d_bias=5 * P + 2, bias_dtype=L.F32), dict(d_weight=2 * P + 1),
    dict(weight_form=L.WEIGHT_INT4, d_weight=2 * P + 64),
    dict(weight_form=L.WEIGHT_INT4, in_features=48),
    dict(ldout=7), dict(ldout=0), dict(ldx=(1 << 30) + 1), dict(ldw=(1 << 30) + 1),
    dict(ldout=(1 << 30) + 1), dict(weight_stride=(1 << 46) + 1),
    # out overlaps an input
    dict(d_out=P), dict(d_out=P + 2 * (3 * 64 + 63)), dict(d_out=2 * P + 16),
    dict(d_bias=3 * P + 8), dict(d_gate=3 * P, ldgate=9), dict(d_gate=3 * P + 2, ldgate=8),
    dict(d_gate=3 * P, ldgate=8, out_dtype=L.F32), dict(d_residual=3 * P, ldresidual=16),
    dict(d_residual=3 * P + 2, ldresidual=8),
    dict(weight_form=L.WEIGHT_INT4, d_out=2 * P + 4600),
]


@pytest.mark.parametrize("kw", BAD, ids=lambda kw: ",".join(f"{k}={v}" for k, v in kw.items()))
def test_refused_before_any_launch(kw):
    lib = L.load()
    assert lib.hct_b200_linear(args(**kw), None) == L.INVALID_ARGUMENT
    assert lib.hct_b200_grouped_linear(args(**kw), None) == L.INVALID_ARGUMENT


@pytest.mark.parametrize("kw", [dict(experts=0), dict(experts=1025), dict(offsets_bits=16),
                                dict(d_offsets=None), dict(d_offsets=4 * P + 2),
                                dict(d_offsets=4 * P + 4, offsets_bits=64), dict(d_offsets=3 * P)])
def test_grouped_refusals(kw):
    assert L.load().hct_b200_grouped_linear(args(**kw), None) == L.INVALID_ARGUMENT


@pytest.mark.parametrize("kw", [dict(rows=0), dict(out_features=0), dict(rows=0, d_out=None, d_x=None)])
def test_nothing_to_do(kw):
    lib = L.load()
    assert lib.hct_b200_linear(args(**kw), None) == L.OK
    assert lib.hct_b200_grouped_linear(args(**kw), None) == L.OK


def test_null_args():
    lib = L.load()
    assert lib.hct_b200_linear(None, None) == L.INVALID_ARGUMENT
    assert lib.hct_b200_grouped_linear(None, None) == L.INVALID_ARGUMENT


def test_side_by_side_columns_of_one_buffer_do_not_overlap():
    """x in columns [0, 64) and out in columns [64, 72) of the same 72-wide rows: allowed,
    so that without a device the call gets as far as the launch."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    rc = L.load().hct_b200_linear(args(ldx=72, d_out=P + 128, ldout=72), None)
    assert rc not in (L.OK, L.INVALID_ARGUMENT)
    rc = L.load().hct_b200_linear(args(ldx=72, d_out=P + 126, ldout=72), None)
    assert rc == L.INVALID_ARGUMENT


def test_no_device_is_an_error():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert L.load().hct_b200_linear(args(), None) not in (L.OK, L.INVALID_ARGUMENT)
    assert L.load().hct_b200_linear_status(None) != L.OK


def test_python_refuses_host_tensors():
    import torch

    import haagenti_b200 as H

    x, w = torch.zeros(2, 8, dtype=torch.float16), torch.zeros(4, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        H.linear(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        H.grouped_linear(x, w[None], torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="offsets"):
        H.grouped_linear(x, w[None], None)
    with pytest.raises(ValueError, match="multiple of 32"):
        H.Int4Weight(b"", 4, 48)
    with pytest.raises(ValueError, match="payload"):
        H.Int4Weight([], 4, 64)


def run_host_check(tmp_path, name):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no C++ compiler")
    exe = tmp_path / name
    subprocess.run([cxx, "-std=c++17", "-O2", "-Wall", "-pthread", "-I",
                    os.path.join(REPO, "haagenti_b200", "csrc"),
                    os.path.join(REPO, "tests", name + ".cpp"), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert got.stdout.strip() == "ok", got.stdout


def test_no_timeout_is_lost_or_reported_twice(tmp_path):
    """The host side of linear_status: counts read in any order and by many threads."""
    run_host_check(tmp_path, "timeouts_check")


def test_properties_are_each_devices_own(tmp_path):
    """What plans ask of a device (its SMs, its clusters): no other device's, no failure remembered,
    from many threads at once."""
    run_host_check(tmp_path, "per_device_check")


def test_int4_weight_is_on_a_cuda_device():
    import haagenti_b200 as H

    for payload in (bytes(4 * 64 * 9 // 16), [bytes(4 * 64 * 9 // 16)]):
        with pytest.raises(ValueError, match="CUDA device"):
            H.Int4Weight(payload, 4, 64, device="cpu")


def test_first_call_is_complete_before_other_threads_see_it(monkeypatch):
    """A call goes ahead once _TAG is filled: everything else that it needs is set by then."""
    from haagenti_b200 import products as P

    class Watched(dict):
        def update(self, *a):
            assert set(P._TYPE) == {0, 1, 2} and callable(P._raw_stream) and P._forward_ad and L._lib
            assert not self
            super().update(*a)

    monkeypatch.setattr(P, "_TAG", Watched())
    monkeypatch.setattr(P, "_TYPE", {})
    monkeypatch.setattr(P, "_raw_stream", None)
    monkeypatch.setattr(P, "_forward_ad", None)
    P._first_call()
    assert sorted(P._TAG.values()) == [0, 1, 2] and {P._TYPE[v] for v in P._TAG.values()} == set(P._TAG)


class Reached(Exception):
    """Raised in the place of making a device current, with that device."""


@pytest.fixture
def two_devices(monkeypatch):
    """torch, as products.py sees it, with device 0 current and devices that cannot be entered."""
    import types

    import torch

    from haagenti_b200 import products as P

    def enter(device):
        raise Reached(torch.device("cuda", device) if isinstance(device, int) else torch.device(device))

    cuda = types.SimpleNamespace(device=enter, current_device=lambda: 0)
    fake = types.SimpleNamespace(cuda=cuda, device=torch.device, uint8=torch.uint8)
    monkeypatch.setattr(P, "_torch", lambda: fake)
    return P, torch, types.SimpleNamespace(device=torch.device("cuda", 1))


def test_a_stream_names_the_device(two_devices):
    """Where only a stream is given, its device is meant and not the current one."""
    P, torch, stream = two_devices
    payload = bytes(4 * 64 * 9 // 16)
    for kw, want in (({}, 0), ({"stream": stream}, 1), ({"device": 1}, 1), ({"device": "cuda:0"}, 0),
                     ({"device": "cuda", "stream": stream}, 1)):
        with pytest.raises(Reached) as e:
            P.linear_status(**{k: v for k, v in kw.items() if v != "cuda"})
        assert e.value.args[0] == torch.device("cuda", want), kw
        with pytest.raises(Reached) as e:
            P.Int4Weight(payload, 4, 64, **kw)
        assert e.value.args[0] == torch.device("cuda", want), kw
    with pytest.raises(ValueError, match="stream belongs"):
        P.Int4Weight(payload, 4, 64, device=0, stream=stream)
