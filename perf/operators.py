"""What the products with decoded weights are measured on: linear and grouped_linear.

    linear          y = act(x Wt + bias) * gate + residual
    grouped_linear  the same for rows sorted by expert, each group with the
                    weight matrix of its own expert

Weights are the two forms in which this library hands them out: dense fp16 or
bf16 matrices (HctReader.decode), or INT4 payloads in the quantize_int4 layout
(HctReader.decompress_all of a plain INT4 file): ceil(n/32) f16 scales, then
nibbles, low nibble first, value (nibble - 8) * scale.  Sizes are those of the
Llama-2-70B and Llama-3-8B tensors that the benchmark decodes, and generic
odd ones.  Experts are of the 8B model's MLP sizes, or smaller.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
OUT = {"f32": 0, "f16": 1, "bf16": 2}
ACT = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
MOST_FLOPS = 1.0e12     # of a drawn case
MOST_WEIGHTS = 4.7e8    # elements of a drawn case's weights


def _linear(name, m, n, k, weight, dtype, out=None, act="none", bias=False, gate=False, residual=False):
    c = {"op": "linear", "m": m, "n": n, "k": k, "weight": weight, "dtype": dtype, "out": out or dtype,
         "act": act, "bias": bias, "gate": gate, "residual": residual}
    return dict(c, name=name) if name else c


def _grouped(name, t, e, n, k, weight, dtype, routing, tail=0, out=None, act="none", bias=False, gate=False,
             residual=False):
    c = {"op": "grouped", "m": t, "e": e, "n": n, "k": k, "weight": weight, "dtype": dtype, "out": out or dtype,
         "act": act, "bias": bias, "gate": gate, "residual": residual, "routing": routing, "tail": tail}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token through the 8B model's o_proj, straight from its INT4 file: latency
        _linear("token-int4", 1, 4096, 4096, "int4", "bf16", residual=True),
        # one token through the 70B model's gate_proj, decoded to bf16, with up_proj's output as the gate
        _linear("token-dense", 1, 28672, 8192, "dense", "bf16", act="silu", gate=True),
        # a decode batch through the 70B model's o_proj in INT4
        _linear("batch16-int4", 16, 8192, 8192, "int4", "f16", residual=True),
        # a ragged batch through the 70B model's k_proj: few rows, few output features, a long sum
        _linear("batch61-dense", 61, 1024, 8192, "dense", "f16", bias=True),
        # nothing divides anything: rows that are not a multiple of 16 bytes
        _linear("odd-dense", 77, 1000, 1001, "dense", "f16", out="f32", act="gelu", bias=True),
        # a prompt through the 8B model's gate_proj in INT4
        _linear("prompt-int4", 2048, 14336, 4096, "int4", "bf16", act="silu", gate=True),
        # a prompt through the 70B model's down_proj: the largest
        _linear("prompt-dense", 4096, 8192, 28672, "dense", "bf16", residual=True),
        # four tokens of two experts each: most experts have one row or none
        _grouped("experts-token-int4", 8, 8, 14336, 4096, "int4", "bf16", 1, act="silu", gate=True),
        # a decode batch over many small experts
        _grouped("experts-batch-dense", 96, 64, 1024, 4096, "dense", "bf16", 2),
        # a middling batch, down projection in INT4
        _grouped("experts-batch-int4", 1024, 8, 4096, 14336, "int4", "f16", 3),
        # ragged groups, empty ones among them, a padded batch's rows behind the last group
        _grouped("experts-odd-dense", 1024, 16, 1000, 1000, "dense", "f16", 4, tail=24, out="f32",
                 act="gelu_tanh", bias=True, residual=True),
        # a prompt's rows over eight experts
        _grouped("experts-prompt-dense", 8192, 8, 14336, 4096, "dense", "bf16", 5, act="silu", gate=True),
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    grouped = rng.random() < 0.5
    weight = rng.choice(["int4", "dense"])
    dtype = rng.choice(["f16", "bf16"])
    while True:
        n = _log(rng, 16, 28672)
        k = _log(rng, 32, 28672)
        if weight == "int4":
            k = max(32, k // 32 * 32)
        elif rng.random() < 0.75:
            k = max(8, k // 8 * 8)
        if rng.random() < 0.6:
            n = max(64, n // 64 * 64)
        m = _log(rng, 1, 8192)
        e = _log(rng, 1, 64) if grouped else 1
        if 2.0 * m * n * k <= MOST_FLOPS and float(e) * n * k <= MOST_WEIGHTS:
            break
    more = {"out": rng.choice([dtype, dtype, "f32"]), "act": rng.choice(list(ACT)), "bias": rng.random() < 0.5,
            "gate": rng.random() < 0.3, "residual": rng.random() < 0.5}
    if not grouped:
        return _linear(None, m, n, k, weight, dtype, **more)
    tail = rng.randrange(m) if rng.random() < 0.3 else 0
    return _grouped(None, m, e, n, k, weight, dtype, rng.randrange(1 << 30), tail=tail, **more)


def sizes(case):
    """Rows of each expert: shares that differ by an order of magnitude, some experts idle."""
    rng = random.Random(case["routing"])
    share = [rng.random() ** 2 * (rng.random() > 0.15) for _ in range(case["e"])]
    share[rng.randrange(case["e"])] += 0.05
    got = [0] * case["e"]
    for i in rng.choices(range(case["e"]), share, k=case["m"] - case["tail"]):
        got[i] += 1
    return got


def work(case):
    m, n, k = case["m"], case["n"], case["k"]
    active = 1
    if case["op"] == "grouped":
        m -= case["tail"]
        active = sum(1 for s in sizes(case) if s)
    per = n * k * 0.5 + n * k / 16 if case["weight"] == "int4" else n * k * 2.0
    out = BYTES[case["out"]]
    b = m * k * 2.0 + active * per + m * n * out
    b += active * n * 2.0 if case["bias"] else 0
    b += m * n * 2.0 if case["gate"] else 0
    b += m * n * out if case["residual"] else 0
    b += 4.0 * (case["e"] + 1) if case["op"] == "grouped" else 0
    return {"bytes": b, "flops": 2.0 * m * n * k}


def _payload(w):
    """quantize_int4's layout of a float matrix: f16 scales of 32 values each, then nibbles."""
    g = w.reshape(-1, 32)
    s = (g.abs().amax(1) / 7).to(torch.float16)
    q = torch.where(s[:, None] > 0, (g / s[:, None].float()).round(), torch.zeros_like(g)).clamp(-8, 7) + 8
    q = q.to(torch.uint8).reshape(-1, 2)
    return torch.cat([s.view(torch.uint8), q[:, 0] | (q[:, 1] << 4)])


def _inputs(case, seed):
    """Tensors of a case from its seed alone: weights N(0, 0.02) with 1 % of the columns 10 times as large,
    activations N(0, 1) with a few large channels."""
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    m, n, k, t = case["m"], case["n"], case["k"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    big = torch.where(torch.rand(k, device=dev, generator=g) < 0.01, 10.0, 1.0)
    x = normal(m, k)
    x[:, :: max(k // 4, 1)] *= 8
    s = {"case": case, "x": x.to(t), "weights": []}
    for _ in range(case.get("e", 1)):
        w = normal(n, k).mul_(0.02).mul_(big)
        s["weights"].append(_payload(w) if case["weight"] == "int4" else w.to(t))
    many = (case["e"],) if case["op"] == "grouped" else ()
    s["bias"] = (0.1 * normal(*many, n)).to(t) if case["bias"] else None
    s["gate"] = normal(m, n).to(t) if case["gate"] else None
    s["residual"] = normal(m, n).to(TYPES[case["out"]]) if case["residual"] else None
    if case["op"] == "grouped":
        s["sizes"] = sizes(case)
        ends = [0]
        for c in s["sizes"]:
            ends.append(ends[-1] + c)
        s["offsets"] = torch.tensor(ends, dtype=torch.int32, device=dev)
        # a caller's own buffer where the batch is padded: its last rows stay as they were
        s["out"] = torch.full((m, n), 3.0, dtype=TYPES[case["out"]], device=dev) if case["tail"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import haagenti_b200 as H

        s["H"] = H
        if case["weight"] == "int4":
            data = s["weights"] if case["op"] == "grouped" else s["weights"][0]
            s["weight"] = H.Int4Weight(data, case["n"], case["k"])
            del s["weights"]
        else:
            s["weight"] = torch.stack(s.pop("weights")) if case["op"] == "grouped" else s.pop("weights")[0]
    return s


def _plain_weight(case, w):
    if case["weight"] == "dense":
        return w.float()
    n, k = case["n"], case["k"]
    scales = w[: n * k // 16].view(torch.float16).float()
    b = w[n * k // 16:]
    q = torch.stack([b & 15, b >> 4], 1).float() - 8.0
    return (q.reshape(-1, 32) * scales[:, None]).reshape(n, k)


def _plain_act(name, z):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.7071067811865476))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    return z


def _plain(case, x, w, bias, gate, residual):
    y = x.float() @ _plain_weight(case, w).t()
    if bias is not None:
        y = y + bias.float()
    y = _plain_act(case["act"], y)
    if gate is not None:
        y = y * gate.float()
    if residual is not None:
        y = y + residual.float()
    return y.to(TYPES[case["out"]])


def run(state):
    case = state["case"]
    if own:
        H = state["H"]
        more = {"bias": state["bias"], "activation": ACT[case["act"]], "gate": state["gate"],
                "residual": state["residual"], "out_dtype": OUT[case["out"]]}
        if case["op"] == "linear":
            return H.linear(state["x"], state["weight"], **more)
        return H.grouped_linear(state["x"], state["weight"], state["offsets"], out=state["out"], **more)
    if case["op"] == "linear":
        return _plain(case, state["x"], state["weights"][0], state["bias"], state["gate"], state["residual"])
    x, out = state["x"], state["out"]
    if out is None:
        out = torch.empty(case["m"], case["n"], dtype=TYPES[case["out"]], device=x.device)
    at = 0
    for e, c in enumerate(state["sizes"]):
        if c:
            r = slice(at, at + c)
            out[r] = _plain(case, x[r], state["weights"][e], state["bias"][e] if case["bias"] else None,
                            state["gate"][r] if case["gate"] else None,
                            state["residual"][r] if case["residual"] else None)
        at += c
    return out


def exact(case, seed):
    """The definition in 64 bits, a block of output features at a time."""
    s = _inputs(case, seed)
    m, n, k = case["m"], case["n"], case["k"]
    sizes_ = s.get("sizes", [m])
    y = torch.full((m, n), 3.0, dtype=torch.float64, device=s["x"].device)
    x = s["x"].double()
    at = 0
    for e, c in enumerate(sizes_):
        rows = torch.arange(at, at + c, device=x.device)
        at += c
        if not c:
            continue
        data = s["weights"][e]
        for low in range(0, n, 4096):
            f = torch.arange(low, min(n, low + 4096), device=x.device)
            if case["weight"] == "dense":
                w = data[f].double()
            else:
                i = f[:, None] * k + torch.arange(k, device=x.device)  # element numbers
                byte = data[n * k // 16 + torch.div(i, 2, rounding_mode="floor")].to(torch.int32)
                nibble = torch.where(i % 2 == 0, byte % 16, torch.div(byte, 16, rounding_mode="floor"))
                w = (nibble - 8).double() * data[: n * k // 16].view(torch.float16)[i // 32].double()
                del i, byte, nibble
            z = torch.einsum("mk,nk->mn", x[rows], w)
            if s["bias"] is not None:
                b = s["bias"].double()
                z += (b[e] if case["op"] == "grouped" else b)[f]
            if case["act"] == "relu":
                z = z.clamp(min=0)
            elif case["act"] == "silu":
                z = z * torch.special.expit(z)
            elif case["act"] == "gelu":
                z = z * torch.special.ndtr(z)
            elif case["act"] == "gelu_tanh":
                z = z * torch.special.expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
            if s["gate"] is not None:
                z = z * s["gate"][rows][:, f].double()
            if s["residual"] is not None:
                z = z + s["residual"][rows][:, f].double()
            y[rows[:, None], f[None, :]] = z
    return y
