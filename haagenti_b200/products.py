"""Products with decoded weights: ``linear`` and ``grouped_linear``.

    y = act(x Wt + bias) * gate + residual

on the GPU, one kernel launch per call and no host synchronisation.  W is a
dense (out_features, in_features) tensor, as ``HctReader.decode`` returns it,
or an ``Int4Weight``: the INT4 payload of a plain INT4 file
(``HctReader.decompress_all``) laid out once for the kernels, so that the
weights are read in 4.5 bits each.  The reference has no counterpart: it hands
its decoded tensors to an external runtime.
"""
from __future__ import annotations

import struct
import threading

from . import (F16, BF16, F32, Unsupported, _as_host_u8, _check, _torch)
from . import _lib as L
from ._lib import ACT_NONE

__all__ = ["Int4Weight", "linear", "grouped_linear", "linear_status"]

_TAG: dict = {}   # torch dtype -> F32 / F16 / BF16
_TYPE: dict = {}  # and back
_raw_stream = None  # device index -> its current stream's cudaStream_t
_forward_ad = None  # torch.autograd.forward_ad


class _Args(threading.local):
    """A thread's hct_b200_linear_args, filled by one pack (half the time of
    setting the fields)."""

    layout = struct.Struct("=15QQIiiiiiii")  # the fields in the header's order

    def __init__(self):
        self.buffer = bytearray(self.layout.size)
        self.args = L.LinearArgs.from_buffer(self.buffer)


_ARGS = _Args()


def _first_call():
    global _raw_stream, _forward_ad
    torch = _torch()
    L.load()
    from torch.autograd import forward_ad as _forward_ad  # noqa: F811
    # the handle alone: torch.cuda.current_stream builds a Stream object, 3 us beside a call's 8
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                          lambda i: torch.cuda.current_stream(i).cuda_stream)
    tags = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
    _TYPE.update({v: k for k, v in tags.items()})
    _TAG.update(tags)  # last, and at once: it tells other threads that all is set


class Int4Weight:
    """A rows x cols matrix in ``quantize_int4`` form (one f16 scale per 32
    values of a row; cols a multiple of 32), or a list of such matrices (one
    per expert, for ``grouped_linear``), laid out for the products.

    ``data`` is a payload: f16 scales, then nibbles, as a CUDA uint8 tensor or
    host bytes; or a list of payloads.  ``device`` is the CUDA device of the
    weight: the payload's, the stream's or the current one by default.  The layout is made
    here, once, and the stream is synchronised before the constructor returns,
    so that the weight may be used on any stream of its device."""

    def __init__(self, data, rows: int, cols: int, device=None, stream=None):
        torch = _torch()
        many = isinstance(data, (list, tuple))
        parts = list(data) if many else [data]
        rows, cols = int(rows), int(cols)
        lib = L.load()
        size = lib.hct_b200_int4_weight_bytes(rows, cols) if rows > 0 and cols > 0 else 0
        if not size:
            raise ValueError(f"an INT4 weight of {rows} x {cols}: cols must be a positive multiple "
                             "of 32 and rows positive")
        if not parts:
            raise ValueError("an INT4 weight needs a payload")
        if device is not None:
            device = torch.device(device)
            if device.type != "cuda":
                raise ValueError(f"an INT4 weight is on a CUDA device, not on {device}")
            if device.index is None:  # the payload's, or the current one
                device = None
        for p in parts:
            if hasattr(p, "is_cuda") and p.is_cuda:
                if p.dtype != torch.uint8 or p.dim() != 1 or not p.is_contiguous():
                    raise ValueError("an INT4 payload is a contiguous 1-D uint8 tensor")
                if device is None:
                    device = p.device
                elif p.device != device:
                    raise ValueError("the payloads of one weight are on one device")
        if device is None:
            device = (stream.device if stream is not None
                      else torch.device("cuda", torch.cuda.current_device()))
        if stream is not None and stream.device != device:
            raise ValueError(f"the stream belongs to {stream.device}, the weight to {device}")
        with torch.cuda.device(device):
            stream = stream if stream is not None else torch.cuda.current_stream()
            with torch.cuda.stream(stream):
                if torch.cuda.is_current_stream_capturing():
                    raise Unsupported(L.UNSUPPORTED, "an INT4 weight cannot be laid out while its "
                                                     "stream is being captured")
                packed = torch.empty(len(parts) * size, dtype=torch.uint8, device=device)
                for i, p in enumerate(parts):
                    if not (hasattr(p, "is_cuda") and p.is_cuda):
                        p = torch.from_numpy(_as_host_u8(p).copy()).to(device)
                    _check(lib.hct_b200_int4_weight_pack(
                        p.data_ptr(), p.numel(), rows, cols, packed.data_ptr() + i * size,
                        stream.cuda_stream))
                stream.synchronize()
        self.rows, self.cols = rows, cols
        self.experts = len(parts) if many else None
        self.packed = packed
        self.home = stream.cuda_stream  # the stream that the memory's allocator knows of
        self.device = device

    @property
    def shape(self):
        s = (self.rows, self.cols)
        return s if self.experts is None else (self.experts,) + s


def _matrix(t, name, shape, dtype, dev):
    """Row stride of an optional (rows, features) operand after its checks."""
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name} must be {shape} of {dtype}, got {tuple(t.shape)} of {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, x on cuda:{dev}")
    ld, step = t.stride()
    if step != 1 and shape[1] > 1:
        raise ValueError(f"the features of {name} must be contiguous")
    return ld


def _product(x, weight, offsets, bias, activation, gate, residual, out_dtype, out, stream):
    torch = _torch()
    if not _TAG:
        _first_call()
    dev = x.get_device()
    if dev < 0 or x.dim() != 2:
        raise ValueError("x must be a 2-D CUDA tensor (rows, in_features)")
    m, k = x.shape
    xt = x.dtype
    x_tag = _TAG.get(xt)
    if not x_tag:  # no type of ours, or F32 (0)
        raise ValueError(f"x must be float16 or bfloat16, got {xt}")
    ldx, step = x.stride()
    if step != 1 and k > 1:
        raise ValueError("the features of x must be contiguous")
    ldw = w_stride = 0
    experts = None
    if isinstance(weight, Int4Weight):
        form, wt = L.WEIGHT_INT4, weight.packed
        n, wk = weight.rows, weight.cols
        experts = weight.experts
    else:
        form, wt = L.WEIGHT_DENSE, weight
        if weight.dtype != xt:
            raise ValueError(f"a dense weight must be of x's type {xt}, got {weight.dtype}")
        if weight.dim() != (2 if offsets is None else 3):
            raise ValueError("a dense weight is (out_features, in_features), with a leading axis "
                             "of experts in grouped_linear")
        if offsets is None:
            n, wk = weight.shape
            ldw, step = weight.stride()
        else:
            experts, n, wk = weight.shape
            w_stride, ldw, step = weight.stride()
        if step != 1 and wk > 1:
            raise ValueError("the input features of a dense weight must be contiguous")
    if wk != k:
        raise ValueError(f"x has {k} features, the weight {wk}")
    if wt.get_device() != dev:
        raise ValueError(f"the weight is on {wt.device}, x on {x.device}")
    bits, off_ptr = 32, 0
    if offsets is None:
        if experts is not None:
            raise ValueError("a weight with experts needs grouped_linear")
        experts = 0
    else:
        if experts is None:
            raise ValueError("grouped_linear needs a weight with experts (an Int4Weight of a list)")
        if offsets.dtype not in (torch.int32, torch.int64) or offsets.get_device() != dev:
            raise ValueError("offsets must be an int32 or int64 tensor on x's device")
        if offsets.dim() != 1 or offsets.shape[0] != experts + 1 or not offsets.is_contiguous():
            raise ValueError(f"offsets must hold experts + 1 = {experts + 1} contiguous values")
        bits = 32 if offsets.dtype == torch.int32 else 64
        off_ptr = offsets.data_ptr()
    if out is not None:
        tag = _TAG.get(out.dtype)
        if tag is None or (out_dtype is not None and out_dtype != tag):
            raise ValueError(f"out is of {out.dtype}, not of out_dtype {out_dtype}")
    else:
        tag = x_tag if out_dtype is None else out_dtype
        if tag not in _TYPE:
            raise ValueError(f"out_dtype must be F32, F16 or BF16, got {out_dtype}")
    ot = _TYPE[tag]
    shape = (m, n)
    bias_tag, bias_ptr, gate_ptr, res_ptr, ldg, ldr = x_tag, 0, 0, 0, 0, 0
    grads = x.requires_grad or wt.requires_grad
    if bias is not None:
        want = (n,) if offsets is None else (experts, n)
        bias_tag = _TAG.get(bias.dtype)
        if (bias_tag != x_tag and bias_tag != F32) or bias.shape != want:
            raise ValueError(f"bias must be {want} of {xt} or float32, got {tuple(bias.shape)} of "
                             f"{bias.dtype}")
        if bias.get_device() != dev or not bias.is_contiguous():
            raise ValueError("bias must be contiguous and on x's device")
        bias_ptr = bias.data_ptr()
        grads |= bias.requires_grad
    if gate is not None:
        ldg, gate_ptr = _matrix(gate, "gate", shape, xt, dev), gate.data_ptr()
        grads |= gate.requires_grad
    if residual is not None:
        ldr, res_ptr = _matrix(residual, "residual", shape, ot, dev), residual.data_ptr()
        grads |= residual.requires_grad
    if out is not None:
        ldo = _matrix(out, "out", shape, ot, dev)
        grads |= out.requires_grad
    if grads and torch.is_grad_enabled():
        raise Unsupported(L.UNSUPPORTED, "the products have no backward pass: detach the tensors "
                                         "or call under torch.no_grad()")
    # dual tensors exist within a dual level alone (one attribute read elsewhere)
    if getattr(_forward_ad, "_current_level", 0) >= 0:
        for t in (x, wt, bias, gate, residual, out):
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise Unsupported(L.UNSUPPORTED, "the products have no forward-mode derivative: "
                                                 "pass the tensors' primal parts")
    lib = L._lib
    fn = lib.hct_b200_linear if offsets is None else lib.hct_b200_grouped_linear
    here = torch.cuda.current_device() == dev
    if here and stream is None:
        if out is None:  # sizes one by one: a tuple takes torch 1 us longer to read
            out = x.new_empty(m, n) if ot is xt else torch.empty(m, n, dtype=ot, device=x.device)
            ldo = n
        a = _ARGS
        try:
            a.layout.pack_into(a.buffer, 0, m, n, k, x.data_ptr(), ldx, wt.data_ptr(), ldw, w_stride,
                               bias_ptr, gate_ptr, ldg, res_ptr, ldr, out.data_ptr(), ldo,
                               off_ptr, experts, bits, x_tag, form, bias_tag, tag, activation, 0)
        except struct.error:  # every other value has been checked
            raise ValueError("activation must be one of the ACT_ constants, "
                             f"got {activation!r}") from None
        raw = _raw_stream(dev)
        rc = fn(a.args, raw)
        if rc:
            _check(rc)
        if form and raw != weight.home:  # freed weights stay until this stream is done
            wt.record_stream(torch.cuda.current_stream())
        return out
    with torch.cuda.device(dev):
        current = torch.cuda.current_stream()
        if stream is None or stream == current:
            return _product(x, weight, offsets, bias, activation, gate, residual, out_dtype, out,
                            None)
        if stream.device.index != dev:
            raise ValueError(f"the stream belongs to {stream.device}, x to {x.device}")
        with torch.cuda.stream(stream):
            o = _product(x, weight, offsets, bias, activation, gate, residual, out_dtype, out, None)
        # the caller's tensors are read on a stream that their allocator does not know of
        for t in (x, wt, offsets, bias, gate, residual, out):
            if t is not None:
                t.record_stream(stream)
        return o


def linear(x, weight, bias=None, activation: int = ACT_NONE, gate=None, residual=None,
           out_dtype: int | None = None, out=None, stream=None):
    """act(x Wt + bias) * gate + residual: (rows, out_features) of ``out_dtype``.

    ``x`` is (rows, in_features) in float16 or bfloat16, with contiguous
    features and any row stride; ``weight`` a dense tensor of x's type or an
    ``Int4Weight``; ``bias`` (out_features,) of x's type or float32;
    ``activation`` one of the ACT_ constants; ``gate`` (rows, out_features) of
    x's type; ``residual`` of the output's type, which is x's by default.
    ``out`` may be ``gate`` or ``residual`` itself.  Sums are held in f32 and
    the result rounded once.  ``out_dtype=F32`` keeps INT4 weights exact; a
    16-bit output of more than 16 rows rounds them to x's type, as ``decode``
    does.
    There is no derivative: tensors that require a gradient are refused while
    autograd records, and dual tensors of forward-mode differentiation always.
    The call does not wait for the device: ``linear_status`` does, and raises if
    a product ran into a device-side timeout."""
    return _product(x, weight, None, bias, activation, gate, residual, out_dtype, out, stream)


def grouped_linear(x, weight, offsets, bias=None, activation: int = ACT_NONE, gate=None,
                   residual=None, out_dtype: int | None = None, out=None, stream=None):
    """``linear`` with one weight per expert: rows [offsets[e], offsets[e+1]) of
    ``x``, which is sorted by expert, go through expert e.

    ``weight`` is a dense (experts, out_features, in_features) tensor or an
    ``Int4Weight`` of a list; ``bias`` (experts, out_features); ``offsets``
    experts + 1 ascending int32 or int64 values on x's device, read there (no
    synchronisation).  Rows before offsets[0] and from offsets[-1] on are left
    as they were in ``out`` (undefined where ``out`` is not given)."""
    if offsets is None:
        raise ValueError("grouped_linear needs offsets")
    return _product(x, weight, offsets, bias, activation, gate, residual, out_dtype, out, stream)


def linear_status(device=None, stream=None):
    """Synchronise the stream and raise if a product on the device ran into a
    device-side timeout that no call has reported yet (its output is then
    undefined).  Products on other streams may be running still: theirs is
    reported by a later call."""
    torch = _torch()
    if device is None:
        device = stream.device if stream is not None else torch.cuda.current_device()
    with torch.cuda.device(device):
        s = stream if stream is not None else torch.cuda.current_stream()
        _check(L.load().hct_b200_linear_status(s.cuda_stream))
