"""Operators of a feed-forward layer in 8 bits (no counterpart in the reference,
whose trunk runs in fp32).

Serving: `add_rms_norm_int8` -> `linear_int8` -> `swiglu_int8` -> `linear_int8`
keeps every row that a product reads in 8 bits. Training: `add_rms_norm` and
`swiglu` differentiate, and `swiglu(..., checkpoint="int8")` keeps what its
backward reads in 8 bits.

Activations are float32, bfloat16 or float16 CUDA tensors (..., channels); the
arithmetic is fp32. A last dimension of stride 1 whose rows lie at one pitch is
taken as it is, other layouts are copied first. There is no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _needs_grad, _require_cuda

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # f2s_dtype
_SWIGLU_GROUP = 128  # F2S_SWIGLU_GROUP


def _dtype(dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"expected float32, bfloat16 or float16, got {dtype}")
    return code


def _rows(t: torch.Tensor):
    """(tensor, rows, pitch) of a (..., channels) tensor read as rows of one pitch."""
    width = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // width, width
    dims = t.dim()
    if t.stride(-1) == 1 and dims >= 2 and t.stride(-2) >= width and all(
            t.stride(i) == t.stride(i + 1) * t.shape[i + 1] for i in range(dims - 2)):
        return t, t.numel() // width, t.stride(-2)
    return t.contiguous(), t.numel() // width, width


def _check_rows(name: str, t: torch.Tensor) -> None:
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} must be (..., channels) with at least one channel, "
                         f"got {tuple(t.shape)}")


def _same_device(first: torch.Tensor, *others) -> None:
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"tensors lie on different devices: {first.device} and {t.device}")


_ENTRIES: dict = {}  # name -> entry point of the loaded library


def _call(device: torch.device, name: str, *args) -> None:
    """Launch on `device`'s current stream, whichever device is current. (The
    stream's handle is asked for directly: building a Stream object for it
    takes longer than a launch.)"""
    entry = _ENTRIES.get(name)
    if entry is None:
        entry = _ENTRIES[name] = getattr(_lib.lib(), name)
    index = device.index
    if index == torch.cuda.current_device():
        status = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            status = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status)


def _empty(like: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(like, memory_format=torch.contiguous_format)


class Int8Rows(NamedTuple):
    """Rows in 8 bits: `values` (..., channels) int8 and `scale` (...) float32,
    standing for values * scale[..., None]. The library's rows start on
    multiples of 16 bytes, which the tensor-core product needs; `values` is
    then a view of a wider buffer where channels is not a multiple of 16."""

    values: torch.Tensor
    scale: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """What the rows stand for, in `dtype`."""
        code = _dtype(dtype)
        values, scale = _check_int8("rows", self)
        out = torch.empty_like(values, dtype=dtype, memory_format=torch.contiguous_format)
        if out.numel() == 0:
            return out
        values, rows, pitch = _rows(values)
        width = values.shape[-1]
        _call(values.device, "f2s_dequantize_rows", values.data_ptr(), pitch, scale.data_ptr(),
              rows, width, out.data_ptr(), width, code)
        return out


def _check_int8(name: str, rows: Int8Rows):
    values, scale = rows
    _check_rows(name, values)
    if values.dtype != torch.int8 or scale.dtype != torch.float32:
        raise ValueError(f"{name} must hold int8 values and float32 scales, got {values.dtype} "
                         f"and {scale.dtype}")
    if scale.shape != values.shape[:-1]:
        raise ValueError(f"{name}: scales {tuple(scale.shape)} do not match values "
                         f"{tuple(values.shape)}")
    _require_cuda(values, scale)
    _same_device(values, scale)
    return values, scale if scale.is_contiguous() else scale.contiguous()


def _empty_int8(like: torch.Tensor, width: int | None = None) -> tuple[Int8Rows, int]:
    """Unset 8-bit rows with the leading shape of `like` (its width unless given)
    and their pitch, a multiple of 16."""
    lead = like.shape[:-1]
    if width is None:
        width = like.shape[-1]
    pitch = -(-width // 16) * 16
    values = like.new_empty((*lead, pitch), dtype=torch.int8)
    if pitch != width:
        values = values[..., :width]
    return Int8Rows(values, like.new_empty(lead, dtype=torch.float32)), pitch


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """Rows (..., channels) in 8 bits: per row, scale = max|x| / 127 and the
    whole numbers nearest to 127 x / max|x| (the even one at a tie). A row with
    a value that is not finite gets the scale NaN. Weights (cols, K) are
    quantised once with it, a scale per output channel. At most 32768
    channels."""
    _check_rows("x", x)
    code = _dtype(x.dtype)
    _require_cuda(x)
    if _needs_grad(x):
        raise ValueError("8-bit rows have no gradient; call quantize_rows under torch.no_grad()")
    out, pitch = _empty_int8(x)
    if x.numel() == 0:
        return out
    x, rows, ldx = _rows(x)
    _call(x.device, "f2s_quantize_rows", x.data_ptr(), ldx, code, rows, x.shape[-1],
          out.values.data_ptr(), pitch, out.scale.data_ptr())
    return out


def linear_int8(x: Int8Rows, weight: Int8Rows, bias: torch.Tensor | None = None, *,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x weight^T + bias of 8-bit rows x (..., K) and weight (cols, K), with a
    scale per token and per output channel: the sum over K is exact in 32-bit
    integers (K at most 131071), scales and bias (cols, of `dtype`) are applied
    in fp32, and the result (..., cols) is rounded to `dtype` once. No
    gradient."""
    code = _dtype(dtype)
    xv, xs = _check_int8("x", x)
    wv, ws = _check_int8("weight", weight)
    if wv.dim() != 2:
        raise ValueError(f"weight must be (cols, K), got {tuple(wv.shape)}")
    cols, K = wv.shape
    if xv.shape[-1] != K:
        raise ValueError(f"x has {xv.shape[-1]} channels, weight {K}")
    _same_device(xv, wv, bias)
    if bias is not None:
        if bias.shape != (cols,) or bias.dtype != dtype:
            raise ValueError(f"bias must be ({cols},) of {dtype}, got {tuple(bias.shape)} of "
                             f"{bias.dtype}")
        if _needs_grad(bias):
            raise ValueError("the 8-bit product has no gradient; call linear_int8 under "
                             "torch.no_grad()")
        bias = bias.contiguous()
    out = xv.new_empty((*xv.shape[:-1], cols), dtype=dtype)
    if out.numel() == 0:
        return out
    xv, rows, ldx = _rows(xv)
    wv, _, ldw = _rows(wv)
    if rows > 2**31 - 1:
        raise ValueError(f"linear_int8 takes at most 2^31 - 1 rows, got {rows}")
    _call(xv.device, "f2s_linear_int8", xv.data_ptr(), ldx, xs.data_ptr(), wv.data_ptr(), ldw,
          ws.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), cols, code,
          rows, cols, K)
    return out


def _check_norm(x, weight, residual):
    _check_rows("x", x)
    code = _dtype(x.dtype)
    if weight.shape != (x.shape[-1],) or weight.dtype != x.dtype:
        raise ValueError(f"weight must be ({x.shape[-1]},) of {x.dtype}, got "
                         f"{tuple(weight.shape)} of {weight.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must be {tuple(x.shape)} of {x.dtype}, got "
                         f"{tuple(residual.shape)} of {residual.dtype}")
    _require_cuda(x, weight)
    if residual is not None:
        _require_cuda(residual)
    _same_device(x, weight, residual)
    return code


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                 eps: float = 1e-6):
    """Add a residual and take the root-mean-square norm of the sum.

    stream = x + residual, rounded to x's type (x itself without a residual);
    normed = stream / sqrt(mean(stream^2) + eps) * weight, of the stream as it
    is stored. x and residual (..., C), weight (C,), all of one type, C at most
    32768 -> (normed, stream). Differentiable in x, residual and weight; the
    weight's gradient is summed over the rows in fp32, in a fixed order."""
    code = _check_norm(x, weight, residual)
    if _needs_grad(x, weight) or (residual is not None and _needs_grad(residual)):
        if residual is None:
            return _AddRmsNorm.apply(x, weight, None, eps, code), x
        return _AddRmsNorm.apply(x, weight, residual, eps, code)
    normed, stream = _norm_forward(x, weight, residual, eps, code)
    return normed, stream


def _norm_forward(x, weight, residual, eps, code):
    normed = _empty(x)
    stream = x if residual is None else _empty(x)
    if x.numel() == 0:
        return normed, stream
    width = x.shape[-1]
    weight = weight.contiguous()
    x, rows, ldx = _rows(x)
    if residual is None:
        _call(x.device, "f2s_add_rms_norm", x.data_ptr(), ldx, None, 0, weight.data_ptr(), code,
              rows, width, eps, None, normed.data_ptr())
    else:
        residual, _, ldr = _rows(residual)
        _call(x.device, "f2s_add_rms_norm", x.data_ptr(), ldx, residual.data_ptr(), ldr,
              weight.data_ptr(), code, rows, width, eps, stream.data_ptr(), normed.data_ptr())
    return normed, stream


class _AddRmsNorm(torch.autograd.Function):
    """add_rms_norm with its backward, which reads the stream (the norm's
    reciprocal root is recomputed from it, so no statistics are kept)."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps, code):
        ctx.set_materialize_grads(False)
        normed, stream = _norm_forward(x, weight, residual, eps, code)
        ctx.save_for_backward(stream, weight)
        ctx.eps, ctx.code, ctx.added = eps, code, residual is not None
        return (normed, stream) if ctx.added else normed

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstream=None):
        stream, weight = ctx.saved_tensors
        need_x, need_weight, need_residual = ctx.needs_input_grad[:3]
        if dy is None:  # only the stream was used
            return (dstream if need_x else None, torch.zeros_like(weight) if need_weight else None,
                    dstream if need_residual else None, None, None)
        width = stream.shape[-1]
        dx = _empty(stream)
        dweight = _empty(weight) if need_weight else None
        if stream.numel() == 0:
            return (dx if need_x else None, dweight.zero_() if need_weight else None,
                    dx if need_residual else None, None, None)
        weight = weight.contiguous()
        s, rows, lds = _rows(stream)
        dy, _, lddy = _rows(dy)
        ds, ldds = None, 0
        if dstream is not None:
            dstream, _, ldds = _rows(dstream)
            ds = dstream.data_ptr()
        ws, size = None, ctypes.c_size_t(0)
        if need_weight:
            _lib.call("f2s_add_rms_norm_backward_workspace_bytes", rows, width, ctypes.byref(size))
            ws = s.new_empty(size.value, dtype=torch.uint8)
        _call(s.device, "f2s_add_rms_norm_backward", s.data_ptr(), lds, weight.data_ptr(), ctx.code,
              rows, width, ctx.eps, dy.data_ptr(), lddy, ds, ldds, dx.data_ptr(),
              None if dweight is None else dweight.data_ptr(),
              None if ws is None else ws.data_ptr(), size.value)
        return dx if need_x else None, dweight, dx if need_residual else None, None, None


def add_rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                      *, eps: float = 1e-6):
    """add_rms_norm with the normed rows in 8 bits, for linear_int8:
    (Int8Rows, stream). The values are the whole numbers nearest to
    127 p / max|p| with p = stream * weight (the norm cancels), the scale is
    max|p| / (127 sqrt(mean(stream^2) + eps)). No gradient."""
    code = _check_norm(x, weight, residual)
    if _needs_grad(x, weight) or (residual is not None and _needs_grad(residual)):
        raise ValueError("8-bit rows have no gradient; call add_rms_norm_int8 under "
                         "torch.no_grad(), or add_rms_norm")
    out, pitch = _empty_int8(x)
    stream = x if residual is None else _empty(x)
    if x.numel() == 0:
        return out, stream
    width = x.shape[-1]
    weight = weight.contiguous()
    x, rows, ldx = _rows(x)
    ldr = 0
    if residual is not None:
        residual, _, ldr = _rows(residual)
    _call(x.device, "f2s_add_rms_norm_int8", x.data_ptr(), ldx,
          None if residual is None else residual.data_ptr(), ldr, weight.data_ptr(), code, rows,
          width, eps, None if residual is None else stream.data_ptr(), out.values.data_ptr(),
          pitch, out.scale.data_ptr())
    return out, stream


def _check_projected(projected: torch.Tensor) -> int:
    _check_rows("projected", projected)
    if projected.shape[-1] % 2:
        raise ValueError(f"projected must be (..., 2 H) = [gate | value], got "
                         f"{tuple(projected.shape)}")
    code = _dtype(projected.dtype)
    _require_cuda(projected)
    return code


def swiglu(projected: torch.Tensor, *, checkpoint: str | None = None) -> torch.Tensor:
    """value * gate * sigmoid(gate) of a packed projection (..., 2 H) =
    [gate | value] -> (..., H). Differentiable. `checkpoint` None keeps the
    projection for the backward; "int8" keeps it in 8 bits (a scale for every
    128 channels of the gate and of the value: 52% of the bytes of a 16-bit
    type), and the backward is that of the kept values: each is off by at most
    half of 1/127 of the largest magnitude in its group."""
    if checkpoint not in (None, "int8"):
        raise ValueError(f"checkpoint must be None or 'int8', got {checkpoint!r}")
    code = _check_projected(projected)
    if _needs_grad(projected):
        return _SwiGlu.apply(projected, checkpoint is not None, code)
    return _swiglu_forward(projected, code, None, None)


def _swiglu_forward(projected, code, kept, scales):
    hidden = projected.shape[-1] // 2
    out = projected.new_empty((*projected.shape[:-1], hidden))
    if out.numel() == 0:
        return out
    p, rows, ld = _rows(projected)
    _call(p.device, "f2s_swiglu", p.data_ptr(), ld, code, rows, hidden, out.data_ptr(),
          None if kept is None else kept.data_ptr(), None if kept is None else scales.data_ptr())
    return out


class _SwiGlu(torch.autograd.Function):
    """swiglu with its backward, from the projection or its 8-bit checkpoint."""

    @staticmethod
    def forward(ctx, projected, keep8, code):
        hidden = projected.shape[-1] // 2
        ctx.shape, ctx.code, ctx.keep8 = projected.shape, code, keep8
        if not keep8:
            ctx.save_for_backward(projected)
            return _swiglu_forward(projected, code, None, None)
        groups = projected.numel() // (2 * hidden) * -(-hidden // _SWIGLU_GROUP)
        kept = projected.new_empty(groups * 2 * _SWIGLU_GROUP, dtype=torch.int8)
        scales = projected.new_empty(2 * groups, dtype=torch.float32)
        ctx.save_for_backward(kept, scales)
        return _swiglu_forward(projected, code, kept, scales)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        grad = dy.new_empty(ctx.shape)
        if grad.numel() == 0:
            return grad, None, None
        hidden = ctx.shape[-1] // 2
        dy, rows, lddy = _rows(dy)
        if ctx.keep8:
            kept, scales = ctx.saved_tensors
            args = (None, 0, kept.data_ptr(), scales.data_ptr())
        else:
            p, _, ld = _rows(ctx.saved_tensors[0])
            args = (p.data_ptr(), ld, None, None)
        _call(dy.device, "f2s_swiglu_backward", *args, dy.data_ptr(), lddy, ctx.code, rows, hidden,
              grad.data_ptr())
        return grad, None, None


def swiglu_int8(projected: torch.Tensor) -> Int8Rows:
    """swiglu with its rows in 8 bits, for linear_int8: as
    quantize_rows(swiglu(projected)) with the product kept in fp32 until it is
    rounded to 8 bits. H at most 32768. No gradient."""
    code = _check_projected(projected)
    if _needs_grad(projected):
        raise ValueError("8-bit rows have no gradient; call swiglu_int8 under torch.no_grad(), "
                         "or swiglu")
    hidden = projected.shape[-1] // 2
    out, pitch = _empty_int8(projected, hidden)
    if out.values.numel() == 0:
        return out
    p, rows, ld = _rows(projected)
    _call(p.device, "f2s_swiglu_int8", p.data_ptr(), ld, code, rows, hidden,
          out.values.data_ptr(), pitch, out.scale.data_ptr())
    return out
