"""Operators of a feed-forward layer in 8 bits (no counterpart in the reference,
whose trunk runs in fp32).

Serving: `add_rms_norm_int8` -> `linear_int8` -> `swiglu_int8` -> `linear_int8`
keeps every row that a product reads in 8 bits. Training: `add_rms_norm` and
`swiglu` differentiate, and `swiglu(..., checkpoint="int8")` keeps what its
backward reads in 8 bits.

Activations are float32, bfloat16 or float16 CUDA tensors (..., channels); the
arithmetic is fp32. A last dimension of stride 1 whose rows lie at one pitch is
taken as it is, other layouts are copied first. Calls run on the current stream
of the tensors' device, may be captured into CUDA graphs, and keep nothing
between one another. Arguments that do not fit raise ValueError. There is no CPU
path, no second derivative, and no forward-mode one (tensors with a tangent are
refused).

The checks, outputs and autograd nodes are native (csrc/feedforward_torch.cpp):
in Python they take longer than the kernels of a decode step.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

_native_module = None


def _native():
    global _native_module
    if _native_module is None:
        _lib.lib()
        try:
            from . import _feedforward
        except ImportError as error:
            raise RuntimeError("_feedforward.so is not built for this interpreter and torch; run "
                               "`python jittor-flow2surf_b200/build.py` (or "
                               "__graft_entry__.build())") from error
        _native_module = _feedforward
    return _native_module


class Int8Rows(NamedTuple):
    """Rows in 8 bits: `values` (..., channels) int8 and `scale` (...) float32,
    standing for values * scale[..., None]. The library's rows start on
    multiples of 16 bytes, which the tensor-core product needs; `values` is
    then a view of a wider buffer where channels is not a multiple of 16, and
    clone, to(device), contiguous, cat and indexing give rows without that pitch:
    linear_int8 takes them too, but on the CUDA cores, 10 to 60 times slower, so
    move and cut such weights before quantize_rows. Scales that want a gradient
    are refused, since none would come."""

    values: torch.Tensor
    scale: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """What the rows stand for, in `dtype`."""
        return _native().dequantize_rows(self.values, self.scale, dtype)


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """Rows (..., channels) in 8 bits: per row, scale = max|x| / 127 and the
    whole numbers nearest to 127 x / max|x| (the even one at a tie). A row with
    a value that is not finite gets the scale NaN. Weights (cols, K) are
    quantised once with it, a scale per output channel. At most 32768
    channels. No gradient."""
    return Int8Rows(*_native().quantize_rows(x))


def linear_int8(x: Int8Rows, weight: Int8Rows, bias: torch.Tensor | None = None, *,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x weight^T + bias of 8-bit rows x (..., K) and weight (cols, K), with a
    scale per token and per output channel: the sum over K is exact in 32-bit
    integers (K at most 131071), scales and bias (cols, of `dtype`) are applied
    in fp32, the token's scale first (a sum times it beyond 3.4e38 is infinite),
    and the result (..., cols) is rounded to `dtype` once. Rows and cols at most
    2^31 - 256. No gradient."""
    xv, xs = x
    wv, ws = weight
    return _native().linear_int8(xv, xs, wv, ws, bias, dtype)


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                 eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """Add a residual and take the root-mean-square norm of the sum.

    stream = x + residual, rounded to x's type (x itself without a residual);
    normed = stream / sqrt(mean(stream^2) + eps) * weight, of the stream as it
    is stored. x and residual (..., C), weight (C,), all of one type, C at most
    32768 -> (normed, stream). Differentiable in x, residual and weight; the
    weight's gradient is summed over the rows in fp32, in a fixed order."""
    return _native().add_rms_norm(x, weight, residual, eps)


def add_rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                      *, eps: float = 1e-6) -> tuple[Int8Rows, torch.Tensor]:
    """add_rms_norm with the normed rows in 8 bits, for linear_int8:
    (Int8Rows, stream). The values are the whole numbers nearest to
    127 p / max|p| with p = stream * weight (the norm cancels, and p may lie past
    fp32 at either end), the scale is max|p| / (127 sqrt(mean(stream^2) + eps)). No
    gradient."""
    values, scale, stream = _native().add_rms_norm_int8(x, weight, residual, eps)
    return Int8Rows(values, scale), stream


def swiglu(projected: torch.Tensor, *, checkpoint: str | None = None) -> torch.Tensor:
    """value * gate * sigmoid(gate) of a packed projection (..., 2 H) =
    [gate | value] -> (..., H). Differentiable. A sigmoid below 2^-126 (gates below
    -87.3) is 0. `checkpoint` None keeps the
    projection for the backward; "int8" keeps it in 8 bits (a scale for every
    128 channels of the gate and of the value: 52% of the bytes of a 16-bit
    type), and the backward is that of the kept values: each is off by at most
    half of 1/127 of the largest magnitude in its group."""
    if checkpoint not in (None, "int8"):
        raise ValueError(f"checkpoint must be None or 'int8', got {checkpoint!r}")
    return _native().swiglu(projected, checkpoint is not None)


def swiglu_int8(projected: torch.Tensor) -> Int8Rows:
    """swiglu with its rows in 8 bits, for linear_int8: as
    quantize_rows(swiglu(projected)) with the product kept in fp32 until it is
    rounded to 8 bits. H at most 32768. No gradient."""
    return Int8Rows(*_native().swiglu_int8(projected))
