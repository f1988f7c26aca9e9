"""The 8-bit feed-forward operators against plain implementations in 64 bits.

Tolerances count roundings: half a step of the output's type relative to the
value, and for the fp32 arithmetic before it u = 2^-24 for each operation on
the way (a sum of n terms: n - 1 roundings whatever its order, or its depth
where the order is known). 8-bit values of rows that are inputs have to be
equal to the nearest whole numbers of the exact quotient.
"""

import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import flow2surf_b200 as f2s
from flow2surf_b200 import _lib
from flow2surf_b200.feedforward import Int8Rows

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# A row's sum of squares: 32 terms a thread at most, then 10 levels of pairs;
# the square root halves it, and its own, the division's and the two products'
# roundings follow.
DEPTH = 32 + 10
NORM = DEPTH / 2 + 4


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the spacing of the subnormal values."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def close(got, want, bound):
    """|got - want| <= bound, elementwise, in 64 bits."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    over = ((got - want).abs() - bound).max().item() if got.numel() else -1.0
    assert over <= 0, f"off by {(got - want).abs().max().item():.3e}, over the bound by {over:.3e}"


def nearest_whole(v, m):
    """Whole numbers nearest to 127 v / m (64 bits), the even one at a tie."""
    below = torch.floor(127 * v / torch.where(m > 0, m, 1.0))
    twice = 254 * v - (2 * below + 1) * m
    up = (twice > 0) | ((twice == 0) & (below.remainder(2) == 1))
    return torch.where(m > 0, below + up, 0.0).to(torch.int8)


def row_scale(m):
    """m / 127 rounded to fp32 once (in torch, an fp32 division by a number is a
    product with its reciprocal)."""
    return (m.double() / 127).float()


def row_max(v):
    return v.abs().amax(-1, keepdim=True)


def normal(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype)


def padded(t, extra=24):
    """The same rows at a wider pitch (a view of a larger buffer)."""
    held = torch.full((*t.shape[:-1], t.shape[-1] + extra), 7, dtype=t.dtype, device=t.device)
    held[..., : t.shape[-1]] = t
    return held[..., : t.shape[-1]]


def shifted(t):
    """The same values from a start that is not 16-byte aligned."""
    held = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    held[1:] = t.reshape(-1)
    return held[1:].view(t.shape)


WIDTHS = [1, 7, 8, 24, 64, 192, 200, 257, 1000, 1024, 1531, 4096, 5000, 8192, 16391, 32768]


def norm64(x, weight, residual, eps):
    stream = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    s, w = stream.double(), weight.double()
    rstd = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    return stream, s, w, rstd


# ---- refusals, on the host ----


def test_refusals_on_the_host():
    x, w = torch.zeros(4, 8), torch.ones(8)
    eight = Int8Rows(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4))
    for call in (lambda: f2s.add_rms_norm(x, w), lambda: f2s.add_rms_norm_int8(x, w),
                 lambda: f2s.quantize_rows(x), lambda: f2s.swiglu(x), lambda: f2s.swiglu_int8(x),
                 lambda: f2s.linear_int8(eight, eight), lambda: eight.dequantize()):
        with pytest.raises(ValueError, match="CUDA tensors"):
            call()
    with pytest.raises(ValueError, match="weight must be"):
        f2s.add_rms_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="weight must be"):
        f2s.add_rms_norm(x.bfloat16(), w)
    with pytest.raises(ValueError, match="residual must be"):
        f2s.add_rms_norm(x, w, torch.zeros(1, 8))
    with pytest.raises(ValueError, match="residual must be"):
        f2s.add_rms_norm_int8(x, w, x.half())
    with pytest.raises(ValueError, match="expected float32, bfloat16 or float16"):
        f2s.add_rms_norm(x.double(), w.double())
    with pytest.raises(ValueError, match="at least one channel"):
        f2s.quantize_rows(torch.zeros(3, 0))
    with pytest.raises(ValueError, match="at least one channel"):
        f2s.quantize_rows(torch.zeros(()))
    with pytest.raises(ValueError, match="2 H"):
        f2s.swiglu(torch.zeros(3, 5))
    with pytest.raises(ValueError, match="checkpoint must be"):
        f2s.swiglu(x, checkpoint="int4")
    with pytest.raises(ValueError, match="int8 values and float32 scales"):
        f2s.linear_int8(Int8Rows(x, torch.zeros(4)), eight)
    with pytest.raises(ValueError, match="do not match values"):
        Int8Rows(eight.values, torch.zeros(3)).dequantize()
    with pytest.raises(ValueError, match="expected float32, bfloat16 or float16"):
        f2s.linear_int8(eight, eight, dtype=torch.int32)


def test_entries_validate_on_the_host():
    """Sizes, limits, pointers and types, before any device work; no rows are
    no work."""
    lib = _lib.lib()
    bad, beyond, ok = _lib.F2S_ERR_INVALID_ARGUMENT, _lib.F2S_ERR_UNSUPPORTED, _lib.F2S_OK
    eps = ctypes.c_float(1e-6)
    norm = lambda rows, C, dtype=0, ld=64: lib.f2s_add_rms_norm(  # noqa: E731
        None, ld, None, 0, None, dtype, rows, C, eps, None, None, None)
    assert norm(0, 64) == ok and norm(3, 64) == bad and norm(3, 0) == bad and norm(-1, 8) == bad
    assert norm(3, 64, 5) == bad and b"unknown dtype" in lib.f2s_last_error()
    assert norm(3, 32769) == beyond and b"at most 32768" in lib.f2s_last_error()
    assert lib.f2s_add_rms_norm(16, 4, None, 0, 16, 0, 3, 64, eps, None, 16, None) == bad
    assert b"pitch" in lib.f2s_last_error()
    assert lib.f2s_add_rms_norm_int8(16, 64, None, 0, 16, 0, 3, 64, eps, None, 16, 8, 16, None) == bad
    size = ctypes.c_size_t()
    assert lib.f2s_add_rms_norm_backward_workspace_bytes(1000, 192, ctypes.byref(size)) == ok
    assert size.value > 0
    assert lib.f2s_add_rms_norm_backward(16, 192, 16, 0, 1000, 192, eps, 16, 192, None, 0, 16, 16,
                                         16, size.value - 1, None) == _lib.F2S_ERR_WORKSPACE
    assert lib.f2s_quantize_rows(None, 8, 0, 0, 8, None, 8, None, None) == ok
    assert lib.f2s_quantize_rows(16, 8, 0, 2, 8, 16, 4, 16, None) == bad
    assert lib.f2s_quantize_rows(16, 40000, 0, 2, 40000, 16, 40000, 16, None) == beyond
    assert lib.f2s_dequantize_rows(16, 8, 16, 2, 8, 16, 8, 3, None) == bad
    linear = lambda rows, cols, K, ld=1 << 20: lib.f2s_linear_int8(  # noqa: E731
        16, ld, 16, 16, ld, 16, None, 16, ld, 0, rows, cols, K, None)
    assert linear(0, 8, 8) == ok and linear(1, 0, 8) == bad and linear(1, 8, 0) == bad
    assert linear(1, 8, 131072) == beyond and linear(1, 8, 16, 4) == bad
    assert lib.f2s_swiglu(None, 16, 0, 0, 8, None, None, None, None) == ok
    assert lib.f2s_swiglu(16, 15, 0, 2, 8, 16, None, None, None) == bad
    assert lib.f2s_swiglu(16, 16, 0, 2, 8, 16, 16, None, None) == bad
    assert lib.f2s_swiglu(16, 16, 0, 2, 8, 16, 12, 16, None) == bad
    assert lib.f2s_swiglu_backward(None, 0, None, None, 16, 8, 0, 2, 8, 16, None) == bad
    assert lib.f2s_swiglu_int8(16, 80000, 0, 2, 40000, 16, 40000, 16, None) == beyond


def test_plain_gradients_against_differences():
    """The formulas that the kernels' gradients are held to, against central
    differences in 64 bits: h^2 truncation and rounding / h, 1e-9 together."""
    g = torch.Generator().manual_seed(3)
    x, dy, ds = (torch.randn(3, 7, generator=g, dtype=torch.float64) for _ in range(3))
    w = torch.randn(7, generator=g, dtype=torch.float64)

    def value(x, w):
        return (x * (x.square().mean(-1, keepdim=True) + 0.1).rsqrt() * w * dy).sum() + (x * ds).sum()

    def difference(f, at, h=1e-5):
        out = torch.empty_like(at)
        for i in range(at.numel()):
            up, down = at.clone(), at.clone()
            up.view(-1)[i] += h
            down.view(-1)[i] -= h
            out.view(-1)[i] = (f(up) - f(down)) / (2 * h)
        return out

    dx, dw, _ = norm_grad64(x, w, dy, ds, 0.1)
    close(dx, difference(lambda v: value(v, w), x), 1e-8)
    close(dw, difference(lambda v: value(x, v), w), 1e-8)
    p = torch.randn(2, 10, generator=g, dtype=torch.float64)
    d = torch.randn(2, 5, generator=g, dtype=torch.float64)
    dp = swiglu_grad64(p[:, :5], p[:, 5:], d)
    close(dp, difference(lambda v: (v[:, :5] * torch.sigmoid(v[:, :5]) * v[:, 5:] * d).sum(), p), 1e-8)


def norm_grad64(s, w, dy, ds, eps):
    """(dx, dw, the pieces whose roundings count)."""
    s, w, dy = s.double(), w.double(), dy.double()
    rstd = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    u, n = dy * w, s * rstd
    dx = rstd * (u - n * (u * n).mean(-1, keepdim=True))
    if ds is not None:
        dx = dx + ds.double()
    return dx, (dy * n).flatten(0, -2).sum(0), (rstd, u, n)


def swiglu_grad64(gate, value, dy):
    gate, value, dy = gate.double(), value.double(), dy.double()
    sigma = torch.sigmoid(gate)
    return torch.cat([dy * value * sigma * (1 + gate * (1 - sigma)), dy * gate * sigma], -1)


# ---- RMS norm ----


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_forward(cuda, width, dtype):
    for rows, layout in ((1, None), (37, None), (5, padded), (6, shifted)):
        for added in (True, False):
            x = normal(rows, width, dtype=dtype, seed=width + rows).to(cuda)
            r = normal(rows, width, dtype=dtype, seed=width + rows + 1, scale=3).to(cuda) if added else None
            w = normal(width, dtype=dtype, seed=width).to(cuda)
            want_stream, s, w64, rstd = norm64(x, w, r, 1e-6)
            xs, rs = (x, r) if layout is None else (layout(x), None if r is None else layout(r))
            y, stream = f2s.add_rms_norm(xs, w, rs)
            assert torch.equal(stream, want_stream)
            y64 = s * rstd * w64
            close(y, y64, y64.abs() * (half_step(dtype) + NORM * U) * 1.001 + smallest(dtype))
            if layout is None and rows == 1:
                continue
            eight, stream = f2s.add_rms_norm_int8(xs, w, rs)
            assert torch.equal(stream, want_stream)
            p = s * w64
            assert torch.equal(eight.values, nearest_whole(p, row_max(p)))
            scale = (row_max(p) * rstd / 127)[:, 0]
            close(eight.scale, scale, scale * (NORM + 2) * U + 1e-45)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 4096), (2, 7), (33, 24), (300, 192), (301, 200), (67, 1531),
                                        (5000, 64), (1300, 1000), (40, 8192), (700, 5000), (3, 32768), (2, 16391)])
def test_norm_backward(cuda, rows, width, dtype):
    x = normal(rows, width, dtype=dtype, seed=1).to(cuda).requires_grad_()
    r = normal(rows, width, dtype=dtype, seed=2, scale=2).to(cuda).requires_grad_()
    w = normal(width, dtype=dtype, seed=3).to(cuda).requires_grad_()
    dy, ds = (normal(rows, width, dtype=dtype, seed=s).to(cuda) for s in (4, 5))
    eps = 1e-5

    def check(s, got_dx, got_dw, ds):
        dx, dw, (rstd, u, n) = norm_grad64(s, w.detach(), dy, ds, eps)
        # u: one rounding; mean(u n): two, the sum's, rstd's and the division;
        # n: rstd's and one; then their product, the difference, rstd, the sum
        mean = (u * n).abs().mean(-1, keepdim=True)
        bound = half_step(dtype) * dx.abs() + U * (rstd * ((NORM + 4) * u.abs() + (DEPTH + 3 * NORM + 6) * n.abs() * mean))
        if ds is not None:
            bound = bound + U * (ds.double().abs() + dx.abs())
        close(got_dx, dx, bound * 1.001 + smallest(dtype))
        terms = (dy.double() * n).abs().sum(0)
        close(got_dw, dw, half_step(dtype) * dw.abs() + U * (rows + NORM + 1) * terms + smallest(dtype))

    y, stream = f2s.add_rms_norm(x, w, r, eps=eps)
    dx, dr, dw = torch.autograd.grad((y, stream), (x, r, w), (dy, ds))
    assert torch.equal(dx, dr)
    check(stream.detach(), dx, dw, ds)
    again = torch.autograd.grad(f2s.add_rms_norm(x, w, r, eps=eps), (x, w), (dy, ds))
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    y, stream = f2s.add_rms_norm(x, w, eps=eps)
    assert stream is x
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    check(x.detach(), dx, dw, None)
    if rows > 2:  # rows at a pitch, from gradients at another
        y, stream = f2s.add_rms_norm(padded(x.detach()).requires_grad_(), w, eps=eps)
        dw2, = torch.autograd.grad(y, w, padded(dy))
        check(x.detach(), dx, dw2, None)


@pytest.mark.gpu
def test_norm_gradients_that_are_not_asked_for(cuda):
    x, r = (normal(5, 64, seed=s).to(cuda).requires_grad_() for s in (1, 2))
    w = normal(64, seed=3).to(cuda).requires_grad_()
    y, stream = f2s.add_rms_norm(x, w, r)
    gx, gr, gw = torch.autograd.grad(stream.sum(), (x, r, w), allow_unused=True)
    assert torch.equal(gx, torch.ones_like(x)) and torch.equal(gr, gx)
    assert gw is None or not gw.any()
    y, _ = f2s.add_rms_norm(x.detach(), w, r.detach())
    gw, = torch.autograd.grad(y.sum(), w)
    y, _ = f2s.add_rms_norm(x, w.detach(), r.detach())
    gx, = torch.autograd.grad(y.sum(), x)
    y, _ = f2s.add_rms_norm(x, w, r)
    both = torch.autograd.grad(y.sum(), (x, w))
    assert torch.equal(gx, both[0]) and torch.equal(gw, both[1])
    x0 = torch.zeros(0, 64, device=cuda, requires_grad=True)
    y, stream = f2s.add_rms_norm(x0, w, x0)
    gx, gw = torch.autograd.grad(y.sum(), (x0, w))
    assert y.shape == gx.shape == (0, 64) and not gw.any()
    # a weight shared by two norms, a residual that is the input itself
    y, stream = f2s.add_rms_norm(x, w, x)
    y, _ = f2s.add_rms_norm(y, w, stream)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    s = x64 + x64
    n = lambda v: v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w64  # noqa: E731
    hx, hw = torch.autograd.grad(n(n(s) + s).sum(), (x64, w64))
    # two norms in a row, every entry of a gradient of order 1: a few hundred roundings
    close(gx, hx, 1e3 * U * hx.abs().max())
    close(gw, hw, 1e3 * U * hw.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_rows_without_a_norm(cuda, dtype):
    """A row of zeros: eps alone; rows past the last one with eps = 0; a value
    that is not finite stays in its row."""
    x = normal(9, 192, dtype=dtype, seed=1).to(cuda)
    x[3] = 0
    w = normal(192, dtype=dtype, seed=2).to(cuda)
    y, _ = f2s.add_rms_norm(x, w)
    assert not y[3].any() and torch.isfinite(y).all()
    eight, _ = f2s.add_rms_norm_int8(x, w)
    assert not eight.values[3].any() and eight.scale[3] == 0
    clean = eight
    x[3] = 1
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    y, _ = f2s.add_rms_norm(xg, wg, eps=0.0)
    gx, gw = torch.autograd.grad(y.float().sum(), (xg, wg))
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all()
    x[5, 17] = float("nan")
    x[7, 0] = float("inf")
    eight, _ = f2s.add_rms_norm_int8(x, w)
    keep = [0, 1, 2, 4, 6, 8]
    assert torch.isnan(eight.scale[[5, 7]]).all() and not eight.values[[5, 7]].any()
    assert torch.equal(eight.values[keep], clean.values[keep])
    assert torch.equal(eight.scale[keep], clean.scale[keep])
    y, _ = f2s.add_rms_norm(x, w)
    assert torch.isnan(y[5]).all() and torch.isfinite(y[keep]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [24, 192, 191, 1530, 4096, 16391])
def test_norm_of_rows_whose_squares_leave_fp32(cuda, width, dtype):
    """Rows of 1e25 and 1e-25 among ordinary ones, with eps = 0. Their values are
    multiplied by a power of two before they are squared, which rounds nothing,
    so the bounds are those of the ordinary rows."""
    x = normal(9, width, dtype=dtype, seed=width)
    x[[1, 8]] *= 1e25
    x[[2, 5]] *= 1e-25
    x = x.to(cuda).requires_grad_()
    w = normal(width, dtype=dtype, seed=1).to(cuda).requires_grad_()
    dy = normal(9, width, dtype=dtype, seed=2).to(cuda)
    _, s, w64, rstd = norm64(x.detach(), w.detach(), None, 0.0)
    y, _ = f2s.add_rms_norm(x, w, eps=0.0)
    y64 = s * rstd * w64
    close(y.detach(), y64, y64.abs() * (half_step(dtype) + NORM * U) * 1.001 + smallest(dtype))
    with torch.no_grad():
        eight, _ = f2s.add_rms_norm_int8(x, w, eps=0.0)
    p = s * w64
    assert torch.equal(eight.values, nearest_whole(p, row_max(p)))
    scale = (row_max(p) * rstd / 127)[:, 0]
    close(eight.scale, scale, scale * (NORM + 2) * U)
    got_dx, got_dw = torch.autograd.grad(y, (x, w), dy)
    dx, dw, (rstd, u, n) = norm_grad64(x.detach(), w.detach(), dy, None, 0.0)
    mean = (u * n).abs().mean(-1, keepdim=True)
    bound = half_step(dtype) * dx.abs() + U * (rstd * ((NORM + 4) * u.abs() + (DEPTH + 3 * NORM + 6) * n.abs() * mean))
    close(got_dx, dx, bound * 1.001 + smallest(dtype))
    terms = (dy.double() * n).abs().sum(0)
    close(got_dw, dw, half_step(dtype) * dw.abs() + U * (9 + NORM + 1) * terms + smallest(dtype))


# ---- 8-bit rows ----


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_quantize_rows(cuda, width, dtype):
    for rows, layout in ((1, None), (37, None), (5, padded), (6, shifted)):
        x = normal(rows, width, dtype=dtype, seed=width + rows).to(cuda)
        eight = f2s.quantize_rows(x if layout is None else layout(x))
        m = row_max(x.double())
        assert torch.equal(eight.values, nearest_whole(x.double(), m))
        assert torch.equal(eight.scale, row_scale(m)[:, 0])
        assert eight.values.stride(0) % 16 == 0
        for to in TYPES:
            want = (eight.values.float() * eight.scale[:, None]).to(to)
            assert torch.equal(eight.dequantize(to), want)
            assert torch.equal(Int8Rows(eight.values.contiguous(), eight.scale).dequantize(to), want)


@pytest.mark.gpu
def test_quantize_rows_at_borders(cuda):
    """Ties of 127 v / m, rows of the smallest and largest magnitudes, of
    zeros, and with values that are not finite."""
    ties = torch.arange(-254, 255, dtype=torch.float32)  # 127 v / 254: every odd v is a tie
    near = torch.nextafter(ties, torch.full_like(ties, 1e9))
    far = torch.nextafter(ties, torch.full_like(ties, -1e9))
    for dtype in TYPES:
        rows = [ties, near.clamp(max=254), far.clamp(min=-254)]
        rows += [ties * 2.0**-10, ties * 2.0**7]
        x = torch.stack(rows).to(dtype).to(cuda)
        if dtype == torch.float32:
            x = torch.cat([x, x * 2.0**-120, x * 2.0**-150, x[:1] * 2.0**112, x[:1] * 0])
        eight = f2s.quantize_rows(x)
        m = row_max(x.double())
        assert torch.equal(eight.values, nearest_whole(x.double(), m))
        assert torch.equal(eight.scale, row_scale(m)[:, 0])
    assert (eight.values[0].float() == (ties / 2).round().to(cuda)).all()  # half to even
    x = normal(4, 100, seed=1).to(cuda)
    want = f2s.quantize_rows(x)
    x[1, 99] = float("-inf")
    x[2, 0] = float("nan")
    eight = f2s.quantize_rows(x)
    assert torch.isnan(eight.scale[1:3]).all() and not eight.values[1:3].any()
    assert torch.equal(eight.values[[0, 3]], want.values[[0, 3]])
    assert torch.isnan(eight.dequantize()[1:3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value_against_many_maxima(cuda, dtype):
    """All positive values of the binades in which 127 v / m is between 1/4 and
    127, for maxima of every kind of significand: exact halves are common here."""
    bits = 7 if dtype == torch.bfloat16 else 10
    significands = torch.arange(2**bits, 2 ** (bits + 1), dtype=torch.float64)
    values = torch.cat([significands * 2.0**e for e in range(-10, 1)]) * 2.0**-bits  # below 2
    step = 1 if dtype == torch.bfloat16 else 5
    maxima = significands[::step] * 2.0**-bits
    x = torch.where(values <= maxima[:, None], values, 0.0)
    x = torch.cat([maxima[:, None], x, -x], 1).to(dtype).to(cuda)
    want = nearest_whole(x.double(), row_max(x.double()))
    assert torch.equal(f2s.quantize_rows(x).values, want)
    # as a norm's products, and as a checkpoint group's values
    one = torch.ones(x.shape[1], dtype=dtype, device=cuda)
    assert torch.equal(f2s.add_rms_norm_int8(x, one)[0].values, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_int8_of_products_at_halves(cuda, dtype):
    """Streams and weights of few bits, whose products make 127 p / m an exact
    half often; each row's largest product is another."""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-255, 256, (400, 2048), generator=g).to(dtype).to(cuda)
    w = torch.randint(1, 256, (2048,), generator=g).to(dtype).to(cuda)
    p = x.double() * w.double()
    twice = 254 * p / row_max(p)
    assert ((twice == twice.round()) & (twice.remainder(2) == 1)).sum() > 100  # halves are there
    assert torch.equal(f2s.add_rms_norm_int8(x, w)[0].values, nearest_whole(p, row_max(p)))


@pytest.mark.gpu
def test_shapes_without_rows_and_of_any_rank(cuda):
    x = normal(2, 3, 5, 40, seed=1).to(cuda)
    eight = f2s.quantize_rows(x)
    assert eight.values.shape == x.shape and eight.scale.shape == (2, 3, 5)
    flat = f2s.quantize_rows(x.view(30, 40))
    assert torch.equal(eight.values.reshape(30, 40), flat.values)
    weight = f2s.quantize_rows(normal(24, 40, seed=2).to(cuda))
    y = f2s.linear_int8(eight, weight, dtype=torch.float32)
    assert torch.equal(y.view(30, 24), f2s.linear_int8(flat, weight, dtype=torch.float32))
    one = f2s.quantize_rows(x[0, 0, 0])
    assert one.scale.shape == () and f2s.linear_int8(one, weight, dtype=torch.float32).shape == (24,)
    assert torch.equal(f2s.linear_int8(one, weight, dtype=torch.float32), y[0, 0, 0])
    swapped = x.transpose(1, 2)  # no one pitch: copied
    assert torch.equal(f2s.quantize_rows(swapped).values, eight.values.transpose(1, 2))
    wide = x[..., :16]  # one pitch over all leading dimensions
    assert torch.equal(f2s.quantize_rows(wide).values, f2s.quantize_rows(wide.contiguous()).values)
    spread = x[0, 0, :1].expand(4, 40)
    assert torch.equal(f2s.quantize_rows(spread).values, eight.values[0, 0, :1].expand(4, 40))
    none = x[:0]
    eight = f2s.quantize_rows(none)
    assert eight.values.shape == (0, 3, 5, 40) and eight.dequantize().shape == (0, 3, 5, 40)
    assert f2s.linear_int8(eight, weight).shape == (0, 3, 5, 24)
    assert f2s.swiglu(none).shape == (0, 3, 5, 20) and f2s.swiglu_int8(none).scale.shape == (0, 3, 5)
    assert f2s.add_rms_norm_int8(none, x[0, 0, 0])[0].values.shape == (0, 3, 5, 40)
    p = none.clone().requires_grad_()
    for kept in (None, "int8"):
        assert torch.autograd.grad(f2s.swiglu(p, checkpoint=kept).sum(), p)[0].shape == none.shape


@pytest.mark.gpu
def test_eight_bit_calls_refuse_gradients(cuda):
    x = torch.zeros(4, 16, device=cuda, requires_grad=True)
    w = torch.ones(16, device=cuda)
    for call in (lambda: f2s.quantize_rows(x), lambda: f2s.add_rms_norm_int8(x, w),
                 lambda: f2s.swiglu_int8(x)):
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    eight = f2s.quantize_rows(x.detach())
    bias = torch.zeros(4, device=cuda, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        f2s.linear_int8(eight, eight, bias, dtype=torch.float32)
    with pytest.raises(ValueError, match="bias must be"):
        f2s.linear_int8(eight, eight, torch.zeros(3, device=cuda), dtype=torch.float32)
    with pytest.raises(ValueError, match="channels"):
        f2s.linear_int8(eight, f2s.quantize_rows(torch.zeros(4, 8, device=cuda)))
    with pytest.raises(ValueError, match="at most 32768"):
        f2s.quantize_rows(torch.zeros(1, 32769, device=cuda))


@pytest.mark.gpu
def test_scales_that_want_a_gradient_are_refused(cuda):
    eight = f2s.quantize_rows(normal(4, 16, seed=1).to(cuda))
    learnt = Int8Rows(eight.values, eight.scale.clone().requires_grad_())
    for call in (lambda: learnt.dequantize(), lambda: f2s.linear_int8(learnt, eight),
                 lambda: f2s.linear_int8(eight, learnt)):
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad():
            call()


# ---- the product ----


def eighths(rows, K, seed, device):
    g = torch.Generator().manual_seed(seed)
    values = torch.randint(-128, 128, (rows, K), generator=g, dtype=torch.int8)
    pitch = -(-K // 16) * 16
    held = torch.full((rows, pitch), 99, dtype=torch.int8)  # not part of any row
    held[:, :K] = values
    return Int8Rows(held.to(device)[:, :K], (0.5 + torch.rand(rows, generator=g)).to(device))


def check_product(x, w, bias, dtype, y):
    total = x.values.double() @ w.values.double().T
    product = total * x.scale.double()[..., None] * w.scale.double()
    want = product if bias is None else product + bias.double()
    # a value half a step or more past the type's largest rounds to infinity
    # (none of these lies within the fp32 roundings of that point)
    largest = torch.finfo(dtype).max * (1 + half_step(dtype) / 2)
    beyond = want.abs() > largest
    assert torch.equal(y.double()[beyond], want[beyond].sign() * float("inf"))
    y, want, product = (t[~beyond] for t in (y, want, product))
    # the integer to fp32, times the token's scale; times the channel's with the bias in one
    close(y, want, half_step(dtype) * want.abs() * 1.001 + U * (2.01 * product.abs() + 1.01 * want.abs()) + smallest(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [1, 15, 16, 33, 128, 129, 192, 1000, 2049, 4096])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 1000), (2, 129), (3, 64), (4, 515), (5, 7), (8, 1024), (16, 96), (17, 200),
                                       (33, 129), (64, 1), (65, 257), (100, 4096), (129, 100), (300, 192), (1000, 771)])
def test_linear_int8(cuda, rows, cols, K, dtype):
    x, w = eighths(rows, K, rows + K, cuda), eighths(cols, K, cols + K + 1, cuda)
    bias = normal(cols, dtype=dtype, seed=cols, scale=100 * K**0.5).to(cuda)
    for b in (bias, None):
        check_product(x, w, b, dtype, f2s.linear_int8(x, w, b, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,K", [(5, 100, 77), (300, 200, 200), (3, 64, 33), (70, 40, 1000)])
def test_linear_int8_of_any_pitch(cuda, rows, cols, K):
    x, w = eighths(rows, K, 1, cuda), eighths(cols, K, 2, cuda)
    want = f2s.linear_int8(x, w, dtype=torch.float32)
    check_product(x, w, None, torch.float32, want)
    for a, b in ((x.values.contiguous(), w.values), (x.values, padded(w.values, 5)),
                 (shifted(x.values), shifted(w.values)), (padded(x.values, 16), padded(w.values, 32))):
        got = f2s.linear_int8(Int8Rows(a, x.scale), Int8Rows(b, w.scale), dtype=torch.float32)
        assert torch.equal(got, want)
    strided = torch.stack([x.scale, x.scale], 1)[:, 0]
    assert torch.equal(f2s.linear_int8(Int8Rows(x.values, strided), w, dtype=torch.float32), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 6, 20, 150])
def test_linear_int8_largest_sums(cuda, rows):
    """Sums next to the ends of 32 bits: K 131,071 of -128 x -128 and -128 x 127."""
    K = 131071
    x = torch.full((rows, K + 1), -128, dtype=torch.int8, device=cuda)[:, :K]
    w = torch.full((40, K + 1), -128, dtype=torch.int8, device=cuda)[:, :K]
    w[1::2] = 127
    one = torch.ones(40, device=cuda)
    y = f2s.linear_int8(Int8Rows(x, one[:1].expand(rows)), Int8Rows(w, one), dtype=torch.float32)
    assert (y[:, 0::2] == float(2**14 * K)).all() and (y[:, 1::2] == float(-128 * 127 * K)).all()
    with pytest.raises(ValueError, match="exact 32-bit sum"):
        f2s.linear_int8(Int8Rows(torch.zeros(1, K + 1, dtype=torch.int8, device=cuda), one[:1]),
                        Int8Rows(torch.zeros(4, K + 1, dtype=torch.int8, device=cuda), one[:4]))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,K", [(1, 4096, 4096), (40, 2048, 8192), (20000, 192, 1536), (20001, 1536, 192), (4096, 4000, 2000)])
def test_linear_int8_large(cuda, rows, cols, K):
    x, w = eighths(rows, K, 1, cuda), eighths(cols, K, 2, cuda)
    bias = normal(cols, dtype=torch.bfloat16, seed=3, scale=1e3).to(cuda)
    check_product(x, w, bias, torch.bfloat16, f2s.linear_int8(x, w, bias))
    _lib.check_device_error()


@pytest.mark.gpu
def test_linear_int8_forms_at_once(cuda):
    """Products of every form on their own streams, 20 of each in flight."""
    shapes = [(2, 512, 1024), (24, 1024, 4096), (60, 300, 2048), (3000, 1024, 1024), (2000, 192, 700)]
    operands = [(eighths(r, K, i, cuda), eighths(c, K, i + 10, cuda)) for i, (r, c, K) in enumerate(shapes)]
    want = [f2s.linear_int8(x, w) for x, w in operands]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in shapes]
    got = [[] for _ in shapes]
    for _ in range(20):
        for i, (x, w) in enumerate(operands):
            with torch.cuda.stream(streams[i]):
                got[i].append(f2s.linear_int8(x, w))
    torch.cuda.synchronize()
    _lib.check_device_error()
    for w, ys in zip(want, got):
        assert all(torch.equal(y, w) for y in ys)


@pytest.mark.gpu
def test_linear_int8_scales_that_are_not_finite(cuda):
    x, w = eighths(40, 64, 1, cuda), eighths(50, 64, 2, cuda)
    want = f2s.linear_int8(x, w, dtype=torch.float32)
    x.scale[3] = float("nan")
    w.scale[5] = 0.0
    y = f2s.linear_int8(x, w, dtype=torch.float32)
    assert torch.isnan(y[3]).all() and not y[:3, 5].any()
    keep = [i for i in range(50) if i != 5]
    assert torch.equal(y[4:][:, keep], want[4:][:, keep])


# ---- SwiGLU ----


def sigmoid_off(g):
    """Relative error of sigma(g): the exponential's 2^-22 and its rounded
    argument (two roundings of |g| log2 e), both scaled by 1 - sigma in the sum,
    and a reciprocal of 2^-23."""
    return (1 - torch.sigmoid(g)) * (2.0**-22 + 3 * U * g.abs()) + 2.0**-23 + 2 * U


def swiglu_grad_bound(gate, value, dy):
    """The fp32 roundings of swiglu_grad64. dg is d sigma v times the factor
    1 + g (1 - sigma), which cancels near g = -1.28: its own error is absolute
    (|g| times that of 1 - sigma, and the sum's), whatever v multiplies it by."""
    gate, value, dy = gate.double(), value.double(), dy.double()
    sigma, off = torch.sigmoid(gate), sigmoid_off(gate)
    front = (dy * sigma * value).abs()
    factor = (1 + gate * (1 - sigma)).abs()
    dgate = front * (factor * (off + 3 * U) + gate.abs() * (sigma * off + U) + U * (1 + gate.abs()))
    return torch.cat([dgate, (dy * sigma * gate).abs() * (off + 2 * U)], -1)


def kept64(v):
    """What the 8-bit checkpoint of (rows, H) values stands for, in fp32."""
    rows, hidden = v.shape
    groups = -(-hidden // 128)
    held = torch.zeros(rows, groups * 128, dtype=torch.float64, device=v.device)
    held[:, :hidden] = v.double()
    held = held.view(rows, groups, 128)
    m = row_max(held)
    got = nearest_whole(held, m).float() * row_scale(m)
    return got.view(rows, -1)[:, :hidden]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (5, 8), (2, 128), (33, 129), (9, 200), (4, 256), (17, 1000),
                                         (3, 1371), (2, 6144), (300, 64)])
def test_swiglu(cuda, rows, hidden, dtype):
    p = normal(rows, 2 * hidden, dtype=dtype, seed=rows + hidden, scale=2).to(cuda)
    p[0, 0], p[-1, hidden - 1] = -100, 90
    dy = normal(rows, hidden, dtype=dtype, seed=5).to(cuda)
    g, v = p[:, :hidden].double(), p[:, hidden:].double()
    y64 = g * torch.sigmoid(g) * v
    for layout in (None, padded, shifted):
        q = (p if layout is None else layout(p)).detach().requires_grad_()
        d = dy if layout is None else layout(dy)
        for checkpoint in (None, "int8"):
            y = f2s.swiglu(q, checkpoint=checkpoint)
            close(y, y64, y64.abs() * (half_step(dtype) + sigmoid_off(g) + 2 * U) * 1.001 + smallest(dtype) + 1e-35)
            with torch.no_grad():
                assert torch.equal(f2s.swiglu(q), y)
            got, = torch.autograd.grad(y, q, d)
            kg, kv = (g, v) if checkpoint is None else (kept64(p[:, :hidden]).double(), kept64(p[:, hidden:]).double())
            want = swiglu_grad64(kg, kv, dy)
            close(got, want, swiglu_grad_bound(kg, kv, dy) + half_step(dtype) * want.abs() * 1.001 + smallest(dtype) + 1e-35)


@pytest.mark.gpu
def test_swiglu_checkpoint_groups(cuda):
    """Each group of 128 channels of gate and value has its own scale: zeros,
    a value that is not finite and a much larger group stay in theirs."""
    p = normal(4, 2 * 300, seed=1).to(cuda)
    p[0, :128] = 0
    p[1, 130] = float("nan")
    p[2, 300:428] *= 1e6
    p[3, 599] = float("inf")
    q = p.clone().requires_grad_()
    got, = torch.autograd.grad(f2s.swiglu(q, checkpoint="int8").sum(), q, retain_graph=False)
    kept = kept64(p[:, :300]), kept64(p[:, 300:])
    ones = torch.ones(4, 300, device=cuda)
    want = swiglu_grad64(*kept, ones)
    bad = torch.zeros(4, 600, dtype=torch.bool, device=cuda)
    bad[1, 128:256] = bad[1, 428:556] = True   # the gate's group, and the value's gradient there
    bad[3, 256:300] = True                     # the gate's gradient where the value is not finite
    assert torch.isnan(got[bad]).all()
    fine = ~bad
    assert torch.isfinite(got[fine]).all()
    bound = swiglu_grad_bound(*kept, ones) + half_step(torch.float32) * want.abs() * 1.001 + 1e-35
    close(got[fine], want[fine], bound[fine])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hidden", [1, 7, 8, 64, 200, 1000, 1371, 6144, 16391, 32768])
def test_swiglu_int8(cuda, hidden, dtype):
    for rows, layout in ((1, None), (19, None), (5, padded), (3, shifted)):
        p = normal(rows, 2 * hidden, dtype=dtype, seed=rows + hidden, scale=2).to(cuda)
        eight = f2s.swiglu_int8(p if layout is None else layout(p))
        g, v = p[:, :hidden].double(), p[:, hidden:].double()
        h = g * torch.sigmoid(g) * v
        m = row_max(h)
        off = (sigmoid_off(g) + 2 * U).amax(-1, keepdim=True)
        # the quotient of two values each off by that: beyond half only next to a border
        quotient = 127 * h / m
        assert ((eight.values.double() - quotient).abs() <= 0.5 + 127 * 2.01 * off).all()
        close(eight.scale, (m / 127)[:, 0], (m / 127 * (off + U) * 1.001)[:, 0])
    p = normal(3, 2 * hidden, dtype=dtype, seed=1).to(cuda)
    p[1] = 0
    p[2, hidden] = float("nan")
    eight = f2s.swiglu_int8(p)
    assert eight.scale[1] == 0 and torch.isnan(eight.scale[2]) and not eight.values[1:].any()


# ---- together, and where they run ----


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 7, 200])
def test_served_feed_forward(cuda, tokens):
    """norm -> product -> SwiGLU -> product in 8 bits, each stage against 64
    bits on the rows that it was given."""
    C, H = 192, 520
    x, r = (normal(tokens, C, dtype=torch.bfloat16, seed=s).to(cuda) for s in (1, 2))
    w = normal(C, dtype=torch.bfloat16, seed=3).to(cuda)
    w1 = f2s.quantize_rows(normal(2 * H, C, seed=4, scale=C**-0.5).to(cuda))
    w2 = f2s.quantize_rows(normal(C, H, seed=5, scale=H**-0.5).to(cuda))
    b1, b2 = (normal(n, dtype=torch.bfloat16, seed=n).to(cuda) for n in (2 * H, C))
    rows, stream = f2s.add_rms_norm_int8(x, w, r)
    projected = f2s.linear_int8(rows, w1, b1)
    hidden = f2s.swiglu_int8(projected)
    out = f2s.linear_int8(hidden, w2, b2)
    check_product(rows, w1, b1, torch.bfloat16, projected)
    check_product(hidden, w2, b2, torch.bfloat16, out)
    # and the whole against the same layer without the 8-bit roundings: each is
    # off by a uniform half step of m / 127, which is at most m / (127 sqrt 12)
    # of root mean square; with m below 6 sigma (gaussian rows of 192 to 520)
    # that is 1.4% for rows and weights, and 2.5% for the heavier-tailed h
    _, s, w64, rstd = norm64(x, w, r, 1e-6)
    p = (s * rstd * w64) @ w1.dequantize().double().T + b1.double()
    h = p[:, :H] * torch.sigmoid(p[:, :H]) * p[:, H:]
    want = h @ w2.dequantize().double().T + b2.double()
    assert (out.double() - want).norm() / want.norm() < 0.06


@pytest.mark.gpu
def test_trained_feed_forward(cuda):
    """A training step's gradients through norm, projections and SwiGLU with
    checkpoints, against 64 bits with the same kept values."""
    T, C, H = 150, 96, 200
    make = lambda *s, seed, scale=1.0: normal(*s, seed=seed, scale=scale).to(cuda).requires_grad_()  # noqa: E731
    x, r, w = make(T, C, seed=1), make(T, C, seed=2), make(C, seed=3)
    w1, w2 = make(2 * H, C, seed=4, scale=C**-0.5), make(C, H, seed=5, scale=H**-0.5)
    y, stream = f2s.add_rms_norm(x, w, r)
    projected = y @ w1.T
    out = stream + f2s.swiglu(projected, checkpoint="int8") @ w2.T
    d = normal(T, C, seed=6).to(cuda)
    got = torch.autograd.grad(out, (x, r, w, w1, w2), d)
    wide = [t.detach().double().requires_grad_() for t in (x, r, w, w1, w2)]
    x6, r6, w6, a6, b6 = wide
    s6 = (x6.float() + r6.float()).double()
    y6 = s6 * (s6.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w6
    p6 = y6 @ a6.T
    kept = torch.cat([kept64(projected.detach()[:, :H]), kept64(projected.detach()[:, H:])], 1).double()
    g6, v6 = p6[:, :H], p6[:, H:]
    h6 = g6 * torch.sigmoid(g6) * v6
    # h's value, and the kept values' slope
    slope = swiglu_grad64(kept[:, :H], kept[:, H:], torch.ones(T, H, device=cuda))
    h6 = h6.detach() + (slope[:, :H] * (g6 - g6.detach())) + slope[:, H:] * (v6 - v6.detach())
    want = torch.autograd.grad(s6 + h6 @ b6.T, wide, d.double())
    # sums of up to 400 fp32 terms at three places: 1e3 roundings of the norm
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 1e3 * U * b.norm()


@pytest.mark.gpu
def test_layer_captured_and_replayed(cuda):
    C, H, T = 128, 256, 24
    w = normal(C, dtype=torch.bfloat16, seed=3).to(cuda)
    w1 = f2s.quantize_rows(normal(2 * H, C, seed=4).to(cuda))
    w2 = f2s.quantize_rows(normal(C, H, seed=5).to(cuda))
    x, r = (normal(T, C, dtype=torch.bfloat16, seed=s).to(cuda) for s in (1, 2))

    def layer(x, r):
        rows, stream = f2s.add_rms_norm_int8(x, w, r)
        return f2s.linear_int8(f2s.swiglu_int8(f2s.linear_int8(rows, w1)), w2), stream

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = layer(x, r)
    torch.cuda.current_stream().wait_stream(side)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        got1 = layer(x, r)
    with torch.cuda.graph(second):
        got2 = layer(r, x)
    for seed in (10, 20):
        x.copy_(normal(T, C, dtype=torch.bfloat16, seed=seed))
        r.copy_(normal(T, C, dtype=torch.bfloat16, seed=seed + 1))
        first.replay()
        second.replay()
        first.replay()
        want = layer(x, r)
        assert all(torch.equal(a, b) for a, b in zip(got1, want))
        assert all(torch.equal(a, b) for a, b in zip(got2, layer(r, x)))


@pytest.mark.gpu
def test_training_captured_and_replayed(cuda):
    x, r = (normal(50, 192, seed=s).to(cuda).requires_grad_() for s in (1, 2))
    w = normal(192, seed=3).to(cuda).requires_grad_()

    def step():
        y, stream = f2s.add_rms_norm(x, w, r)
        h = f2s.swiglu(y, checkpoint="int8")
        return torch.autograd.grad(h.sum() + stream.square().sum(), (x, r, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.copy_(normal(50, 192, seed=7))
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_capture_beside_a_live_eager_graph(cuda):
    """A backward captured while an eager graph of the same leaves is alive cannot
    be captured (its leaves belong to the eager stream): an error in Python, in a
    process that lives on."""
    code = """
import sys, torch
sys.path.insert(0, "jittor-flow2surf_b200")
import flow2surf_b200 as f2s
x = torch.randn(8, 64, device="cuda", requires_grad=True)
w = torch.ones(64, device="cuda", requires_grad=True)
step = lambda: torch.autograd.grad(f2s.swiglu(f2s.add_rms_norm(x, w)[0], checkpoint="int8").sum(), (x, w))
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    step()
torch.cuda.current_stream().wait_stream(side)
alive = f2s.add_rms_norm(x, w)
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph):
        step()
    print("captured")
except RuntimeError as error:
    print("raised")
print("lives on")
"""
    root = Path(__file__).resolve().parent.parent
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and done.stdout.split()[-2:] == ["lives", "on"], done.stderr[-2000:]


@pytest.mark.gpu
def test_second_derivatives_are_refused(cuda):
    x = normal(4, 64, seed=1).to(cuda).requires_grad_()
    w = normal(64, seed=2).to(cuda).requires_grad_()
    for out in (f2s.add_rms_norm(x, w)[0], f2s.swiglu(x), f2s.swiglu(x, checkpoint="int8")):
        gx, = torch.autograd.grad(out.sum(), x, create_graph=True)  # a first one is given
        with pytest.raises(RuntimeError):  # x is not reached by it
            torch.autograd.grad(gx.sum(), x, retain_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            gx.sum().backward()


@pytest.mark.gpu
def test_kept_values_that_were_changed_are_refused(cuda):
    """What a backward reads may not have been written since (its stream, here)."""
    x, r = (normal(4, 64, seed=s).to(cuda).requires_grad_() for s in (1, 2))
    w = normal(64, seed=3).to(cuda).requires_grad_()
    y, stream = f2s.add_rms_norm(x, w, r)
    with torch.no_grad():
        stream.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)


@pytest.mark.gpu
def test_layer_on_two_streams_at_once(cuda):
    w1 = f2s.quantize_rows(normal(512, 256, seed=4).to(cuda))
    xs = [normal(600, 256, seed=s).to(cuda) for s in (1, 2)]
    layer = lambda x: f2s.swiglu_int8(f2s.linear_int8(f2s.quantize_rows(x), w1))  # noqa: E731
    want = [layer(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(layer(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y.values, want[i].values) and torch.equal(y.scale, want[i].scale)


@pytest.mark.gpu
def test_nothing_is_written_beside_the_rows(cuda):
    """Through the C entries: buffers keep what lies between the rows' ends and
    the pitch, and behind the last row."""
    rows, C, N, pitch = 5, 40, 24, 64
    x = normal(rows, C, dtype=torch.bfloat16, seed=1).to(cuda)
    w = torch.ones(C, dtype=torch.bfloat16, device=cuda)
    q = torch.full((rows + 3, pitch), 55, dtype=torch.int8, device=cuda)
    scale = torch.full((rows + 3,), 55.0, device=cuda)
    st = _lib.stream_handle()

    def untouched():
        assert (q[rows:] == 55).all() and (q[:, C:] == 55).all() and (scale[rows:] == 55).all()
        q.fill_(55)
        scale.fill_(55)

    for _ in range(2):
        _lib.call("f2s_quantize_rows", x.data_ptr(), C, 1, rows, C, q.data_ptr(), pitch, scale.data_ptr(), st)
        weight = Int8Rows(q[:rows, :C].clone(), scale[:rows].clone())
        untouched()
        _lib.call("f2s_add_rms_norm_int8", x.data_ptr(), C, None, 0, w.data_ptr(), 1, rows, C, 1e-6, None,
                  q.data_ptr(), pitch, scale.data_ptr(), st)
        untouched()
        p = torch.cat([x, x], 1)
        _lib.call("f2s_swiglu_int8", p.data_ptr(), 2 * C, 1, rows, C, q.data_ptr(), pitch, scale.data_ptr(), st)
        untouched()
        y = torch.full((rows + 3, pitch), 55.0, dtype=torch.bfloat16, device=cuda)
        _lib.call("f2s_dequantize_rows", weight.values.data_ptr(), C, weight.scale.data_ptr(), rows, C, y.data_ptr(),
                  pitch, 1, st)
        assert (y[rows:] == 55).all() and (y[:, C:] == 55).all()
    for n, K, m in ((24, 48, 5), (24, 48, 200), (23, 48, 40), (130, 48, 300)):
        a, b = eighths(m, K, 1, cuda), eighths(n, K, 2, cuda)
        want = f2s.linear_int8(a, b, dtype=torch.float32)
        for ldy in (n + 8, n + 9):
            y = torch.full((m + 3, ldy), 55.0, device=cuda)
            _lib.call("f2s_linear_int8", a.values.data_ptr(), K, a.scale.data_ptr(), b.values.data_ptr(), K,
                      b.scale.data_ptr(), None, y.data_ptr(), ldy, 0, m, n, K, st)
            assert torch.equal(y[:m, :n], want) and (y[m:] == 55).all() and (y[:, n:] == 55).all()


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """Rows that lie more than 2^31 elements apart."""
    C, pitch = 96, 2**30 + 16
    held = torch.empty(2 * pitch + C, dtype=torch.bfloat16, device=cuda)
    x = torch.as_strided(held, (3, C), (pitch, 1))
    x.copy_(normal(3, C, dtype=torch.bfloat16, seed=1))
    near = x.contiguous()
    w = normal(C, dtype=torch.bfloat16, seed=2).to(cuda)
    assert torch.equal(f2s.quantize_rows(x).values, f2s.quantize_rows(near).values)
    assert torch.equal(f2s.add_rms_norm(x, w, x)[0], f2s.add_rms_norm(near, w, near)[0])
    assert torch.equal(f2s.swiglu(x), f2s.swiglu(near))
    assert torch.equal(f2s.swiglu_int8(x).values, f2s.swiglu_int8(near).values)
    del held, x
    held = torch.empty(2 * (pitch + pitch) + C, dtype=torch.int8, device=cuda)
    x8 = torch.as_strided(held, (3, C), (2 * pitch, 1))
    eight = f2s.quantize_rows(near)
    x8.copy_(eight.values)
    wide, close_by = Int8Rows(x8, eight.scale), Int8Rows(eight.values, eight.scale)
    weight = eighths(64, C, 3, cuda)
    assert torch.equal(wide.dequantize(), close_by.dequantize())
    assert torch.equal(f2s.linear_int8(wide, weight), f2s.linear_int8(close_by, weight))
    assert torch.equal(f2s.linear_int8(weight, wide), f2s.linear_int8(weight, close_by))
