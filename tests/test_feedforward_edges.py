"""The 8-bit feed-forward operators at the ends of their ranges, and calls that
their documentation allows but ordinary tests do not make.

References, helpers and the way tolerances are counted are those of
test_feedforward.py; 8-bit values have to be the nearest whole numbers of the
exact quotient.
"""

import threading

import pytest
import torch
from torch.autograd import forward_ad

import flow2surf_b200 as f2s
from flow2surf_b200.feedforward import Int8Rows
from test_feedforward import (DEPTH, NORM, TYPES, U, WIDTHS, close, eighths, half_step, nearest_whole, norm64,
                              norm_grad64, normal, row_max, smallest)

# fp32 streams and weights s, w of 24 bits with 254 s1 w1 - c s0 w0 = r for c odd:
# 127 p / m is r / (2 m) off the half c / 2, less than 64-bit products tell (they
# have 56 bits). (s0, w0, s1, w1, c, r), s0 w0 the larger product.
NEXT_TO_HALVES = [
    (16374893, 16219904, 15165803, 16203002, 235, 4),
    (16101769, 16130341, 14068111, 16499603, 227, -1),
    (16679204, 16069049, 14716702, 14698572, 205, -4),
    (16637806, 15750364, 16438509, 13242591, 211, 2),
    (16301801, 16312208, 16179395, 16112083, 249, -2),
    (16719859, 16164048, 15467849, 16440575, 239, 2),
    (16646973, 15920774, 13441091, 16535252, 213, 2),
    (16442797, 16735767, 16560288, 15243182, 233, -3),
    (16373941, 16552341, 15664237, 14373156, 211, -3),
    (16622725, 16199528, 16492751, 15362987, 239, -2),
    (15860984, 15875619, 15848809, 13448347, 215, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, -20, -90, 38])
@pytest.mark.parametrize("width", [2, 8, 200, 5000])
def test_norm_int8_of_products_next_to_halves(cuda, width, shift):
    """The exact quotient decides, whatever power of two the products carry."""
    for s0, w0, s1, w1, c, r in NEXT_TO_HALVES:
        assert 254 * s1 * w1 - c * s0 * w0 == r and c % 2 and 0 < s1 * w1 <= s0 * w0
        x, w = torch.zeros(3, width), torch.ones(width)
        x[1, :2] = torch.tensor([s0, s1]) * 2.0**shift
        x[2, :2] = torch.tensor([s0, -s1]) * 2.0**shift
        w[:2] = torch.tensor([w0, w1]) * 2.0**shift
        values = f2s.add_rms_norm_int8(x.to(cuda), w.to(cuda))[0].values
        q = (c + 1) // 2 if r > 0 else c // 2
        assert values[1:, :2].tolist() == [[127, q], [127, -q]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [24, 192, 191, 1530, 4096, 16391])
@pytest.mark.parametrize("loud", [1e15, 1e30, 8.0, 1e-10, 1e-20, 1e-33])
def test_norm_int8_of_products_that_leave_fp32(cuda, loud, width, dtype):
    """Finite rows whose products s w lie beyond fp32 at either end, among ordinary
    ones: each keeps its exact rounding, and a scale of its own."""
    sizes = torch.tensor([1.0, 3e37, 1e-25, 1e25, 1e-30, 1.0, 1e10, 1e-37, 1e20])
    x = normal(9, width, seed=width).clamp(-5, 5) * sizes[:, None]
    x[5] = 0
    x = x.to(dtype).to(cuda)
    w = normal(width, dtype=dtype, seed=1, scale=loud).to(cuda)
    rows = [0, 1, 2, 3, 4, 6, 7, 8]
    for eps in (0.0, 1e-6):
        for r in (None, torch.zeros_like(x)):
            _, s, w64, rstd = norm64(x, w, r, eps)
            p = s * w64
            eight, _ = f2s.add_rms_norm_int8(x, w, r, eps=eps)
            assert torch.equal(eight.values, nearest_whole(p, row_max(p)))
            scale = (row_max(p) * rstd / 127)[:, 0]
            close(eight.scale[rows], scale[rows], scale[rows] * (NORM + 2) * U + 1e-45)
            assert eps == 0 or eight.scale[5] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_int8_of_halves_below_the_smallest_normal(cuda, dtype):
    """Products of few bits that all lie below 2^-141, where exact halves are common."""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-255, 256, (60, 2048), generator=g).to(dtype) * 2.0**-82
    w = torch.randint(1, 256, (2048,), generator=g).to(dtype) * 2.0**-70
    p = x.double() * w.double()
    twice = 254 * p / row_max(p)
    assert ((twice == twice.round()) & (twice.remainder(2) == 1)).sum() > 10  # halves are there
    values = f2s.add_rms_norm_int8(x.to(cuda), w.to(cuda))[0].values
    assert torch.equal(values.cpu(), nearest_whole(p, row_max(p)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [24, 192, 4096])
def test_norm_int8_of_rows_that_are_not_finite_beside_large_products(cuda, width, dtype):
    x = normal(8, width, dtype=dtype, seed=1).to(cuda)
    x[1] *= 1e25
    x[2, 3], x[3, 0], x[4] = float("nan"), float("inf"), 0.0
    w = normal(width, dtype=dtype, seed=2, scale=1e15).to(cuda)
    w[0] = 0  # an infinite value times it is none
    eight, _ = f2s.add_rms_norm_int8(x, w)
    assert torch.isnan(eight.scale[2:4]).all() and not eight.values[2:5].any() and eight.scale[4] == 0
    keep = [0, 1, 5, 6, 7]
    p = x[keep].double() * w.double()
    assert torch.equal(eight.values[keep], nearest_whole(p, row_max(p))) and torch.isfinite(eight.scale[keep]).all()
    x[2, 3] = x[3, 0] = 0
    none, _ = f2s.add_rms_norm_int8(x, torch.zeros_like(w))
    assert not none.values.any() and not none.scale.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [24, 192, 191, 1530, 4096, 16391])
@pytest.mark.parametrize("sizes", [(1e-40, 1e-39, 1e-41), (3e-40, 1e-39, 2e-39)])
def test_norm_of_rows_whose_reciprocal_leaves_fp32(cuda, sizes, width, dtype):
    """Subnormal rows with eps 0: their reciprocal root is past 3.4e38, the normed
    rows and the weight's gradient are of order 1. A row that is 0 in bf16 (its
    smallest value is 9e-41) has none of them: 0 / 0."""

    def close_or_none(got, want, bound):
        none = torch.isnan(want)
        assert torch.equal(torch.isnan(got), none)
        close(got[~none], want[~none], bound[~none])

    x = normal(9, width, dtype=dtype, seed=width)
    x[[1, 4, 5]] = (x[[1, 4, 5]] * torch.tensor(sizes)[:, None]).to(dtype)
    x = x.to(cuda).requires_grad_()
    w = normal(width, dtype=dtype, seed=1).to(cuda).requires_grad_()
    dy = normal(9, width, dtype=dtype, seed=2).to(cuda)
    dy[[1, 4, 5]] *= 1e-9  # so that dx is finite
    _, s, w64, rstd = norm64(x.detach(), w.detach(), None, 0.0)
    assert (rstd > 3.5e38).sum() >= 1
    y, _ = f2s.add_rms_norm(x, w, eps=0.0)
    y64 = s * rstd * w64
    close_or_none(y.detach(), y64, y64.abs() * (half_step(dtype) + NORM * U) * 1.001 + smallest(dtype))
    with torch.no_grad():
        eight, _ = f2s.add_rms_norm_int8(x, w, eps=0.0)
    p = s * w64
    assert torch.equal(eight.values, nearest_whole(p, row_max(p)))
    scale = (row_max(p) * rstd / 127)[:, 0]
    close_or_none(eight.scale, scale, scale * (NORM + 2) * U)
    got_dx, got_dw = torch.autograd.grad(y, (x, w), dy)
    dx, dw, (rstd, u, n) = norm_grad64(x.detach(), w.detach(), dy, None, 0.0)
    mean = (u * n).abs().mean(-1, keepdim=True)
    bound = half_step(dtype) * dx.abs() + U * (rstd * ((NORM + 4) * u.abs() + (DEPTH + 3 * NORM + 6) * n.abs() * mean))
    close_or_none(got_dx, dx, bound * 1.001 + smallest(dtype))
    terms = (dy.double() * n).abs().sum(0)
    close_or_none(got_dw, dw, half_step(dtype) * dw.abs() + U * (9 + NORM + 1) * terms + smallest(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_int8_of_one_token(cuda, width, dtype):
    """A decode step's row, as it lies."""
    x, r = (normal(1, width, dtype=dtype, seed=width + i).to(cuda) for i in (0, 1))
    w = normal(width, dtype=dtype, seed=2).to(cuda)
    for added in (r, None):
        eight, stream = f2s.add_rms_norm_int8(x, w, added)
        want, s, w64, rstd = norm64(x, w, added, 1e-6)
        assert torch.equal(stream, want)
        p = s * w64
        assert torch.equal(eight.values, nearest_whole(p, row_max(p)))
        scale = (row_max(p) * rstd / 127)[:, 0]
        close(eight.scale, scale, scale * (NORM + 2) * U + 1e-45)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_checkpoints_of_every_16_bit_value(cuda, dtype):
    """Groups that hold all positive values of the binades in which 127 v / m is
    between 1/4 and 127, for maxima of every kind of significand."""
    bits = 7 if dtype == torch.bfloat16 else 10
    significands = torch.arange(2**bits, 2 ** (bits + 1), dtype=torch.float64)
    values = torch.cat([significands * 2.0**e for e in range(-10, 1)]) * 2.0**-bits  # below 2
    values = torch.nn.functional.pad(values, (0, -len(values) % 127)).view(-1, 127)
    maxima = (significands[:: 1 if dtype == torch.bfloat16 else 5] * 2.0**-bits)[:, None, None]
    held = torch.where(values <= maxima, values, 0.0)
    held = torch.cat([maxima.expand(-1, len(values), 1), held], 2)  # (maxima, groups, 128)
    rows, groups = held.shape[:2]
    want = nearest_whole(held, row_max(held))
    gate = held.flatten(1)
    kept, scale = keep_groups(torch.cat([gate, -gate], 1).to(dtype).to(cuda))
    assert torch.equal(kept[:, :, 0].cpu(), want) and torch.equal(kept[:, :, 1].cpu(), -want)
    assert torch.equal(scale.cpu(), (maxima / 127).float().expand(rows, groups, 2))


def keep_groups(projected):
    """The forward's checkpoint of whole groups: values (rows, groups, 2, 128) in
    the channels' order, scales (rows, groups, 2)."""
    rows, hidden = projected.shape[0], projected.shape[1] // 2
    groups = hidden // 128

    def call(p):
        y = p.new_empty(len(p), hidden)
        kept = torch.empty(len(p), groups, 2, 128, dtype=torch.int8, device=p.device)
        scale = torch.empty(len(p), groups, 2, device=p.device)
        f2s._lib.call("f2s_swiglu", p.data_ptr(), 2 * hidden, {torch.bfloat16: 1, torch.float16: 2}[p.dtype], len(p), hidden,
                      y.data_ptr(), kept.data_ptr(), scale.data_ptr(), f2s._lib.stream_handle())
        return kept, scale

    # where each channel's byte lies: that of a group whose values name their channels
    named = torch.arange(128, device=projected.device).repeat(2 * groups).to(projected.dtype)
    place = call(named[None])[0][0].long().argsort(-1)
    kept, scale = call(projected)
    return kept.gather(3, place.expand(rows, -1, -1, -1)), scale


def test_forward_mode_derivatives_are_refused():
    """On the host, before anything else of the call: no output without its tangent."""
    plain = torch.ones(4, 8)
    w, eight = torch.ones(8), Int8Rows(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4))
    with forward_ad.dual_level():
        for grad in (False, True):
            x = forward_ad.make_dual(plain.clone().requires_grad_(grad), torch.ones(4, 8))
            dual_w = forward_ad.make_dual(w.clone().requires_grad_(grad), w)
            scale = forward_ad.make_dual(torch.ones(4).requires_grad_(grad), torch.ones(4))
            learnt = Int8Rows(eight.values, scale)
            calls = [lambda: f2s.add_rms_norm(x, w), lambda: f2s.add_rms_norm(plain, dual_w),
                     lambda: f2s.add_rms_norm(plain, w, x), lambda: f2s.add_rms_norm_int8(plain, w, x),
                     lambda: f2s.swiglu(x), lambda: f2s.swiglu(x, checkpoint="int8"), lambda: f2s.swiglu_int8(x),
                     lambda: f2s.quantize_rows(x), lambda: learnt.dequantize(), lambda: f2s.linear_int8(learnt, eight),
                     lambda: f2s.linear_int8(eight, learnt),
                     lambda: f2s.linear_int8(eight, eight, scale, dtype=torch.float32)]
            for call in calls:
                with pytest.raises(ValueError, match="forward-mode"):
                    call()
                with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                    call()
        primal = forward_ad.unpack_dual(x).primal
        with pytest.raises(ValueError, match="CUDA tensors"):  # without its tangent it is an ordinary one
            f2s.swiglu(primal)


@pytest.mark.gpu
def test_forward_mode_derivatives_on_the_device_are_refused(cuda):
    x, w = normal(4, 64, seed=1).to(cuda), normal(64, seed=2).to(cuda)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda t: f2s.add_rms_norm(t, w), lambda t: f2s.swiglu(t), lambda t: f2s.quantize_rows(t)):
            with pytest.raises(ValueError, match="forward-mode"):
                call(dual)
            call(x)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,K", [(24, 515, 4096), (24, 2048, 8192), (60, 300, 2048), (300, 192, 200), (3000, 1024, 4096),
                                         (5000, 4096, 192)])
def test_linear_int8_beside_a_wait_that_ran_out(cuda, rows, cols, K):
    """A wait that ran out elsewhere ends the product's waits early: nothing is
    written beside its rows, the error is reported, and the next call is whole."""
    x, w = eighths(rows, K, 1, cuda), eighths(cols, K, 2, cuda)
    want = f2s.linear_int8(x, w)
    f2s._lib.check_device_error()
    y = torch.full((rows + 3, cols), 55.0, dtype=torch.bfloat16, device=cuda)
    f2s._lib.call("f2s_selftest_wait_timeout", 64, f2s._lib.stream_handle())
    for _ in range(5):
        f2s._lib.call("f2s_linear_int8", x.values.data_ptr(), x.values.stride(0), x.scale.data_ptr(), w.values.data_ptr(),
                      w.values.stride(0), w.scale.data_ptr(), None, y.data_ptr(), cols, 1, rows, cols, K,
                      f2s._lib.stream_handle())
    with pytest.raises(f2s._lib.Flow2SurfError, match="device error 1"):
        f2s._lib.check_device_error()
    assert (y[rows:] == 55).all()
    for _ in range(3):
        assert torch.equal(f2s.linear_int8(x, w), want)
    f2s._lib.check_device_error()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [8, 600])
def test_linear_int8_from_a_thread_without_a_context(cuda, rows):
    """The first CUDA call of a host thread may be one of the C entry."""
    x, w = eighths(rows, 256, 1, cuda), eighths(192, 256, 2, cuda)
    want = f2s.linear_int8(x, w)
    y = torch.empty_like(want)
    torch.cuda.synchronize()
    entry, status = f2s._lib.lib().f2s_linear_int8, []
    args = (x.values.data_ptr(), 256, x.scale.data_ptr(), w.values.data_ptr(), 256, w.scale.data_ptr(), None, y.data_ptr(),
            192, 1, rows, 192, 256, torch.cuda.Stream().cuda_stream)
    thread = threading.Thread(target=lambda: status.append((entry(*args), f2s._lib.lib().f2s_last_error())))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert status[0][0] == f2s._lib.F2S_OK, status
    assert torch.equal(y, want)


@pytest.mark.gpu
def test_linear_int8_from_two_host_threads(cuda):
    """Calls of one kernel with much and little shared memory, from threads that hold
    no lock of Python's (as a C++ host's): every launch is accepted."""
    shapes = [(8, 2048, 8192), (8, 130, 128), (8, 2000, 4096), (300, 1024, 1024), (300, 100, 512)]
    work = []
    for i, (rows, cols, K) in enumerate(shapes):
        x, w = eighths(rows, K, i, cuda), eighths(cols, K, i + 10, cuda)
        y = torch.empty(rows, cols, dtype=torch.bfloat16, device=cuda)
        args = (x.values.data_ptr(), x.values.stride(0), x.scale.data_ptr(), w.values.data_ptr(), w.values.stride(0),
                w.scale.data_ptr(), None, y.data_ptr(), cols, 1, rows, cols, K)
        work.append((f2s.linear_int8(x, w), x, w, y, args, torch.cuda.Stream()))
    torch.cuda.synchronize()
    entry, refused = f2s._lib.lib().f2s_linear_int8, []

    def calls(args, stream):
        for _ in range(2000):
            if entry(*args, stream.cuda_stream) != f2s._lib.F2S_OK:
                refused.append(f2s._lib.lib().f2s_last_error())
                return

    threads = [threading.Thread(target=calls, args=item[4:]) for item in work]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert not refused, refused
    for want, *_, y, _, _ in work:
        assert torch.equal(y, want)


def test_sizes_next_to_31_bits_are_refused():
    """Tiles end up to 255 rows, columns or channels past a size."""
    lib, most = f2s._lib.lib(), 2**31 - 256
    for rows, cols in ((most + 1, 8), (8, most + 1), (2**31 - 1, 8)):
        assert lib.f2s_linear_int8(16, 16, 16, 16, 16, 16, None, 16, 2**31, 0, rows, cols, 16, None) == f2s._lib.F2S_ERR_UNSUPPORTED
        assert b"2^31 - 256" in lib.f2s_last_error()
    assert lib.f2s_dequantize_rows(16, 2**31, 16, 1, most + 1, 16, 2**31, 1, None) == f2s._lib.F2S_ERR_UNSUPPORTED
    # and what is allowed gets as far as the null pointers
    assert lib.f2s_linear_int8(None, 16, 16, 16, 16, 16, None, 16, 2**31, 0, most, 8, 16, None) == f2s._lib.F2S_ERR_INVALID_ARGUMENT
    assert lib.f2s_dequantize_rows(None, 2**31, 16, 1, most, 16, 2**31, 1, None) == f2s._lib.F2S_ERR_INVALID_ARGUMENT


@pytest.mark.gpu
def test_gradients_of_the_two_addends_are_tensors_of_their_own(cuda):
    """One buffer holds dx for both; what backward() leaves in .grad is not shared."""
    x, r = (normal(5, 64, seed=s).to(cuda).requires_grad_() for s in (1, 2))
    w = normal(64, seed=3).to(cuda).requires_grad_()
    for _ in range(2):  # the second accumulates
        y, stream = f2s.add_rms_norm(x, w, r)
        (y.sum() + stream.sum()).backward()
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()
    held = r.grad.clone()
    x.grad.zero_()
    assert torch.equal(r.grad, held)
    x.grad = r.grad = None
    f2s.add_rms_norm(x, w, r)[1].sum().backward()  # the stream alone
    x.grad.zero_()
    assert (r.grad == 1).all()
