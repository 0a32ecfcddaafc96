"""The layer operators at the edges of their range.  Tolerances count roundings, as in test_gpu_layers.py."""
import copy
import gc
import pickle

import pytest
import torch
from torch import nn

import card_amd
from card_amd._lib import CardError
from tests import layer_reference as ref
from tests.layer_reference import TINY, U, U32, assert_within
from tests.test_gpu_layers import DEV, TYPES, chain, ids, lin_bound, rand, rows8, weights

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ norm
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,cols", [(1, 20), (3, 40), (33, 64), (5, 100), (7, 250), (2, 300)])
def test_rms_norm_weight_gradient_without_eps(dtype, rows, cols):
    """Rows that share a workgroup with places behind the last row."""
    x, g, w = rand(rows, cols, dtype=dtype), rand(rows, cols, seed=3, dtype=dtype), 1 + 0.3 * rand(cols, seed=2)
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = torch.autograd.grad(card_amd.rms_norm(xg, wg, eps=0.0), (xg, wg), g)
    dx, dw, size, dw_size = ref.rms_norm_backward(x, w, g, eps=0.0)
    assert_within(got[0], dx, dx.abs() * U[dtype] * (1 + 2 ** -8) + (2 * chain(cols) + 8) * U32 * size + TINY[dtype], "dx")
    assert_within(got[1], dw, dw.abs() * U32 + (rows + chain(cols) + 8) * U32 * dw_size, "dw")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("cols", [3, 64, 500, 2100, 9000])
def test_rms_norm_e4m3_of_tiny_rows(dtype, cols):
    """q * scale stands for y down to the smallest numbers.  eps = 1 leaves such rows as they are."""
    powers = [-100, -110, -115, -118, -119, -120, -121, -123, -126, -128, -130, -133, -136, -140, -145]
    x = torch.stack([rand(cols, seed=k).clamp(-4, 4) * 2.0 ** p for k, p in enumerate(powers)]).to(dtype)
    q, scale = card_amd.rms_norm_e4m3(x, eps=1.0)
    want, _ = ref.rms_norm(x, eps=1.0)
    got = q.float().double().cpu() * scale.double().cpu()[:, None]
    # half a step of e4m3, relative or (below its normal numbers) 2^-10 of the scale; scales below 2^-126 carry 17 bits or more
    # (they are 2^-140 at least), the products before it 32-bit roundings, and y is a multiple of 2^-149
    rel = (chain(cols) / 2 + 8) * U32 + 2.0 ** -17
    assert_within(got.float().double(), want, want.abs() * (2.0 ** -4 + rel) + 2.0 ** -10 * scale.double().cpu()[:, None] + 3 * 2.0 ** -150, "q * scale")
    amax = want.abs().amax(-1)
    least = torch.where(amax > 0, 2.0 ** -140, 0.0)          # bf16 has no number below 2^-133: the last rows are zeros there
    assert_within(scale, torch.maximum(amax / 448, least), (amax / 448) * rel + 2.0 ** -149, "scale")
    assert bool((q.float().abs().amax(-1).cpu()[amax > 2.0 ** -131] == 448).all())          # 448 * 2^-140 < 2^-131
    zero = card_amd.rms_norm_e4m3(torch.zeros(2, cols, device=DEV, dtype=dtype), eps=1.0)
    assert bool((zero[1] == 0).all()) and bool((zero[0].float() == 0).all())


# ------------------------------------------------------------------------------------------------ 4-bit weights
# (20, 12300, 24): the columns in shares; (4, 129, 16400): weights past the caches
INF_SHAPES = [(4, 31, 33), (5, 200, 40), (20, 136, 5000), (4, 129, 16400), (20, 12300, 24)]


@pytest.mark.parametrize("rows,in_f,out_f", INF_SHAPES)
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_linear4_infinite_rows(dtype, group, rows, in_f, out_f):
    """An infinite x is an infinity of the weight's sign in every output, NaN where the weight is 0 or infinities meet."""
    q, s, z, b = weights(out_f, in_f, group, True)
    lin = card_amd.QuantLinear(q, s, z, b, group=group)
    x = rand(rows, in_f, seed=5, dtype=dtype)
    clean = lin.forward(x, out_dtype=torch.float32)
    bad = x.clone()
    bad[0, 5], bad[1, in_f - 1] = float("inf"), -float("inf")
    bad[2, 3], bad[2, 30] = float("inf"), float("inf")
    for gamma, slope in ((None, None), (rand(out_f, seed=6), 0.01)):
        want, size = ref.linear4(q, s, z, b, group, bad, None, gamma, slope)
        y = lin.forward(bad, gamma=gamma, slope=slope, out_dtype=torch.float32)
        assert_within(y, want, lin_bound(want, size, group, in_f, torch.float32))
        assert bool(torch.isinf(y[0]).any())
    assert torch.equal(lin.forward(bad, out_dtype=torch.float32)[3:], clean[3:])


@pytest.mark.parametrize("rows,in_f,out_f", INF_SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
def test_linear4_rows_near_the_end_of_the_range(dtype, rows, in_f, out_f):
    """Finite rows whose sums with 16 + q pass the largest float, results that do not."""
    q, s, z, b = weights(out_f, in_f, 64, True)
    s = s * 2.0 ** -10
    lin = card_amd.QuantLinear(q, s, z, b, group=64)
    x = (rand(rows, in_f, seed=5).clamp(-3.9, 3.9) * 2.0 ** 126).to(dtype)
    x[-1] = 1.0
    want, size = ref.linear4(q, s, z, b, 64, x)
    assert bool((want.abs() < 2.0 ** 127).all())
    assert_within(lin.forward(x, out_dtype=torch.float32), want, lin_bound(want, size, 64, in_f, torch.float32))


def test_quantize_weight_of_odd_ranges():
    """Ranges below the normal numbers and past the largest one; a group that holds a NaN or an infinity is NaN."""
    group = 32
    w = rand(9, 96, seed=3).clamp(-3, 3)
    w[1] *= 2.0 ** -126
    w[2] *= 2.0 ** -135
    w[3] = w[3].abs() * 2.0 ** -130
    w[4] = w[4].clamp(-1.9, 1.9) * 2.0 ** 127
    w[4, 0], w[4, 1] = 1.9 * 2.0 ** 127, -1.9 * 2.0 ** 127
    w[5, 40], w[6, 70], w[7, 3] = float("nan"), float("inf"), -float("inf")
    q, s, z = card_amd.quantize_weight(w, group=group)
    at = torch.arange(96) // group
    step = s.cpu().double()[:, at]
    deq = (q.cpu().double() - z.cpu().double()[:, at]) * step
    w64 = w.cpu().double()
    bad = torch.zeros(9, 96, dtype=torch.bool)
    bad[5, 32:64], bad[6, 64:], bad[7, :32] = True, True, True
    assert bool(torch.isnan(deq[bad]).all())
    # a scale below the normal numbers is off by 2^-150, sixteen steps of it
    bound = step * (0.5 + 20 * 4 * U32) + 4 * U32 * w64.abs() + 16 * 2.0 ** -150
    assert bool(((deq - w64).abs() <= bound)[~bad].all())
    assert bool((s[1:5] > 0).all()) and bool(torch.isfinite(s[:5]).all())


# ------------------------------------------------------------------------------------------------ copies
def test_copies_of_packed_weights():
    """A shallow copy holds the weights when the original is gone; other copies are refused."""
    net = nn.Sequential(nn.Linear(96, 40), nn.LeakyReLU(), nn.Dropout(0.2), nn.Linear(40, 3)).to(DEV).eval()
    x = rand(5, 96)
    for make in (lambda: card_amd.QuantLinear(*weights(24, 96, 32, True), group=32), lambda: card_amd.GuidanceNet.from_module(net),
                 lambda: card_amd.GuidanceNet.from_module(net, weight_bits=4)):
        a = make()
        want = a(x)
        for how in (copy.deepcopy, pickle.dumps):
            with pytest.raises(CardError, match="pack them again"):
                how(a)
        b = copy.copy(a)
        del a
        gc.collect()
        others = [make() for _ in range(4)]          # would lie where freed weights were
        assert torch.equal(b(x), want)
        del others


# ------------------------------------------------------------------------------------------------ derivatives
def calls(x, w, lin):
    return [lambda x: card_amd.dropout(x, 0.3, seed=1), lambda x: card_amd.dropout(x.detach(), 0.3, seed=1, residual=x), lambda x: card_amd.rms_norm(x, w),
            lambda x: card_amd.rms_norm(x.detach(), w, residual=x)[0], lambda x: card_amd.rms_norm(x.detach(), x[0]), lambda x: card_amd.rms_norm_e4m3(x, w)[1],
            lambda x: card_amd.rms_norm_e4m3(x.detach(), x[0])[1], lin, lambda x: lin(x.detach(), gamma=x[0, :8].contiguous())]


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw
    x, t, w = rand(4, 64), rand(4, 64, seed=1), 1 + 0.1 * rand(64, seed=2)
    lin = card_amd.QuantLinear(*weights(8, 64, 32, True), group=32)
    for leaf in (False, True):
        for k, call in enumerate(calls(x, w, lin)):
            with fw.dual_level():
                dual = fw.make_dual(x.clone().requires_grad_(leaf), t)
                with pytest.raises(CardError, match="forward-mode|no backward"):
                    call(dual)
    a = x.clone().requires_grad_(True)
    for y in (card_amd.dropout(a, 0.3, seed=1), card_amd.rms_norm(a, w)):
        with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, a, fw.make_dual(x, t), retain_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, a, torch.stack((x, t)), is_grads_batched=True)
    for call in calls(x, w, lin):          # and behind the level all is as before
        assert torch.isfinite(call(x)).all()


def test_transforms_and_traces_are_refused():
    x, w = rand(4, 64), 1 + 0.1 * rand(64, seed=2)
    lin = card_amd.QuantLinear(*weights(8, 64, 32, True), group=32)
    for call in calls(x, w, lin)[:1] + calls(x, w, lin)[2:3] + calls(x, w, lin)[5:6] + [lambda x: lin(x)]:          # a trace wants a function
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x[None])
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x,), (x,))
        with pytest.raises(CardError, match="trace"):
            torch.jit.trace(call, x, check_trace=False)


@pytest.mark.parametrize("rows,in_f,out_f", [(128, 200, 72), (512, 1000, 130), (6400, 136, 48), (65535, 100, 40), (1000, 70, 4200), (300, 40, 16400)])
@pytest.mark.parametrize("dtype", TYPES + [torch.float8_e4m3fn], ids=ids)
def test_linear4_of_many_rows(dtype, rows, in_f, out_f):
    q, s, z, b = weights(out_f, in_f, 64, True)
    lin = card_amd.QuantLinear(q, s, z, b, group=64)
    x, xs = rows8(rows, in_f) if dtype is torch.float8_e4m3fn else (rand(rows, in_f, seed=5, dtype=dtype), None)
    want, size = ref.linear4(q, s, z, b, 64, x, xs, None, 0.01)
    y = lin.forward(x, xs, slope=0.01)
    assert_within(y, want, lin_bound(want, size, 64, in_f, y.dtype))
    # a row is the same in a call of few rows of the same form (more than 16)
    part = slice(rows - 20, rows)
    assert torch.equal(lin.forward(x[part], None if xs is None else xs[part], slope=0.01), y[part])


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_weight_is_the_nearest(group):
    """q = round(w / scale) + zero clamped to 0..15: off by half a step at most, also at the ends of the range, where what the
    clamp takes away is what rounding the zero point moved."""
    w = rand(61, 333, seed=3) + 0.5 * rand(61, 1, seed=4)
    q, s, z = card_amd.quantize_weight(w, group=group)
    at = torch.arange(333) // group
    step = s.cpu().double()[:, at]
    deq = (q.cpu().double() - z.cpu().double()[:, at]) * step
    w64 = w.cpu().double()
    # scale, its reciprocal and the quotient are rounded: a few 2^-24 of |w| + 15 steps
    assert bool(((deq - w64).abs() <= step * (0.5 + 20 * 4 * U32) + 4 * U32 * w64.abs()).all())


@pytest.mark.parametrize("rows,in_f,out_f,group", [(13, 465, 13, 128), (1, 4096, 512, 128), (60, 70, 9, 64), (24, 4096, 5000, 32), (20, 2048, 16400, 64), (16, 12000, 100, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn], ids=ids)
def test_linear4_fp32_results_of_short_rows(dtype, rows, in_f, out_f, group):
    """fp32 results of rows of 8 and 16 bits are as exact as a product of 32 bits, root mean square: products of bf16 and e4m3 rows
    have 13 bits at most, and their sums over a group are all but exact; those of fp16 rows have 16, and the two sums, some five
    times their difference together, are rounded at their last place."""
    q, s, z, b = weights(out_f, in_f, group, True)
    x, xs = rows8(rows, in_f) if dtype is torch.float8_e4m3fn else (rand(rows, in_f, seed=5, dtype=dtype), None)
    want, _ = ref.linear4(q, s, z, None, group, x, xs)
    y = card_amd.QuantLinear(q, s, z, group=group)(x, xs, out_dtype=torch.float32).cpu().double()
    n = -(-in_f // 32) + -(-in_f // group)
    assert float((y - want).norm() / want.norm()) <= (n ** 0.5 + (5 if dtype is torch.float16 else 0)) * U32
