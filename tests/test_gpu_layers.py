"""The layer operators (card_amd.layers: dropout, rms_norm, rms_norm_e4m3, QuantLinear) against their formulas in 64 bits.

Tolerances count roundings: half a step of the output's type on the result (U), and 2^-24 for each 32-bit operation on the
way, relative to the terms that it adds."""
import gc

import pytest
import torch

import card_amd
from card_amd._lib import CardError
from tests import layer_reference as ref
from tests.layer_reference import TINY, U, U32, assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda v: str(v).replace("torch.", "")  # noqa: E731


def rand(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def off_by(t, k):
    """t's values in memory that starts k elements after an allocation's start"""
    buf = torch.empty(t.numel() + k, dtype=t.dtype, device=t.device)
    v = buf[k:].view(t.shape)
    v.copy_(t)
    return v


# ------------------------------------------------------------------------------------------------ dropout
def drop_bound(want, x, p, residual, dtype, terms=1):
    # the scale and its product (and the sum): one rounding each; then the output's
    s = 1 / (1 - p) if p < 1 else 0.0
    size = x.detach().cpu().double().abs() * s
    if residual is not None:
        size = size + residual.detach().cpu().double().abs()
    return U[dtype] * want.abs() * (1 + 2 ** -8) + (2 + terms) * U32 * size + TINY[dtype]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape,n_z,offset,draw", [((1, 1), 1, 0, 0), ((1, 3), 1, 3, 1), ((7, 100), 1, 0, 2), ((5, 129), 3, 5, 0), ((33, 8), 7, 2 ** 34 + 6, 0),
                                                    ((2, 3, 40), 2, 1, 9), ((3, 1), 70, 2, 0), ((1, 4099), 1, 2 ** 62, 2 ** 31 - 1), ((4, 64), 300, 0, 0)])
def test_dropout_forward_and_backward(dtype, shape, n_z, offset, draw):
    p, seed = 0.3, 0xFEDCBA9876543210
    out_shape = shape if n_z == 1 else shape[:-1] + (n_z, shape[-1])
    x, r, g = rand(*shape, dtype=dtype), rand(*out_shape, seed=1, dtype=dtype), rand(*out_shape, seed=2, dtype=dtype)
    kw = dict(seed=seed, elem_offset=offset, draw=draw, n_z=n_z)
    for res in (None, r):
        want, mask = ref.dropout(x, p, residual=res, **kw)
        xg = x.clone().requires_grad_(True)
        rg = None if res is None else res.clone().requires_grad_(True)
        y = card_amd.dropout(xg, p, residual=rg, **kw)
        assert y.dtype is dtype and tuple(y.shape) == tuple(out_shape)
        xe = x if n_z == 1 else x.unsqueeze(-2).expand(out_shape)
        assert_within(y, want, drop_bound(want, xe, p, res, dtype), "y")
        assert torch.equal(card_amd.dropout(x, p, residual=res, **kw), y.detach())          # with and without a graph
        grads = torch.autograd.grad(y, [xg] if rg is None else [xg, rg], g)
        gs = torch.where(mask, g.cpu().double() / (1 - p), torch.zeros((), dtype=torch.float64))
        size = gs.abs() if n_z == 1 else gs.abs().sum(-2)
        dx = gs if n_z == 1 else gs.sum(-2)
        # a sum of n_z terms rounds at most n_z times, and the scale and its product once each
        assert_within(grads[0], dx, U[dtype] * dx.abs() * (1 + 2 ** -8) + (n_z + 2) * U32 * size + TINY[dtype], "dx")
        if rg is not None:
            assert torch.equal(grads[1], g)


def test_dropout_extremes_of_p_and_values():
    x = rand(300, 7)
    r = rand(300, 7, seed=1)
    assert torch.equal(card_amd.dropout(x, 0.0, seed=1), x)
    assert torch.equal(card_amd.dropout(x, 1.0, seed=1), torch.zeros_like(x))
    assert torch.equal(card_amd.dropout(x, 1.0, seed=1, residual=r), r)
    bad = x.clone()
    bad[::2] = float("inf")
    bad[1::2] = float("nan")
    mask = ref.keep_mask(bad.numel(), 0.5, 3).reshape(bad.shape)
    y = card_amd.dropout(bad, 0.5, seed=3).cpu()
    assert bool((y[~mask] == 0).all()) and not torch.isfinite(y[mask]).any()
    tiny = 2.0 ** -31                                   # two of 2^32 values of a word drop an element
    assert torch.equal(card_amd.dropout(x, tiny, seed=5).cpu() != 0, ref.keep_mask(x.numel(), tiny, 5).reshape(x.shape))
    for shape in ((0, 5), (5, 0), (0,)):
        z = torch.zeros(shape, device=DEV, requires_grad=True)
        y = card_amd.dropout(z, 0.5, seed=1, n_z=3)
        assert tuple(y.shape) == shape[:-1] + (3, shape[-1])
        assert torch.autograd.grad(y.sum(), z)[0].shape == z.shape


def test_dropout_is_one_mask_under_sharding_views_and_alignment():
    x = rand(64, 33, dtype=torch.bfloat16)
    whole = card_amd.dropout(x, 0.2, seed=9)
    parts = [card_amd.dropout(x[a:b], 0.2, seed=9, elem_offset=a * 33) for a, b in ((0, 1), (1, 20), (20, 64))]
    assert torch.equal(torch.cat(parts), whole)
    assert torch.equal(card_amd.dropout(off_by(x, 3), 0.2, seed=9, residual=off_by(torch.zeros_like(x), 1)), whole)
    assert torch.equal(card_amd.dropout(x.t().contiguous().t(), 0.2, seed=9), whole)
    assert not torch.equal(card_amd.dropout(x, 0.2, seed=9, draw=1), whole)
    assert not torch.equal(card_amd.dropout(x, 0.2, seed=10), whole)
    # a gradient that is an expanded scalar
    xg = x.clone().requires_grad_(True)
    g = torch.autograd.grad(card_amd.dropout(xg, 0.2, seed=9).sum(), xg)[0]
    assert torch.equal(g != 0, ref.keep_mask(x.numel(), 0.2, 9).reshape(x.shape).to(DEV))


def test_dropout_share_of_dropped_elements():
    y = card_amd.dropout(torch.ones(1 << 22, device=DEV), 0.1, seed=77)
    dropped = float((y == 0).double().mean())
    assert abs(dropped - 0.1) < 6 * (0.1 * 0.9 / 2 ** 22) ** 0.5          # six standard deviations of a binomial share


def test_dropout_seed_tensor_and_replays():
    """A captured graph draws the mask of the numbers that its seed tensor holds when it is replayed; forward and backward."""
    x = rand(50, 37).requires_grad_(True)
    g = rand(50, 37, seed=1)
    state = torch.tensor([5, 8], dtype=torch.int64, device=DEV)
    eager = card_amd.dropout(x.detach(), 0.4, seed=5, elem_offset=8 + 3)
    assert torch.equal(card_amd.dropout(x.detach(), 0.4, seed=state, elem_offset=3), eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(card_amd.dropout(x, 0.4, seed=state), x, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = card_amd.dropout(x, 0.4, seed=state)
        dx = torch.autograd.grad(y, x, g)[0]
    for seed, off in ((5, 0), (6, 4), (-7, 1), (5, 0)):
        state.copy_(torch.tensor([seed, off]))
        graph.replay()
        torch.cuda.synchronize()
        want, mask = ref.dropout(x, 0.4, seed=seed & (2 ** 64 - 1), elem_offset=off)
        assert_within(y, want, drop_bound(want, x, 0.4, None, torch.float32))
        assert torch.equal(dx != 0, mask.to(DEV))
        card_amd.dropout(x.detach(), 0.1, seed=1)          # the program's own eager work in between
    # numbers that change between the two passes are an error, not another mask
    y = card_amd.dropout(x, 0.4, seed=state)
    state.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, g)


def test_dropout_past_32_bits_of_elements():
    rows, cols = 65537, 65536
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device=DEV)
    y = card_amd.dropout(x, 0.5, seed=4)
    for lo in (0, rows - 2):
        mask = ref.keep_mask(2 * cols, 0.5, 4, elem_offset=lo * cols).reshape(2, cols)
        assert torch.equal(y[lo:lo + 2].cpu() == 2, mask)


# ------------------------------------------------------------------------------------------------ norm
# widths around every change of form: threads per row and vectors per thread, of 4 (fp32) and 8 (16 bits) elements
WIDTHS = [1, 2, 7, 32, 33, 64, 65, 256, 257, 500, 512, 513, 1000, 1025, 2048, 2049, 4096, 5003, 8193]


def chain(cols):
    """32-bit roundings in a sum over a row, at most: a thread's own values, the join, and the three of the mean, the sum
    with eps and its root -- a thread holds at most 64 values, rows are joined over at most 16 waves"""
    return 64 + 6 + 16 + 4


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_forward(dtype, cols, residual):
    rows = 5 if cols > 64 else 37
    x, r = rand(rows, cols, dtype=dtype), rand(rows, cols, seed=1, dtype=dtype, scale=3.0) if residual else None
    x[2] = 0.0
    if residual:
        r[2] = 0.0
    for w in (None, 1 + 0.3 * rand(cols, seed=2), (1 + 0.3 * rand(cols, seed=2)).to(dtype)):
        out = card_amd.rms_norm(x, w, residual=r, eps=1e-5)
        want, h = ref.rms_norm(x, w, r, eps=1e-5)
        y = out[0] if residual else out
        # rstd carries half the sum's roundings; h, the root, the division and two products add five
        assert_within(y, want, want.abs() * (U[dtype] * (1 + 2 ** -8) + (chain(cols) / 2 + 5) * U32) + TINY[dtype], "y")
        if residual:
            assert_within(out[1], h, h.abs() * (U[dtype] + U32) + TINY[dtype], "h")
    assert bool((y[2] == 0).all())


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("cols", WIDTHS)
def test_rms_norm_e4m3(dtype, cols):
    rows = 5 if cols > 64 else 37
    x, r = rand(rows, cols, dtype=dtype), rand(rows, cols, seed=1, dtype=dtype, scale=3.0)
    w = 1 + 0.3 * rand(cols, seed=2)
    x[2], r[2] = 0.0, 0.0
    for res in (None, r):
        out = card_amd.rms_norm_e4m3(x, w, residual=res)
        want, h = ref.rms_norm(x, w, res)
        q, scale = out[0], out[1]
        assert q.dtype is torch.float8_e4m3fn and tuple(scale.shape) == (rows,)
        amax = want.abs().amax(-1)
        rel = (chain(cols) / 2 + 5) * U32
        assert_within(scale, amax / 448, amax / 448 * (rel + 2 * U32), "scale")
        v = torch.where(amax[:, None] > 0, want * (448 / amax.clamp_min(1e-300))[:, None], torch.zeros_like(want))
        # e4m3: half a step is 2^-4 of the value, or 2^-10 below its smallest normal number; the value itself carries rel twice
        # (y and amax), the quotient and the product
        assert_within(q.float(), v, v.abs() * (2.0 ** -4 + 2 * rel + 3 * U32) + 2.0 ** -10, "q")
        assert bool((q.float().abs().amax(-1)[amax > 0] == 448).all())
        if res is not None:
            assert_within(out[2], h, h.abs() * (U[dtype] + U32) + TINY[dtype], "h")
        assert float(scale[2]) == 0 and bool((q[2].float() == 0).all())


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_backward(dtype, cols, residual):
    rows = 5 if cols > 64 else 300
    x, r = rand(rows, cols, dtype=dtype), rand(rows, cols, seed=1, dtype=dtype) if residual else None
    g, gh = rand(rows, cols, seed=3, dtype=dtype), rand(rows, cols, seed=4, dtype=dtype)
    for w in (None, 1 + 0.3 * rand(cols, seed=2), (1 + 0.3 * rand(cols, seed=2)).to(dtype)):
        leaves = [t.clone().requires_grad_(True) for t in (x, r, w) if t is not None]
        it = iter(leaves)
        xg, rg, wg = next(it), next(it) if residual else None, next(it) if w is not None else None
        out = card_amd.rms_norm(xg, wg, residual=rg)
        h = out[1].detach() if residual else x
        grads = torch.autograd.grad(out if residual else (out,), leaves, (g, gh) if residual else (g,))
        dx, dw, size, dw_size = ref.rms_norm_backward(h, w, g, gh if residual else None)
        # rows of at most 8 vectors are computed in 64 bits; elsewhere the sums carry chain() roundings and the rest eight
        err = 2.0 ** -40 if cols <= 8 * 16 // dtype.itemsize else (2 * chain(cols) + 8) * U32
        assert_within(grads[0], dx, dx.abs() * U[dtype] * (1 + 2 ** -8) + err * size + TINY[dtype], "dx")
        if residual:
            assert torch.equal(grads[1], grads[0])
        if w is not None:
            assert grads[-1].dtype is w.dtype
            assert_within(grads[-1], dw, dw.abs() * U[w.dtype] * (1 + 2 ** -8) + (rows + chain(cols) + 8) * U32 * dw_size + TINY[w.dtype], "dw")
            again = torch.autograd.grad(card_amd.rms_norm(xg, wg, residual=rg) if residual else (card_amd.rms_norm(xg, wg),),
                                        leaves, (g, gh) if residual else (g,))
            assert torch.equal(again[-1], grads[-1])          # a fixed order of sums


def test_rms_norm_gradients_against_differences():
    cols, rows = 40, 3
    x, r, w = rand(rows, cols), rand(rows, cols, seed=1), 1 + 0.3 * rand(cols, seed=2)
    g, gh = rand(rows, cols, seed=3), rand(rows, cols, seed=4)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    grads = torch.autograd.grad(card_amd.rms_norm(leaves[0], leaves[2], residual=leaves[1]), leaves, (g, gh))

    def loss(x, r, w):
        y, h = ref.rms_norm(x, w, r)
        return float((y * g.cpu().double()).sum() + (h * gh.cpu().double()).sum())
    for which in range(3):
        base = [t.cpu().double() for t in (x, r, w)]
        d = torch.randn(base[which].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(which))
        step = 1e-5
        hi, lo = list(base), list(base)
        hi[which], lo[which] = base[which] + step * d, base[which] - step * d
        num = (loss(*hi) - loss(*lo)) / (2 * step)
        got = float((grads[which].cpu().double() * d).sum())
        # central differences: third derivatives times step^2 (about 1e-9 of the terms) and 32-bit gradients
        assert abs(num - got) < 1e-5 * float((grads[which].cpu().double() * d).abs().sum())


def test_rms_norm_only_one_of_its_results_is_used():
    x, r, w = (t.requires_grad_(True) for t in (rand(4, 100), rand(4, 100, seed=1), 1 + rand(100, seed=2)))
    g = rand(4, 100, seed=3)
    y, h = card_amd.rms_norm(x, w, residual=r)
    dx, dr, dw = torch.autograd.grad(h, (x, r, w), g, retain_graph=True)
    assert torch.equal(dx, g) and torch.equal(dr, g) and bool((dw == 0).all())
    both = torch.autograd.grad((y, h), (x, w), (g, torch.zeros_like(g)), retain_graph=True)
    only = torch.autograd.grad(y, (x, w), g)
    assert torch.equal(both[0], only[0]) and torch.equal(both[1], only[1])


def test_rms_norm_values_that_are_not_finite_stay_in_their_rows():
    x, w = rand(6, 300), 1 + 0.2 * rand(300, seed=1)
    clean = card_amd.rms_norm(x, w)
    cq, cs = card_amd.rms_norm_e4m3(x, w)
    bad = x.clone()
    bad[1, 7], bad[3, 299], bad[4, 0] = float("nan"), float("inf"), -float("inf")
    y = card_amd.rms_norm(bad, w)
    q, scale = card_amd.rms_norm_e4m3(bad, w)
    fine = torch.tensor([0, 2, 5], device=DEV)
    assert torch.equal(y[fine], clean[fine]) and torch.equal(q[fine].float(), cq[fine].float()) and torch.equal(scale[fine], cs[fine])
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[3, 299])) and bool((y[3, :299] == 0).all())
    assert bool(torch.isnan(scale[[1, 3, 4]]).all()) and bool(torch.isnan(q[[1, 3, 4]].float()).all())


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_rms_norm_views_alignment_and_empty(dtype):
    x, w, r = rand(9, 515, dtype=dtype), 1 + 0.2 * rand(515, seed=1), rand(9, 515, seed=2, dtype=dtype)
    y, h = card_amd.rms_norm(x, w, residual=r)
    y2, h2 = card_amd.rms_norm(off_by(x, 1), off_by(w, 3), residual=off_by(r, 5))
    assert torch.equal(y, y2) and torch.equal(h, h2)
    y3, _ = card_amd.rms_norm(x.reshape(3, 3, 515).transpose(0, 1), w, residual=r.reshape(3, 3, 515).transpose(0, 1))
    assert torch.equal(y3.transpose(0, 1).reshape(9, 515), y)
    e = torch.zeros(0, 515, device=DEV, dtype=dtype, requires_grad=True)
    wg = w.clone().requires_grad_(True)
    out = card_amd.rms_norm(e, wg)
    assert out.shape == (0, 515)
    de, dw = torch.autograd.grad(out.sum(), (e, wg))
    assert de.shape == (0, 515) and torch.equal(dw, torch.zeros_like(w))
    assert card_amd.rms_norm_e4m3(e.detach())[1].shape == (0,)


@pytest.mark.parametrize("cols", [16385, 32768, 65536])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_rms_norm_long_rows(dtype, cols):
    x, r, w = rand(3, cols, dtype=dtype), rand(3, cols, seed=1, dtype=dtype), 1 + 0.2 * rand(cols, seed=2)
    g, gh = rand(3, cols, seed=3, dtype=dtype), rand(3, cols, seed=4, dtype=dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, h = card_amd.rms_norm(leaves[0], leaves[2], residual=leaves[1])
    want, hw = ref.rms_norm(x, w, r)
    assert_within(y, want, want.abs() * (U[dtype] * (1 + 2 ** -8) + (chain(cols) / 2 + 5) * U32) + TINY[dtype], "y")
    dx, _, dw = torch.autograd.grad((y, h), leaves, (g, gh))
    wx, ww, size, dw_size = ref.rms_norm_backward(h, w, g, gh)
    assert_within(dx, wx, wx.abs() * U[dtype] * (1 + 2 ** -8) + (2 * chain(cols) + 8) * U32 * size + TINY[dtype], "dx")
    assert_within(dw, ww, (3 + chain(cols) + 8) * U32 * dw_size + U32 * ww.abs(), "dw")
    q, scale, _ = card_amd.rms_norm_e4m3(x, w, residual=r)
    amax = want.abs().amax(-1)
    assert_within(scale, amax / 448, amax / 448 * ((chain(cols) / 2 + 7) * U32), "scale")


def test_rms_norm_past_32_bits_of_elements():
    rows, cols = 65537, 65536
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[-1] *= 2
    w = torch.arange(cols, device=DEV, dtype=torch.float32) / cols
    y = card_amd.rms_norm(x, w, eps=0.0)
    assert torch.equal(y[0], w.to(torch.bfloat16)) and torch.equal(y[-1], w.to(torch.bfloat16))


# ------------------------------------------------------------------------------------------------ 4-bit weights
def weights(out_f, in_f, group, zero, seed=0):
    g = torch.Generator().manual_seed(seed)
    groups = -(-in_f // group)
    q = torch.randint(0, 16, (out_f, in_f), generator=g, dtype=torch.uint8)
    scale = (0.5 + torch.rand(out_f, groups, generator=g)) / in_f ** 0.5
    z = torch.randint(0, 16, (out_f, groups), generator=g, dtype=torch.uint8) if zero else None
    bias = torch.randn(out_f, generator=g)
    return [t if t is None else t.to(DEV) for t in (q, scale, z, bias)]


def rows8(m, k, seed=5):
    x = rand(m, k, seed=seed)
    s = x.abs().amax(-1).clamp_min(1e-9) / 448
    return (x / s[:, None]).to(torch.float8_e4m3fn), s


def lin_bound(want, size, group, in_f, out_dtype):
    # products of a group round at most once each, the groups' sums twice each (scale, sum), the epilogue four times
    return U[out_dtype] * want.abs() * (1 + 2 ** -8) + (group + 2 * (-(-in_f // group)) + 4) * U32 * size + TINY[out_dtype]


SHAPES = [(1, 1, 1), (1, 64, 16), (2, 31, 33), (3, 100, 50), (5, 1001, 77), (16, 128, 128), (17, 129, 15), (33, 257, 100), (64, 512, 48), (1, 4096, 512),
          (8, 2048, 1000), (100, 300, 130), (9, 392, 5000), (3, 200, 16400), (20, 136, 16389), (40, 129, 16384),
          (30, 4100, 40), (20, 12300, 24), (40, 4216, 33), (3, 9000, 17)]


@pytest.mark.parametrize("rows,in_f,out_f", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES + [torch.float8_e4m3fn], ids=ids)
def test_linear4(dtype, group, rows, in_f, out_f):
    for zero in (False, True):
        q, s, z, b = weights(out_f, in_f, group, zero)
        lin = card_amd.QuantLinear(q, s, z, b, group=group)
        x, xs = rows8(rows, in_f) if dtype is torch.float8_e4m3fn else (rand(rows, in_f, seed=5, dtype=dtype), None)
        for gamma, slope in ((None, None), (rand(out_f, seed=6), 0.01)):
            want, size = ref.linear4(q, s, z, b, group, x, xs, gamma, slope)
            for out in (None, torch.float32) if dtype is not torch.float32 else (None, torch.bfloat16):
                y = lin.forward(x, xs, gamma=gamma, slope=slope, out_dtype=out)
                ot = out or (torch.bfloat16 if xs is not None else dtype)
                assert y.dtype is ot
                assert_within(y, want, lin_bound(want, size, group, in_f, ot), (zero, slope, ot))
    # without a bias, and from memory that starts anywhere: the same bits
    nob = card_amd.QuantLinear(q, s, z, group=group)
    assert_within(nob.forward(x, xs, out_dtype=torch.float32), ref.linear4(q, s, z, None, group, x, xs)[0],
                  lin_bound(*ref.linear4(q, s, z, None, group, x, xs), group, in_f, torch.float32))
    moved = off_by(x, 1) if dtype is not torch.float8_e4m3fn else off_by(x.view(torch.uint8), 3).view(torch.float8_e4m3fn)
    assert torch.equal(nob.forward(moved, xs), nob.forward(x, xs))


@pytest.mark.parametrize("rows,in_f,out_f,group", [(13, 465, 13, 128), (1, 4096, 512, 128), (60, 70, 9, 64), (24, 4096, 5000, 32), (20, 2048, 16400, 64)])
def test_linear4_fp32_is_as_exact_as_an_fp32_product(rows, in_f, out_f, group):
    """The sums of 16 + q on the way cost nothing: a result is off like one that is rounded once for 32 columns and once for a
    group (half a step each, at random), root mean square."""
    q, s, z, b = weights(out_f, in_f, group, True)
    x = rand(rows, in_f, seed=5)
    want, _ = ref.linear4(q, s, z, None, group, x)
    y = card_amd.QuantLinear(q, s, z, group=group)(x).cpu().double()
    n = -(-in_f // 32) + -(-in_f // group)
    assert float((y - want).norm() / want.norm()) <= n ** 0.5 * U32


def test_linear4_row_results_do_not_depend_on_their_neighbours():
    q, s, z, b = weights(200, 640, 64, True)
    lin = card_amd.QuantLinear(q, s, z, b, group=64)
    x = rand(64, 640, dtype=torch.bfloat16)
    clean = lin.forward(x)
    bad = x.clone()
    bad[5], bad[40, 3] = float("nan"), float("inf")
    y = lin.forward(bad)
    keep = [i for i in range(64) if i not in (5, 40)]
    assert torch.equal(y[keep], clean[keep]) and bool(torch.isnan(y[5]).all()) and not bool(torch.isfinite(y[40]).any())


def test_linear4_shares_of_the_columns_need_their_workspace():
    """Few outputs and long rows: the columns are split over workgroups, with the caller's scratch between the two launches."""
    import ctypes as C
    from card_amd import _lib
    L = _lib.lib()
    q, s, z, b = weights(40, 4100, 128, True)
    lin = card_amd.QuantLinear(q, s, z, b, group=128)
    x, y, n = rand(30, 4100), torch.full((30, 40), 7.0, device=DEV), C.c_uint64()
    assert L.card_linear4_workspace_bytes(lin._h, _lib.DTYPE_F32, 30, C.byref(n)) == 0 and n.value >= 2 * 30 * 40 * 4
    ws = torch.empty(n.value + 8, dtype=torch.uint8, device=DEV)
    call = lambda w, k: L.card_linear4_forward(lin._h, x.data_ptr(), _lib.DTYPE_F32, None, 30, None, 1.0, y.data_ptr(), _lib.DTYPE_F32, w, k, None)  # noqa: E731
    for w, k in ((None, 0), (None, n.value), (ws.data_ptr(), n.value - 1), (ws.data_ptr() + 8, n.value)):
        assert call(w, k) == -1 and "workspace" in L.card_last_error().decode()
    torch.cuda.synchronize()
    assert bool((y == 7).all())
    assert call(ws.data_ptr(), n.value) == 0
    torch.cuda.synchronize()
    assert torch.equal(y, lin(x))
    assert L.card_linear4_workspace_bytes(lin._h, _lib.DTYPE_BF16, 1, C.byref(n)) == 0 and n.value == 0
    assert L.card_linear4_workspace_bytes(lin._h, 9, 1, C.byref(n)) == -1 and L.card_linear4_workspace_bytes(lin._h, 0, -1, C.byref(n)) == -1
    assert L.card_linear4_workspace_bytes(lin._h, 0, 65536, C.byref(n)) == -2


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_linear4_large_values(dtype):
    """Rows near the top of the type's range: products are held in 32 bits."""
    q, s, z, b = weights(40, 256, 32, True)
    x = rand(4, 256, dtype=dtype) * (1e4 if dtype is torch.float16 else 1e30)
    s = s * 1e-3
    lin = card_amd.QuantLinear(q, s, z, b, group=32)
    want, size = ref.linear4(q, s, z, b, 32, x)
    assert_within(lin.forward(x, out_dtype=torch.float32), want, lin_bound(want, size, 32, 256, torch.float32))


def test_linear4_views_and_empty():
    q, s, z, b = weights(24, 96, 32, True)
    lin = card_amd.QuantLinear(q.t().contiguous().t(), s, z, b, group=32)
    x = rand(2, 3, 96)
    y = lin(x)
    assert y.shape == (2, 3, 24) and torch.equal(y.reshape(6, 24), lin(x.reshape(6, 96)))
    assert torch.equal(lin(x.transpose(0, 1)).transpose(0, 1), y)
    assert torch.equal(lin(x[0, 0]), y[0, 0])
    assert lin(torch.zeros(0, 96, device=DEV)).shape == (0, 24)
    assert lin(torch.zeros(0, 96, device=DEV, dtype=torch.float8_e4m3fn), torch.zeros(0, device=DEV)).shape == (0, 24)


@pytest.mark.parametrize("group", [32, 128])
def test_quantize_weight(group):
    w = rand(37, 300, seed=3)
    w[0], w[1, :group], w[2] = 0.0, 0.5, -w[2].abs()
    q, s, z = card_amd.quantize_weight(w, group=group)
    at = torch.arange(300) // group
    deq = (q.cpu().double() - z.cpu().double()[:, at]) * s.cpu().double()[:, at]
    # half a step from rounding the value, half from rounding the zero point at the range's ends
    assert bool(((deq - w.cpu().double()).abs() <= s.cpu().double()[:, at] * (1 + 1e-5)).all())
    assert bool((deq[0] == 0).all()) and int(q.max()) <= 15 and int(z.max()) <= 15
    # the values and zero span the sixteen steps
    parts = [w.cpu()[:, i:i + group] for i in range(0, 300, group)]
    span = torch.stack([p.amax(1).clamp_min(0) - p.amin(1).clamp_max(0) for p in parts], 1)
    assert torch.allclose(s.cpu() * 15, span, rtol=4 * 2.0 ** -24, atol=0)
    lin = card_amd.QuantLinear.from_float(w, group=group)
    x = rand(3, 300, seed=4)
    assert torch.equal(lin(x), card_amd.QuantLinear(q, s, z, group=group)(x))


def test_quantize_weight_of_more_groups_than_a_launch_has_waves():
    rows, cols = 1 << 21, 1024                   # 2^26 groups, a wave each
    gen = torch.Generator(device=DEV).manual_seed(3)
    w = torch.randn(rows, cols, device=DEV, generator=gen)
    whole = card_amd.quantize_weight(w, group=32)
    for part in (slice(0, 64), slice(rows // 2 - 32, rows // 2 + 32), slice(rows - 64, rows)):
        for a, b in zip(whole, card_amd.quantize_weight(w[part].contiguous(), group=32)):
            assert torch.equal(a[part], b)
    assert bool((whole[1] > 0).all())


def test_weights_that_do_not_fit_leave_no_error_behind():
    """549 GB of weights are refused by the allocator, before anything is launched; the next call is none the worse."""
    import ctypes as C
    from card_amd import _lib
    d, h, t = _lib.Linear4Desc(), C.c_void_p(), torch.zeros(16, device=DEV)
    d.struct_bytes, d.in_features, d.out_features, d.group = C.sizeof(_lib.Linear4Desc), _lib.LINEAR4_MAX_FEATURES, _lib.LINEAR4_MAX_FEATURES, 128
    d.q = d.scale = t.data_ptr()
    assert _lib.lib().card_linear4_create(C.byref(d), None, C.byref(h)) != 0 and not h.value
    x = rand(4, 64)
    assert torch.equal(card_amd.dropout(x, 0.0, seed=1), x)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ together
def test_a_layer_as_it_is_served_and_trained():
    """residual -> norm -> 8 bits -> 4-bit product -> LeakyReLU, and the training form of its ends: norm, dropout."""
    rows, cols, out_f = 20, 640, 320
    x, r, w = rand(rows, cols, dtype=torch.bfloat16), rand(rows, cols, seed=1, dtype=torch.bfloat16), 1 + 0.1 * rand(cols, seed=2)
    q4, s4, z4, b4 = weights(out_f, cols, 64, True)
    lin = card_amd.QuantLinear(q4, s4, z4, b4, group=64)
    q, s, h = card_amd.rms_norm_e4m3(x, w, residual=r)
    y = lin(q, s, slope=0.01, out_dtype=torch.float32)
    want, size = ref.linear4(q4, s4, z4, b4, 64, q, s, None, 0.01)          # from the 8-bit rows on
    assert_within(y, want, lin_bound(want, size, 64, cols, torch.float32))
    # 8-bit rows are within 2^-4 of the norm's: so is the product, relative to its terms
    yn, _ = ref.rms_norm(x, w, r)
    full, size = ref.linear4(q4, s4, z4, b4, 64, yn.float(), None, None, 0.01)
    at = torch.arange(cols) // 64
    terms = yn.abs() @ ((q4.cpu().double() - z4.cpu().double()[:, at]) * s4.cpu().double()[:, at]).abs().t()
    low = (yn.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -10) @ torch.ones(1, out_f, dtype=torch.float64)
    mags = ((q4.cpu().double() - z4.cpu().double()[:, at]) * s4.cpu().double()[:, at]).abs().sum(1)
    assert bool(((y.cpu().double() - full).abs() <= 2.0 ** -4 * terms * (1 + 1e-3) + low * mags + 1e-4).all())

    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    d = card_amd.dropout(leaves[0], 0.25, seed=11, draw=2, residual=leaves[1])
    n = card_amd.rms_norm(d, leaves[2])
    g = rand(rows, cols, seed=7, dtype=torch.bfloat16)
    dx, dr, dw = torch.autograd.grad(n, leaves, g)
    wd, mask = ref.dropout(x, 0.25, seed=11, draw=2, residual=r)
    wdd, ww, size, dw_size = ref.rms_norm_backward(d, w, g)
    assert_within(dr, wdd, U[torch.bfloat16] * wdd.abs() * (1 + 2 ** -8) + (2 * chain(cols) + 8) * U32 * size + TINY[torch.bfloat16])
    assert_within(dx, torch.where(mask, dr.cpu().double() / 0.75, torch.zeros((), dtype=torch.float64)), U[torch.bfloat16] * 1.01 * dr.cpu().double().abs() / 0.75)
    assert_within(dw, ww, (rows + chain(cols) + 8) * U32 * dw_size + U32 * ww.abs())


def test_serving_layer_in_a_captured_graph_and_on_another_stream():
    x, r, w = rand(4, 256, dtype=torch.bfloat16), rand(4, 256, seed=1, dtype=torch.bfloat16), 1 + 0.1 * rand(256, seed=2)
    lin = card_amd.QuantLinear(*weights(256, 256, 32, True), group=32)
    lin2 = card_amd.QuantLinear(*weights(128, 256, 128, False, seed=1), group=128)

    def layer():
        q, s, h = card_amd.rms_norm_e4m3(x, w, residual=r)
        y = lin(q, s, slope=0.0)
        return lin2(card_amd.dropout(y, 0.5, seed=3, n_z=3, residual=None)), h
    want = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = layer()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):          # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = layer()
        graphs.append((graph, got))
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    base = x.clone()
    for k in range(4):
        x.copy_(base * (k + 1))
        graphs[k % 2][0].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(graphs[k % 2][1], layer())), k
    x.copy_(base)


def test_gradients_where_only_some_inputs_ask_for_one():
    x, r, w, g = rand(6, 130), rand(6, 130, seed=1), 1 + 0.2 * rand(130, seed=2), rand(6, 130, seed=3)
    gh = rand(6, 130, seed=4)
    full = [t.clone().requires_grad_(True) for t in (x, r, w)]
    want = torch.autograd.grad(card_amd.rms_norm(full[0], full[2], residual=full[1]), full, (g, gh))
    drop = torch.autograd.grad(card_amd.dropout(full[0], 0.3, seed=1, residual=full[1]), full[:2], g)
    for asks in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)):
        t = [v.clone().requires_grad_(bool(a)) for v, a in zip((x, r, w), asks)]
        leaves = [v for v, a in zip(t, asks) if a]
        got = torch.autograd.grad(card_amd.rms_norm(t[0], t[2], residual=t[1]), leaves, (g, gh))
        assert len(got) == sum(asks) and all(torch.equal(a, b) for a, b in zip(got, [v for v, a in zip(want, asks) if a])), asks
        if asks[0] or asks[1]:
            leaves = [v for v, a in zip(t[:2], asks) if a]
            got = torch.autograd.grad(card_amd.dropout(t[0], 0.3, seed=1, residual=t[1]), leaves, g)
            assert all(torch.equal(a, b) for a, b in zip(got, [v for v, a in zip(drop, asks) if a])), asks
    # without a residual the weight is the second input
    wg = w.clone().requires_grad_(True)
    dw = torch.autograd.grad(card_amd.rms_norm(x, wg), wg, g)[0]
    assert_within(dw, ref.rms_norm_backward(x, w, g)[1], (6 + chain(130) + 8) * U32 * ref.rms_norm_backward(x, w, g)[3])


def test_one_tensor_as_input_and_residual():
    x, w, g, gh = rand(5, 77), 1 + 0.2 * rand(77, seed=2), rand(5, 77, seed=3), rand(5, 77, seed=4)
    a, b, c = x.clone().requires_grad_(True), x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    two = torch.autograd.grad(card_amd.rms_norm(b, w, residual=c), (b, c), (g, gh))
    assert torch.equal(torch.autograd.grad(card_amd.rms_norm(a, w, residual=a), a, (g, gh))[0], two[0] + two[1])
    two = torch.autograd.grad(card_amd.dropout(b, 0.4, seed=2, residual=c), (b, c), g)
    assert torch.equal(torch.autograd.grad(card_amd.dropout(a, 0.4, seed=2, residual=a), a, g)[0], two[0] + two[1])
    # accumulated into .grad, where the two gradients of a norm are one tensor
    y, h = card_amd.rms_norm(b, w, residual=c)
    torch.autograd.backward((y, h), (g, gh))
    first = b.grad.clone()
    b.grad.mul_(2)
    assert torch.equal(c.grad, first)


def test_second_order_is_refused():
    x = rand(3, 40).requires_grad_(True)
    for y in (card_amd.dropout(x, 0.2, seed=1), card_amd.rms_norm(x)):
        with pytest.raises(RuntimeError, match="first order"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_training_step_in_a_captured_graph():
    """norm and dropout, forward and backward, captured together; replays with the program's own work in between."""
    w = (1 + 0.1 * rand(256, seed=2)).requires_grad_(True)
    x, r = rand(40, 256, dtype=torch.bfloat16).requires_grad_(True), rand(40, 256, seed=1, dtype=torch.bfloat16).requires_grad_(True)
    g = rand(40, 256, seed=3, dtype=torch.bfloat16)

    def train():
        d = card_amd.dropout(x, 0.25, seed=9, residual=r)
        y, h = card_amd.rms_norm(d, w, residual=r)
        return torch.autograd.grad((y, h), (x, r, w), (g, g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            train()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = train()
        graphs.append((graph, got))
    for k in range(4):
        with torch.no_grad():
            x.mul_(1.5)
            g.add_(0.25)
        graphs[k % 2][0].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(graphs[k % 2][1], train())), k


@pytest.mark.parametrize("name", ["dropout", "norm"])
@pytest.mark.parametrize("how", ["grad", "backward"])
def test_captured_backward_beside_an_eager_graph_of_the_same_leaves(name, how):
    """Refused: the leaves' gradient nodes are on the eager pass's stream.  Without the eager graph, and on two streams of one
    capture, it runs.  The leaf x does not lie row by row."""
    x, r, w = rand(64, 40).t().requires_grad_(True), rand(40, 64, seed=1).requires_grad_(True), (1 + 0.1 * rand(64, seed=2)).requires_grad_(True)
    g = rand(40, 64, seed=3)
    leaves = (x, r) if name == "dropout" else (x, r, w)

    def forward():
        return card_amd.dropout(x, 0.3, seed=1, residual=r) if name == "dropout" else card_amd.rms_norm(x, w, residual=r)[0]

    def backward(y):
        if how == "grad":
            return torch.autograd.grad(y, leaves, g)
        y.backward(g)
        return [t.grad for t in leaves]
    want = [t.clone() for t in backward(forward())]
    for t in leaves:
        t.grad = None
    eager = forward()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        y = forward()
        with pytest.raises(RuntimeError, match="before the capture"):
            backward(y)
    del eager, y
    gc.collect()                                         # what the exception's frames held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = backward(forward())
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        forward()
    for t in leaves:
        t.grad = None
    del got
    graph, two = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        one = forward()                                  # the leaves' gradient nodes are on this stream, the pass on another
        two.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(two):
            got = torch.autograd.grad(forward(), leaves, g)
        torch.cuda.current_stream().wait_stream(two)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("cols", [40, 200, 1000, 6001, 9000])
def test_large_calls_are_their_parts(dtype, cols):
    """Calls of more than 300 MB take kernels of their own: a row has the same bits there as in a small call."""
    rows = 320_000_000 // (4 * cols * dtype.itemsize) + 37
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, r, g, gh = (torch.randn(rows, cols, device=DEV, generator=gen).to(dtype) for _ in range(4))
    w = 1 + 0.1 * rand(cols, seed=2)
    part = slice(rows - 50, rows)

    def train(x, r, g, gh, offset):
        a, b, c = x.clone().requires_grad_(True), r.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y, h = card_amd.rms_norm(a, c, residual=b)
        dx = torch.autograd.grad((y, h), (a, c), (g, gh))
        d = card_amd.dropout(a, 0.3, seed=5, elem_offset=offset, residual=b)
        q, s, h8 = card_amd.rms_norm_e4m3(x, w, residual=r)
        return [y, h, dx[0], d, torch.autograd.grad(d, a, g)[0], q.view(torch.uint8), s, h8, card_amd.rms_norm(x, w), card_amd.dropout(x, 0.3, seed=5, elem_offset=offset)], dx[1]
    whole, dw = train(x, r, g, gh, 0)
    parts, _ = train(x[part], r[part], g[part], gh[part], (rows - 50) * cols)
    for k, (a, b) in enumerate(zip(whole, parts)):
        assert torch.equal(a[part], b), k
    # the weight's gradient in 64 bits, on the device: rows + chain() + 8 roundings of the sum of magnitudes at most
    h = whole[1].double()
    unit = g.double() * h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6)
    assert bool(((dw.double() - unit.sum(0)).abs() <= (rows + chain(cols) + 8) * U32 * unit.abs().sum(0)).all())


def test_calls_from_several_threads():
    import threading
    x, w = rand(64, 512), 1 + 0.1 * rand(512, seed=1)
    lin = card_amd.QuantLinear(*weights(96, 512, 64, True), group=64)
    want = [card_amd.rms_norm(x, w), card_amd.dropout(x, 0.5, seed=3), lin(x)]
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = [card_amd.rms_norm(x, w), card_amd.dropout(x, 0.5, seed=3), lin(x)]
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_refusals_on_the_device():
    x = rand(4, 64)
    with pytest.raises(CardError, match="dtype"):
        card_amd.dropout(x.double(), 0.1, seed=1)
    with pytest.raises(CardError, match="outside"):
        card_amd.dropout(x, 1.5, seed=1)
    with pytest.raises(CardError, match="outside"):
        card_amd.dropout(x, float("nan"), seed=1)
    with pytest.raises(CardError, match="residual"):
        card_amd.dropout(x, 0.1, seed=1, n_z=2, residual=x)
    with pytest.raises(CardError, match="out of range"):
        card_amd.dropout(x, 0.1, seed=1, n_z=0)
    with pytest.raises(CardError, match="out of range"):
        card_amd.dropout(x, 0.1, seed=1, elem_offset=-1)
    with pytest.raises(CardError, match="two int64"):
        card_amd.dropout(x, 0.1, seed=torch.zeros(2, device=DEV))
    with pytest.raises(CardError, match="weight"):
        card_amd.rms_norm(x, rand(63))
    with pytest.raises(CardError, match="weight"):
        card_amd.rms_norm(x.half(), rand(64).bfloat16())
    with pytest.raises(CardError, match="residual"):
        card_amd.rms_norm(x, residual=x.half())
    with pytest.raises(CardError, match="eps"):
        card_amd.rms_norm(x, eps=-1.0)
    with pytest.raises(CardError, match=r"\(-2\)"):
        card_amd.rms_norm(torch.zeros(1, 65537, device=DEV))
    with pytest.raises(CardError, match="no backward"):
        card_amd.rms_norm_e4m3(x.clone().requires_grad_(True))
    q, s, z, b = weights(8, 64, 32, True)
    with pytest.raises(CardError, match="group"):
        card_amd.QuantLinear(q, s, z, b, group=16)
    with pytest.raises(CardError, match="scale is"):
        card_amd.QuantLinear(q, s, z, b, group=64)
    with pytest.raises(CardError, match="uint8"):
        card_amd.QuantLinear(q.int(), s, z, b, group=32)
    lin = card_amd.QuantLinear(q, s, z, b, group=32)
    with pytest.raises(CardError, match="expected"):
        lin(x[:, :63])
    with pytest.raises(CardError, match="x_scale"):
        lin(x, torch.ones(4, device=DEV))
    with pytest.raises(CardError, match="x_scale"):
        lin(x.to(torch.float8_e4m3fn))
    with pytest.raises(CardError, match="gamma"):
        lin(x, gamma=torch.ones(7, device=DEV))
    with pytest.raises(CardError, match="no backward"):
        lin(x.clone().requires_grad_(True))
    with pytest.raises(CardError, match=r"\(-2\)"):
        lin(torch.zeros(65536, 64, device=DEV))
    with pytest.raises(CardError, match="slope"):
        lin(x, slope=float("nan"))
    assert torch.isfinite(lin(x)).all()          # and the library still runs the valid call
