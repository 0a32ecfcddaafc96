"""The layer operators in 64 bits, from their formulas: what tests/test_gpu_layers.py and tests/test_layers_cpu.py compare with."""
import numpy as np
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}          # half a step, relative
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}      # half a subnormal step
U32 = 2.0 ** -24


def philox_words(blocks, seed, draw):
    """(n, 4) words of Philox4x32-10 (Salmon et al. 2011) at the counters (block lo, block hi, draw, 1); blocks: uint64."""
    m = np.uint64(0xFFFFFFFF)
    c = [blocks & m, blocks >> np.uint64(32), np.full_like(blocks, draw), np.ones_like(blocks)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & m, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1)


def keep_mask(n, p, seed, elem_offset=0, draw=0):
    e = np.arange(n, dtype=np.uint64) + np.uint64(elem_offset)
    first = int(elem_offset) >> 2
    last = (int(elem_offset) + max(n, 1) - 1) >> 2
    words = philox_words(np.arange(last - first + 1, dtype=np.uint64) + np.uint64(first), seed & (2 ** 64 - 1), draw)
    r = words[(e >> np.uint64(2)) - np.uint64(first), (e & np.uint64(3)).astype(np.int64)]
    return torch.from_numpy(r >= np.uint64(round(p * 2 ** 32)))


def dropout(x, p, *, seed, elem_offset=0, draw=0, n_z=1, residual=None):
    """(y, mask) in float64 on the CPU"""
    x = x.detach().cpu().double()
    shape = x.shape if n_z == 1 else x.shape[:-1] + (n_z, x.shape[-1])
    mask = keep_mask(int(np.prod(shape)), p, seed, elem_offset, draw).reshape(shape)
    xe = x if n_z == 1 else x.unsqueeze(-2).expand(shape)
    y = torch.where(mask, xe / (1 - p) if p < 1 else torch.zeros_like(xe), torch.zeros((), dtype=torch.float64))
    return (y if residual is None else y + residual.detach().cpu().double()), mask


def rms_norm(x, weight=None, residual=None, eps=1e-6):
    """(y, h) in float64 on the CPU"""
    h = x.detach().cpu().double()
    if residual is not None:
        h = h + residual.detach().cpu().double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return (y if weight is None else y * weight.detach().cpu().double()), h


def rms_norm_backward(h, weight, g, gh=None, eps=1e-6):
    """(dx, dweight, size of dx's terms, size of dweight's terms) in float64 on the CPU"""
    h, g = h.detach().cpu().double(), g.detach().cpu().double()
    w = torch.ones(h.shape[-1], dtype=torch.float64) if weight is None else weight.detach().cpu().double()
    n = h.shape[-1]
    rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    gw = g * w
    dx = rstd * gw - h * rstd ** 3 * (gw * h).sum(-1, keepdim=True) / n
    size = (rstd * gw).abs() + (h * rstd ** 3).abs() * (gw * h).abs().sum(-1, keepdim=True) / n
    if gh is not None:
        dx = dx + gh.detach().cpu().double()
        size = size + gh.detach().cpu().double().abs()
    unit = (h * rstd * g).reshape(-1, n)
    return dx, unit.sum(0), size, unit.abs().sum(0)


def linear4(q, scale, zero, bias, group, x, x_scale=None, gamma=None, slope=None):
    """(y, size) in float64 on the CPU; size: the sum of the products' magnitudes with 16 added to each of q and zero, as
    kernels hold them on the way"""
    q, s, x = q.cpu().double(), scale.cpu().double(), x.detach().cpu().float().double()
    at = torch.arange(q.shape[1]) // group
    z = torch.full_like(s, 8.0) if zero is None else zero.cpu().double()
    w = (q - z[:, at]) * s[:, at]
    size = x.abs() @ ((q + z[:, at] + 32) * s[:, at].abs()).t()
    y = x @ w.t()
    if x_scale is not None:
        y, size = y * x_scale.cpu().double().unsqueeze(-1), size * x_scale.cpu().double().abs().unsqueeze(-1)
    if bias is not None:
        y, size = y + bias.cpu().double(), size + bias.cpu().double().abs()
    if gamma is not None:
        y, size = y * gamma.cpu().double(), size * gamma.cpu().double().abs()
    if slope is not None:
        y = torch.where(y > 0, y, y * slope)
    return y, size


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound element by element (float64), and NaN / infinities alike"""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    d = (got - want).abs()[fine]
    b = (bound if torch.is_tensor(bound) else torch.full_like(want, bound)).expand(want.shape)[fine]
    if d.numel():
        worst = int((d - b).argmax())
        assert bool((d <= b).all()), (what, "worst", float(d[worst]), "allowed", float(b[worst]), "value", float(want[fine][worst]))
