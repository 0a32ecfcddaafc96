"""The guidance network f_phi with the layer operators: Monte-Carlo dropout (GuidanceNet.mc_dropout) and 4-bit weights
(GuidanceNet.from_module(..., weight_bits=4)), against the formulas in 64 bits; and the 4-bit network inside a sampling call.

Tolerances follow the errors through the layers: `forward64` returns with each value the sum of the magnitudes that it was
added from, and a 32-bit network is off by at most the roundings on the way times that (each layer adds in + 4 of them)."""
import pytest
import torch
from torch import nn

import card_amd
from card_amd._lib import CardError
from card_amd.guidance import GuidanceNet, QuantGuidanceNet
from card_amd.sampler import Sampler, make_coef_table
from card_amd.synth import guided_state_dict, make_schedule
from tests import layer_reference as ref
from tests.test_gpu_parity import RefShapedGuided
from tests.layer_reference import U32, assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def network(dims, *, bn=False, norm=False, p=0.2, slope=0.01, seed=0):
    """The layout of regression/model.py:70-79, with RMSNorm ahead of the Linear layers where norm"""
    torch.manual_seed(seed)
    layers = []
    for i, (a, b) in enumerate(zip(dims, dims[1:])):
        if norm:
            layers.append(nn.RMSNorm(a, eps=1e-6))
            nn.init.normal_(layers[-1].weight, 1.0, 0.2)
        layers.append(nn.Linear(a, b))
        if i < len(dims) - 2:
            if bn:
                layers.append(nn.BatchNorm1d(b))
                layers[-1].running_mean.normal_(0, 0.3)
                layers[-1].running_var.uniform_(0.5, 1.5)
                nn.init.uniform_(layers[-1].weight, 0.5, 1.5)
            layers += [nn.LeakyReLU(slope), nn.Dropout(p)]
    return nn.Sequential(*layers).eval()


def forward64(net, x, n_z, seed, chain_offset=0, quant=None, drop=True):
    """(y, size) (rows, n_z, out) in float64: the modules one by one; quant: the dequantised (weight, bias) of each Linear"""
    rows = x.shape[0]
    h = x.cpu().double().repeat_interleave(n_z, 0)
    size, layer, fold = h.abs(), -1, None
    for m in net:
        if isinstance(m, nn.RMSNorm):
            raise AssertionError("networks with norms are compared layer by layer")
        if isinstance(m, nn.Linear):
            layer += 1
            W, b = (m.weight.detach().cpu().double(), m.bias.detach().cpu().double()) if quant is None else quant[layer]
            h, size = h @ W.t() + b, size @ W.abs().t() + b.abs()
            fold = quant is not None
        elif isinstance(m, nn.BatchNorm1d) and not fold:
            s = m.weight.detach().cpu().double() / torch.sqrt(m.running_var.cpu().double() + m.eps)
            t = m.bias.detach().cpu().double() - m.running_mean.cpu().double() * s
            h, size = h * s + t, size * s.abs() + t.abs()
        elif isinstance(m, nn.LeakyReLU):
            h = torch.where(h > 0, h, h * m.negative_slope)
        elif isinstance(m, nn.Dropout) and drop and m.p > 0:
            keep = ref.keep_mask(h.numel(), m.p, seed, chain_offset * h.shape[1], draw=layer).reshape(h.shape)
            h, size = torch.where(keep, h / (1 - m.p), torch.zeros((), dtype=torch.float64)), torch.where(keep, size / (1 - m.p), torch.zeros((), dtype=torch.float64))
    return h.reshape(rows, n_z, -1), size.reshape(rows, n_z, -1)


def roundings(dims, extra=0):
    return sum(d + 8 + extra for d in dims[:-1])


@pytest.mark.parametrize("dims,bn", [([13, 100, 50, 1], False), ([90, 100, 50, 1], True), ([1, 7, 3], False), ([5, 2], False), ([9, 33, 64, 17, 4], True)])
@pytest.mark.parametrize("rows,n_z,offset", [(1, 1, 0), (7, 5, 0), (33, 16, 100), (3, 200, 2 ** 30 + 1)])
def test_mc_dropout_fp32(dims, bn, rows, n_z, offset):
    net = network(dims, bn=bn)
    x = torch.randn(rows, dims[0], generator=torch.Generator().manual_seed(1))
    want, size = forward64(net, x, n_z, 77, offset)
    g = GuidanceNet.from_module(net.to(DEV))
    got = g.mc_dropout(x.to(DEV), n_z, seed=77, chain_offset=offset)
    assert_within(got, want, roundings(dims) * U32 * size + 1e-30)
    # rows of a shard are the whole call's
    if rows > 2:
        assert torch.equal(g.mc_dropout(x[2:].to(DEV), n_z, seed=77, chain_offset=offset + 2 * n_z), got[2:])
    if len(dims) > 2 and rows * n_z > 60:
        assert not torch.equal(got, g.mc_dropout(x.to(DEV), n_z, seed=78, chain_offset=offset))
    # eval mode is what it was
    assert torch.equal(g.forward(x.to(DEV)), GuidanceNet.from_module(net).forward(x.to(DEV)))


def dequantised(net, group):
    """The (weight, bias) in float64 that QuantGuidanceNet's layers hold, from the same folding and quantisation"""
    out, mods = [], list(net)
    for i, m in enumerate(mods):
        if not isinstance(m, nn.Linear):
            continue
        W, b = m.weight.detach().float(), m.bias.detach().float()
        if i + 1 < len(mods) and isinstance(mods[i + 1], nn.BatchNorm1d):
            n = mods[i + 1]
            s = n.weight.detach() / torch.sqrt(n.running_var + n.eps)
            t = n.bias.detach() - n.running_mean * s
            W, b = W * s[:, None], b * s + t
        q, sc, z = card_amd.quantize_weight(W, group=group)
        at = torch.arange(W.shape[1]) // group
        out.append(((q.cpu().double() - z.cpu().double()[:, at]) * sc.cpu().double()[:, at], b.cpu().double()))
    return out


@pytest.mark.parametrize("dims,bn,group", [([13, 100, 50, 1], False, 64), ([90, 300, 2000, 40, 3], True, 128), ([5, 2], False, 32), ([1500, 1100, 1], False, 32)])
@pytest.mark.parametrize("rows,n_z", [(1, 1), (9, 7), (40, 3)])
def test_4bit_network(dims, bn, group, rows, n_z):
    net = network(dims, bn=bn).to(DEV)
    x = torch.randn(rows, dims[0], generator=torch.Generator().manual_seed(1)).to(DEV)
    g = GuidanceNet.from_module(net, weight_bits=4, group=group)
    assert isinstance(g, QuantGuidanceNet)
    quant = dequantised(net, group)
    # on the way the kernel's sums hold 16 + q and 16 + zero: at most 62 steps a weight, and a step is at most its row's largest weight
    for drop in (False, True):
        want, size = forward64(net, x, n_z, 5, 0, [(w, b) for w, b in quant], drop)
        big = forward64(net, x.abs(), n_z, 5, 0, [(w.abs() + 62 * step(w), b.abs()) for w, b in quant], drop)[0].abs()
        got = g.mc_dropout(x, n_z, seed=5) if drop else g.forward(x)[:, None, :].expand(rows, n_z, dims[-1])
        assert_within(got, want, roundings(dims) * U32 * big + 1e-30)


def step(w):
    """an upper bound of a row's quantisation step: its largest magnitude (q - zero is a whole number, so 1 of it or more)"""
    return w.abs().amax(1, keepdim=True).expand_as(w)


def test_4bit_network_with_norms_is_its_layers():
    dims, group = [200, 320, 96, 5], 32
    net = network(dims, norm=True).to(DEV)
    x = torch.randn(11, 200, generator=torch.Generator().manual_seed(1)).to(DEV)
    g = GuidanceNet.from_module(net, weight_bits=4, group=group)
    h, lins, norms = x, [m for m in net if isinstance(m, nn.Linear)], [m for m in net if isinstance(m, nn.RMSNorm)]
    for l, (lin, norm) in enumerate(zip(lins, norms)):
        q, s = card_amd.rms_norm_e4m3(h, norm.weight.detach(), eps=1e-6)
        h = card_amd.QuantLinear.from_float(lin.weight.detach(), lin.bias.detach(), group=group).forward(q, s, slope=0.01 if l < 2 else None, out_dtype=torch.float32)
    assert torch.equal(g.forward(x), h)
    # and near the module itself: 4-bit weights and 8-bit rows, a sanity bound on a network of order one
    with torch.no_grad():
        full = net(x)
    assert float((h - full).norm() / full.norm()) < 0.5
    with pytest.raises(CardError, match="weight_bits=4 only"):
        GuidanceNet.from_module(net)


def test_4bit_network_in_a_sampling_call():
    T, x_dim, n_z = 20, 13, 6
    net = network([13, 100, 50, 1]).to(DEV)
    s = Sampler.from_state_dict(guided_state_dict(x_dim, T), device=DEV)
    alphas, _, omabs = make_schedule("linear", T, 1e-4, 0.02)
    coef = make_coef_table(alphas, omabs).to(DEV)
    x = torch.randn(30, x_dim, generator=torch.Generator().manual_seed(2)).to(DEV)
    g = GuidanceNet.from_module(net, weight_bits=4)
    got = s.run(x, None, None, coef, T, seed=3, n_z=n_z, fphi=g)
    y0 = g.forward(x)
    assert torch.equal(s.last_y_0_hat, y0)
    assert torch.equal(got, s.run(x, y0, y0, coef, T, seed=3, n_z=n_z))
    assert s.run(x, None, None, coef, T, seed=3, n_z=n_z, fphi=g, plan=True)["launches"] >= 1
    model = RefShapedGuided(guided_state_dict(x_dim, T), True, True).to(DEV).eval()
    _, y0b = card_amd.p_sample_loop_from_x(model, g, x, T, alphas.to(DEV), omabs.to(DEV), n_z=n_z, only_last_sample=True, seed=3)
    assert torch.equal(y0b, y0)
    # the fp32 network is as before
    f = GuidanceNet.from_module(net)
    assert torch.equal(s.run(x, None, None, coef, T, seed=3, n_z=n_z, fphi=f), s.run(x, f.forward(x), f.forward(x), coef, T, seed=3, n_z=n_z))


def test_refusals():
    net = network([13, 20, 1]).to(DEV)
    x = torch.zeros(2, 13, device=DEV)
    g, q = GuidanceNet.from_module(net), GuidanceNet.from_module(net, weight_bits=4)
    for f in (g, q):
        with pytest.raises(CardError, match="x must be"):
            f.mc_dropout(x[:, :5], 3, seed=1)
        with pytest.raises(CardError, match="out of range"):
            f.mc_dropout(x, 0, seed=1)
        with pytest.raises(CardError, match="out of range"):
            f.mc_dropout(x, 1, seed=1, chain_offset=-1)
        assert f.mc_dropout(x[:0], 3, seed=1).shape == (0, 3, 1) and f.forward(x[:0]).shape == (0, 1)
    with pytest.raises(CardError, match="weight_bits=8"):
        GuidanceNet.from_module(net, weight_bits=8)
    with pytest.raises(CardError, match="group"):
        GuidanceNet.from_module(net, weight_bits=4, group=48)
    odd = nn.Sequential(nn.Dropout(0.5), nn.Linear(13, 4), nn.LeakyReLU(), nn.Linear(4, 1)).to(DEV).eval()
    with pytest.raises(CardError, match="Dropout"):
        GuidanceNet.from_module(odd).mc_dropout(x, 2, seed=1)
    with pytest.raises(CardError, match="Dropout"):
        GuidanceNet.from_ols(torch.zeros(14, 1, device=DEV)).mc_dropout(x, 2, seed=1)
    wide = network([13, 1025, 1]).to(DEV)          # past the fp32 kernel's width, not past the 4-bit layers'
    with pytest.raises(CardError, match="1024"):
        GuidanceNet.from_module(wide)
    assert torch.isfinite(GuidanceNet.from_module(wide, weight_bits=4).forward(x)).all()
    with pytest.raises(CardError, match="out of range"):          # elements are counted in 63 bits
        GuidanceNet.from_module(network([13, 3000, 1]).to(DEV), weight_bits=4).mc_dropout(x, 2, seed=1, chain_offset=2 ** 52 - 1)
