"""The guidance network on the device at the edges: what its cache notices, its layers one by one, its masks under chain offsets."""
import copy

import pytest
import torch
from torch import nn

import card_amd
from card_amd._lib import CardError
from card_amd.guidance import GuidanceNet, guidance_for
from tests import layer_reference as ref
from tests.layer_reference import TINY, U32, assert_within
from tests.test_gpu_guidance_layers import network
from tests.test_gpu_layers import DEV, lin_bound

pytestmark = pytest.mark.gpu


def test_cached_guidance_follows_the_modules_numbers():
    """Dropout rates, slopes and BatchNorm's eps are part of the network as its weights are."""
    net = network([6, 20, 10, 1], bn=True).to(DEV)
    x = torch.randn(8, 6, generator=torch.Generator().manual_seed(1)).to(DEV)
    first = guidance_for(net)
    assert guidance_for(net) is first

    def change(kind, **kw):
        for m in net:
            if isinstance(m, kind):
                for k, v in kw.items():
                    setattr(m, k, v)
    for kind, kw in ((nn.Dropout, dict(p=0.5)), (nn.LeakyReLU, dict(negative_slope=0.3)), (nn.BatchNorm1d, dict(eps=0.2))):
        before = guidance_for(net)
        change(kind, **kw)
        now, fresh = guidance_for(net), GuidanceNet.from_module(copy.deepcopy(net))
        assert now is not before and guidance_for(net) is now
        assert torch.equal(now(x), fresh(x)) and torch.equal(now.mc_dropout(x, 20, seed=1), fresh.mc_dropout(x, 20, seed=1))
        assert not torch.equal(now.mc_dropout(x, 20, seed=1), before.mc_dropout(x, 20, seed=1))
    # modules that hold no tensors, and train mode of a part
    net[2] = nn.ReLU()
    with pytest.raises(CardError, match="slopes"):
        guidance_for(net)
    net[2] = nn.LeakyReLU(0.3)
    now = guidance_for(net)
    net[1].train()
    with pytest.raises(CardError, match="eval mode"):
        guidance_for(net)
    net[1].eval()
    assert torch.equal(guidance_for(net)(x), now(x))


def folded64(net):
    """Each Linear's (weight, bias) in float64 with the BatchNorm behind it"""
    out, mods = [], list(net)
    for i, m in enumerate(mods):
        if isinstance(m, nn.Linear):
            W, b = m.weight.detach().cpu().double(), m.bias.detach().cpu().double()
            if i + 1 < len(mods) and isinstance(mods[i + 1], nn.BatchNorm1d):
                n = mods[i + 1]
                s = n.weight.detach().cpu().double() / torch.sqrt(n.running_var.cpu().double() + n.eps)
                W, b = W * s[:, None], (b - n.running_mean.cpu().double()) * s + n.bias.detach().cpu().double()
            out.append((W, b))
    return out


def walk(net, g, x, n_z, seed, chain_offset, group, rates):
    """g.mc_dropout by its layers, each compared with its formula on the values that it was given"""
    rows, h, chains = x.shape[0], x, 1
    for l, ((W, b), (_, _, _, lin)) in enumerate(zip(folded64(net), g.layers)):
        last = l == len(g.layers) - 1
        # the weights that the layer holds: half a step of their group from the folded ones
        q, s, z = card_amd.quantize_weight(W.float().to(DEV), group=group)
        at = torch.arange(W.shape[1]) // group
        step = s.cpu().double()[:, at]
        eye = torch.eye(W.shape[1], device=DEV)
        held = torch.cat([lin.forward(part, out_dtype=torch.float32) for part in eye.split(1024)]).cpu().double().t()          # + bias, rounded once
        assert bool(((held - b[:, None] - W).abs() <= 0.51 * step + 64 * U32 * (W.abs() + b.abs()[:, None] + 32 * step)).all()), l
        y = lin.forward(h, slope=None if last else 0.01, out_dtype=torch.float32)
        want = h.cpu().double() @ ((q.cpu().double() - z.cpu().double()[:, at]) * step).t() + b
        size = h.cpu().double().abs() @ ((q.cpu().double() + z.cpu().double()[:, at] + 32) * step).t() + b.abs()
        # 4-bit values next to a border may go either way between the two foldings: a step of those columns at most
        flips = h.cpu().double().abs() @ (step * near_border(W, s, z, at)).t()
        if not last:
            want = torch.where(want > 0, want, 0.01 * want)
        assert_within(y, want, lin_bound(want, size, group, W.shape[1], torch.float32) + 8 * U32 * size + flips, ("layer", l))
        h = y
        if not last and rates[l] > 0:
            nz, chains = (n_z, n_z) if chains == 1 else (1, chains)
            wide = h if nz == 1 else h[:, None, :].expand(rows, nz, h.shape[1])
            wide = wide.reshape(rows * chains, h.shape[1])
            keep = ref.keep_mask(wide.numel(), rates[l], seed, chain_offset * wide.shape[1], draw=l).reshape(wide.shape)
            d = card_amd.dropout(h, rates[l], seed=seed, elem_offset=chain_offset * h.shape[1], draw=l, n_z=nz).reshape(wide.shape)
            want = torch.where(keep, wide.cpu().double() / (1 - rates[l]), torch.zeros((), dtype=torch.float64))
            assert_within(d, want, 3 * U32 * want.abs() + TINY[torch.float32], ("dropout", l))
            h = d
    return h.reshape(rows, chains, -1).expand(rows, n_z, h.shape[1])


def near_border(W, s, z, at):
    """1 where w / scale is within 2^-18 of a rounding border"""
    r = (W / s.cpu().double()[:, at].clamp_min(1e-300)) % 1
    return ((r - 0.5).abs() < 2.0 ** -18).double()


@pytest.mark.parametrize("dims,bn,group,rates", [([13, 100, 50, 1], False, 64, (0.2, 0.2)), ([90, 300, 2000, 40, 3], True, 128, (0.5, 0.1, 0.2)),
                                                  ([1500, 1100, 1], False, 32, (0.3,)), ([20, 33, 65, 7], True, 32, (0.0, 0.4))])
@pytest.mark.parametrize("rows,n_z,offset", [(1, 1, 0), (9, 7, 0), (5, 12, 1001), (3, 40, 2 ** 40 + 3)])
def test_4bit_network_layer_by_layer(dims, bn, group, rates, rows, n_z, offset):
    net = network(dims, bn=bn)
    for m, p in zip([m for m in net if isinstance(m, nn.Dropout)], rates):
        m.p = p
    net = net.to(DEV)
    x = torch.randn(rows, dims[0], generator=torch.Generator().manual_seed(1)).to(DEV)
    g = GuidanceNet.from_module(net, weight_bits=4, group=group)
    got = g.mc_dropout(x, n_z, seed=5, chain_offset=offset)
    assert torch.equal(got, walk(net, g, x, n_z, 5, offset, group, rates))
    assert torch.equal(g.forward(x), walk(net, g, x, 1, 5, offset, group, (0.0,) * len(rates))[:, 0])
    if rows * n_z >= 60:          # other numbers, other masks
        assert not torch.equal(got, g.mc_dropout(x, n_z, seed=6, chain_offset=offset))
        assert not torch.equal(got, g.mc_dropout(x, n_z, seed=5, chain_offset=offset + 1))
        assert not torch.equal(got, g.forward(x)[:, None, :].expand_as(got))


def test_4bit_mc_dropout_of_shards_and_of_many_chains():
    """Rows of a shard are the whole call's, also where the call is cut at 65535 chains (twice here)."""
    net = network([13, 100, 50, 2]).to(DEV)
    g = GuidanceNet.from_module(net, weight_bits=4)
    x = torch.randn(1400, 13, generator=torch.Generator().manual_seed(1)).to(DEV)
    whole = g.mc_dropout(x, 100, seed=9, chain_offset=12345)
    assert tuple(whole.shape) == (1400, 100, 2)
    for a, b in ((0, 20), (640, 700), (1300, 1400)):
        assert torch.equal(g.mc_dropout(x[a:b], 100, seed=9, chain_offset=12345 + a * 100), whole[a:b])
    f = GuidanceNet.from_module(net)          # the same masks as the fp32 network's: its outputs are near
    assert float((whole - f.mc_dropout(x, 100, seed=9, chain_offset=12345)).norm() / whole.norm()) < 0.3 * float((whole - f.mc_dropout(x, 100, seed=10)).norm() / whole.norm())
    rows = torch.randn(70000, 13, generator=torch.Generator().manual_seed(2)).to(DEV)
    y = g.forward(rows)
    assert torch.equal(y[65500:65600], g.forward(rows[65500:65600]))
