"""The guidance network on the device at the edges: what its cache notices, its layers one by one, its masks under chain offsets."""
import copy

import pytest
import torch
from torch import nn

from card_amd._lib import CardError
from card_amd.guidance import GuidanceNet, guidance_for
from tests.test_gpu_guidance_layers import network
from tests.test_gpu_layers import DEV

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
