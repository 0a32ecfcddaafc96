"""What card_amd.describe_guidance takes a Sequential for, without a GPU: what it accepts, the description computes."""
import pytest
import torch
from torch import nn

from card_amd._lib import CardError
from card_amd.guidance import _bn_fold, _settings, describe_guidance


def evaluate(d, x):
    """The network that a description stands for, in float64"""
    h = x
    for l, (W, b, bn, norm) in enumerate(zip(d["weights"], d["biases"], d["batchnorm"], d["norms"])):
        if norm is not None:
            h = norm(h)
        h = nn.functional.linear(h, W, b)
        if bn is not None:
            s, t = _bn_fold(bn)
            h = h * s + t
        if l < len(d["weights"]) - 1:
            h = torch.where(h > 0, h, d["negative_slope"] * h)
    return h


def lin(a=4, b=4):
    return nn.Linear(a, b)


def bn():
    m = nn.BatchNorm1d(4)
    m.running_mean.normal_(0, 0.3)
    m.running_var.uniform_(0.5, 1.5)
    nn.init.uniform_(m.weight, -1.5, 1.5)
    return m


ACCEPTED = {
    "one layer": lambda: [lin()],
    "the reference's order": lambda: [lin(), bn(), nn.LeakyReLU(0.1), nn.Dropout(0.2), lin(), bn(), nn.LeakyReLU(0.1), nn.Dropout(0.2), lin(4, 1)],
    "relu": lambda: [lin(), nn.ReLU(), lin(), nn.ReLU(), nn.ReLU(), lin()],
    "leaky of slope 0 and relu": lambda: [lin(), nn.LeakyReLU(0.0), lin(), nn.ReLU(), lin()],
    "slope 1": lambda: [lin(), nn.LeakyReLU(1.0), lin()],
    "dropout ahead of the activation": lambda: [lin(), nn.Dropout(0.3), nn.LeakyReLU(0.1), lin(), nn.Dropout(0.5)],
    "dropout ahead of BatchNorm": lambda: [lin(), nn.Dropout(0.3), bn(), nn.LeakyReLU(0.1), lin()],
    "identities": lambda: [nn.Identity(), lin(), nn.Identity(), nn.LeakyReLU(0.1), nn.Identity(), lin(), nn.Identity()],
    "norms": lambda: [nn.RMSNorm(4), lin(), bn(), nn.LeakyReLU(0.1), nn.RMSNorm(4), lin()],
}
REFUSED = {
    "BatchNorm behind the activation": lambda: [lin(), nn.LeakyReLU(), bn(), lin()],
    "BatchNorm behind activation and Dropout": lambda: [lin(), nn.ReLU(), nn.Dropout(0.1), bn(), lin()],
    "no activation between two Linear layers": lambda: [lin(), lin()],
    "no activation behind BatchNorm": lambda: [lin(), bn(), lin()],
    "only Dropout between two Linear layers": lambda: [lin(), nn.LeakyReLU(), lin(), nn.Dropout(0.1), lin()],
    "an activation behind the output": lambda: [lin(), nn.LeakyReLU(), lin(), nn.LeakyReLU()],
    "ReLU behind the only layer": lambda: [lin(), nn.ReLU()],
    "an activation ahead of the first layer": lambda: [nn.LeakyReLU(), lin(), nn.LeakyReLU(), lin()],
    "two activations": lambda: [lin(), nn.LeakyReLU(0.1), nn.LeakyReLU(0.1), lin()],
    "different slopes": lambda: [lin(), nn.LeakyReLU(0.1), lin(), nn.LeakyReLU(0.2), lin()],
    "LeakyReLU and ReLU": lambda: [lin(), nn.LeakyReLU(0.1), lin(), nn.ReLU(), lin()],
    "ReLU and LeakyReLU": lambda: [lin(), nn.ReLU(), lin(), nn.LeakyReLU(0.1), lin()],
}


@pytest.mark.parametrize("name", ACCEPTED)
def test_a_description_computes_its_module(name):
    torch.manual_seed(0)
    net = nn.Sequential(*ACCEPTED[name]()).double().eval()
    x = torch.randn(50, 4, dtype=torch.float64)
    with torch.no_grad():
        assert torch.allclose(evaluate(describe_guidance(net), x), net(x), rtol=1e-12, atol=1e-13)


@pytest.mark.parametrize("name", REFUSED)
def test_orders_that_the_networks_do_not_compute_are_refused(name):
    with pytest.raises(CardError, match="f_phi"):
        describe_guidance(nn.Sequential(*REFUSED[name]()).eval())


def test_settings_are_numbers():
    """A module of another kind around the network may hold anything under these names."""
    net = nn.Sequential(*ACCEPTED["the reference's order"]()).eval()
    net.eps, net.p = torch.ones(3), nn.Linear(2, 2)
    assert _settings(net) == _settings(net)
    before = _settings(net)
    net[3].p = 0.3
    assert _settings(net) != before
