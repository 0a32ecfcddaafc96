"""Who owns a packed network (card_amd._lib.Handle), without a GPU: the objects here hold handles of nothing."""
import copy
import ctypes as C
import gc
import pickle

import pytest

from card_amd import _lib
from card_amd._lib import CardError
from card_amd.guidance import GuidanceNet, QuantGuidanceNet
from card_amd.layers import QuantLinear
from card_amd.sampler import Sampler


def owner(cls, gone):
    o = object.__new__(cls)
    o._h = _lib.Handle(4096, lambda h: gone.append(h.value))
    return o


@pytest.mark.parametrize("cls", [QuantLinear, GuidanceNet, Sampler])
def test_a_shallow_copy_keeps_the_weights(cls):
    gone = []
    a = owner(cls, gone)
    b = copy.copy(a)
    assert b._h is a._h and a._h.value == 4096
    del a
    gc.collect()
    assert gone == []
    del b
    gc.collect()
    assert gone == [4096]


@pytest.mark.parametrize("cls", [QuantLinear, GuidanceNet, Sampler])
def test_deep_copies_and_pickles_are_refused(cls):
    gone = []
    a = owner(cls, gone)
    net = object.__new__(QuantGuidanceNet)
    net._h, net.layers = None, [(False, None, 0.0, a)]
    for what in (a, net, [a], {"g": net}):
        for how in (copy.deepcopy, pickle.dumps, lambda o: pickle.dumps(o, protocol=2)):
            with pytest.raises(CardError, match="pack them again"):
                how(what)
    copy.copy(net)
    del net, what, a
    gc.collect()
    assert gone == [4096]


def test_a_handle_is_a_pointer_to_the_library():
    gone = []
    h = _lib.Handle(4096, lambda h: gone.append(h.value))
    a = _lib.RunArgs()
    a.fphi = h
    assert a.fphi == 4096 and C.c_void_p.from_param(h) is h
