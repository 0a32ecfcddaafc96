"""The layer operators without a GPU: what their C entry points refuse before they touch a device, what the Python functions
say to CPU tensors, and the test's own 64-bit formulas against torch."""
import ctypes as C

import pytest
import torch

import card_amd
from card_amd import _lib
from card_amd._lib import CardError
from tests import layer_reference as ref

E_INVALID, E_UNSUPPORTED = -1, -2
P = 4096          # an address that is never dereferenced


def msg():
    return _lib.lib().card_last_error().decode()


@pytest.mark.parametrize("change,code,needle", [
    (dict(dtype=7), E_INVALID, "dtype"), (dict(dtype=_lib.DTYPE_E4M3), E_INVALID, "dtype"), (dict(rows=-1), E_INVALID, "rows"), (dict(cols=-1), E_INVALID, "cols"),
    (dict(n_z=0), E_INVALID, "n_z"), (dict(p=-0.1), E_INVALID, "p="), (dict(p=1.1), E_INVALID, "p="), (dict(p=float("nan")), E_INVALID, "p="),
    (dict(draw=-1), E_INVALID, "draw"), (dict(elem_offset=1 << 63), E_INVALID, "elem_offset"), (dict(x=None), E_INVALID, "null"), (dict(out=None), E_INVALID, "null"),
    (dict(rows=1 << 40, cols=1 << 30), E_INVALID, "63 bits"), (dict(rows=1 << 30, cols=1 << 20, n_z=1 << 5), E_UNSUPPORTED, "workgroups"),
    (dict(rows=1 << 24, cols=1 << 10), E_UNSUPPORTED, "workgroups"), (dict(dtype=2, rows=1 << 25, cols=1 << 10), E_UNSUPPORTED, "workgroups"),
])
def test_dropout_refusals(change, code, needle):
    L = _lib.lib()
    a = dict(x=P, out=P, dtype=0, rows=4, cols=4, n_z=1, p=0.5, elem_offset=0, draw=0)
    a.update(change)
    tail = (a["dtype"], a["rows"], a["cols"], a["n_z"], a["p"], 1, a["elem_offset"], None, a["draw"], None)
    assert L.card_dropout(a["x"], None, a["out"], *tail) == code and needle in msg(), msg()
    if "workgroups" not in needle:          # backward takes a workgroup per chunk of x, not of the masks
        assert L.card_dropout_backward(a["x"], a["out"], *tail) == code and needle in msg(), msg()


def test_dropout_backward_of_many_short_rows_is_refused():
    """A thread for each 16 bytes of dx and no fewer than one to a row: 2^32 of them are no launch."""
    L = _lib.lib()
    assert L.card_dropout_backward(P, P, _lib.DTYPE_BF16, 1 << 32, 1, 2, 0.5, 1, 0, None, 0, None) == E_UNSUPPORTED and "workgroups" in msg(), msg()


def test_nothing_to_do_is_no_error():
    L = _lib.lib()
    assert L.card_dropout(None, None, None, 0, 0, 5, 1, 0.5, 1, 0, None, 0, None) == 0
    assert L.card_dropout_backward(None, None, 1, 5, 0, 3, 0.5, 1, 0, None, 0, None) == 0
    assert L.card_rms_norm(None, None, None, 0, 0, 0, 8, 1e-6, None, None, 0, None, None) == 0
    assert L.card_rms_norm_backward(None, None, None, None, 0, 0, 0, 8, 1e-6, None, None, None, 0, None) == 0


@pytest.mark.parametrize("change,code,needle", [
    (dict(dtype=3), E_INVALID, "dtype"), (dict(dtype=1, wt=2), E_INVALID, "weight dtype"), (dict(rows=-1), E_INVALID, "rows"), (dict(cols=0), E_INVALID, "cols"),
    (dict(cols=_lib.NORM_MAX_COLS + 1), E_UNSUPPORTED, "cols"), (dict(eps=-1.0), E_INVALID, "eps"), (dict(eps=float("nan")), E_INVALID, "eps"), (dict(eps=float("inf")), E_INVALID, "eps"),
    (dict(x=None), E_INVALID, "null"), (dict(y=None), E_INVALID, "null"), (dict(residual=P), E_INVALID, "residual and h"), (dict(h=P), E_INVALID, "residual and h"),
    (dict(yt=1), E_INVALID, "y_dtype"), (dict(yt=3), E_INVALID, "scale"), (dict(scale=P), E_INVALID, "scale"), (dict(rows=1 << 60), E_INVALID, "63 bits"),
])
def test_rms_norm_refusals(change, code, needle):
    a = dict(x=P, residual=None, w=P, dtype=0, wt=0, rows=4, cols=8, eps=1e-6, h=None, y=P, yt=0, scale=None)
    a.update(change)
    assert _lib.lib().card_rms_norm(a["x"], a["residual"], a["w"], a["dtype"], a["wt"], a["rows"], a["cols"], a["eps"], a["h"], a["y"],
                                    a["yt"], a["scale"], None) == code and needle in msg(), msg()


def test_rms_norm_backward_refusals():
    L = _lib.lib()
    n = C.c_uint64()
    assert L.card_rms_norm_backward_workspace_bytes(0, 100, 300, C.byref(n)) == 0 and 300 * 4 <= n.value <= 100 * 300 * 4
    need = n.value
    assert L.card_rms_norm_backward_workspace_bytes(0, 100, 300, None) == E_INVALID
    call = lambda h=P, w=P, dx=P, dw=P, ws=P, nb=need: L.card_rms_norm_backward(h, w, P, None, 0, 0, 100, 300, 1e-6, dx, dw, ws, nb, None)  # noqa: E731
    assert call(h=None) == E_INVALID and "null" in msg()
    assert call(dx=None) == E_INVALID and "null" in msg()
    assert call(w=None) == E_INVALID and "without a weight" in msg()
    assert call(ws=None) == E_INVALID and "workspace" in msg()
    assert call(nb=need - 1) == E_INVALID and "workspace" in msg()
    assert call(ws=P + 8) == E_INVALID and "aligned" in msg()


@pytest.mark.parametrize("change,code,needle", [
    (dict(struct_bytes=8), E_INVALID, "struct_bytes"), (dict(in_features=0), E_INVALID, "features"), (dict(out_features=-3), E_INVALID, "features"),
    (dict(in_features=_lib.LINEAR4_MAX_FEATURES + 1), E_UNSUPPORTED, "at most"), (dict(group=16), E_UNSUPPORTED, "group"), (dict(group=256), E_UNSUPPORTED, "group"),
    (dict(q=None), E_INVALID, "null"), (dict(scale=None), E_INVALID, "null"),
])
def test_linear4_create_refusals(change, code, needle):
    d = _lib.Linear4Desc()
    d.struct_bytes, d.in_features, d.out_features, d.group, d.q, d.scale = C.sizeof(_lib.Linear4Desc), 64, 64, 32, P, P
    for k, v in change.items():
        setattr(d, k, v)
    h = C.c_void_p(1)
    assert _lib.lib().card_linear4_create(C.byref(d), None, C.byref(h)) == code and needle in msg() and not h.value


def test_linear4_other_refusals():
    L = _lib.lib()
    h = C.c_void_p()
    assert L.card_linear4_create(None, None, C.byref(h)) == E_INVALID
    assert L.card_linear4_forward(None, P, 0, None, 1, None, 1.0, P, 0, None, 0, None) == E_INVALID and "null handle" in msg()
    assert L.card_linear4_quantize(P, 4, 4, 48, P, P, P, None) == E_UNSUPPORTED
    assert L.card_linear4_quantize(P, 0, 4, 32, P, P, P, None) == E_INVALID
    assert L.card_linear4_quantize(None, 4, 4, 32, P, P, P, None) == E_INVALID
    n = C.c_uint64()
    assert L.card_linear4_workspace_bytes(None, 0, 1, C.byref(n)) == E_INVALID and "null" in msg()
    L.card_linear4_destroy(None)


def test_desc_layout(tmp_path):
    import os
    import subprocess
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "card_hip.h"\nint main(void){printf("%zu %zu %zu %d %d %d %d\\n", sizeof(card_linear4_desc),'
                   ' offsetof(card_linear4_desc, q), offsetof(card_linear4_desc, bias), CARD_DTYPE_E4M3, CARD_NORM_MAX_COLS, CARD_LINEAR4_MAX_FEATURES,'
                   ' CARD_LINEAR4_MAX_ROWS); return 0;}\n')
    exe = tmp_path / "sz"
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    D = _lib.Linear4Desc
    assert got == [C.sizeof(D), D.q.offset, D.bias.offset, _lib.DTYPE_E4M3, _lib.NORM_MAX_COLS, _lib.LINEAR4_MAX_FEATURES, _lib.LINEAR4_MAX_ROWS]


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 32)
    for call in (lambda: card_amd.dropout(x, 0.1, seed=1), lambda: card_amd.rms_norm(x), lambda: card_amd.rms_norm_e4m3(x),
                 lambda: card_amd.quantize_weight(x),
                 lambda: card_amd.QuantLinear(torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1), group=32)):
        with pytest.raises(CardError, match="AMD GPU only"):
            call()


def test_reference_formulas():
    """The 64-bit formulas the GPU tests compare with, against torch and against differences."""
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(5, 24, generator=g, dtype=torch.float64, requires_grad=True), torch.randn(24, generator=g, dtype=torch.float64, requires_grad=True)
    go = torch.randn(5, 24, generator=g, dtype=torch.float64)
    y = torch.nn.functional.rms_norm(x, (24,), w, eps=1e-6)
    assert torch.allclose(ref.rms_norm(x, w)[0], y.detach(), rtol=1e-13)
    dx, dw = torch.autograd.grad(y, (x, w), go)
    rx, rw, _, _ = ref.rms_norm_backward(x, w, go)
    assert torch.allclose(rx, dx, rtol=1e-12, atol=1e-14) and torch.allclose(rw, dw, rtol=1e-12, atol=1e-14)
    # Philox4x32-10 in Python integers
    import numpy as np
    words = ref.philox_words(np.array([3, 2 ** 40 + 5], dtype=np.uint64), 0x0123456789ABCDEF, 2)
    for b, row in zip((3, 2 ** 40 + 5), words):
        c, k = [b & 0xFFFFFFFF, b >> 32, 2, 1], [0x89ABCDEF, 0x01234567]
        for _ in range(10):
            p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        assert [int(v) for v in row] == c
    m = ref.keep_mask(10, 0.5, 7, elem_offset=6)
    assert torch.equal(m, ref.keep_mask(16, 0.5, 7)[6:])
    # 4-bit weights: one column by hand
    y, _ = ref.linear4(torch.tensor([[3, 15]], dtype=torch.uint8), torch.tensor([[2.0]]), torch.tensor([[5]], dtype=torch.uint8), torch.tensor([1.0]), 32,
                       torch.tensor([[1.0, -1.0]]), gamma=torch.tensor([2.0]), slope=0.5)
    assert float(y) == ((3 - 5) * 2 * 1 + (15 - 5) * 2 * -1 + 1) * 2 * 0.5


def test_describe_guidance_finds_dropout_rates_and_norms():
    from torch import nn
    from card_amd.guidance import describe_guidance
    net = nn.Sequential(nn.Linear(4, 8), nn.LeakyReLU(), nn.Dropout(0.2), nn.RMSNorm(8), nn.Linear(8, 6), nn.LeakyReLU(), nn.Linear(6, 1)).eval()
    d = describe_guidance(net)
    assert d["dropout"] == [0.2, 0.0] and d["norms"] == [None, net[3], None] and d["dims"] == [4, 8, 6, 1]
    lin = lambda: nn.Linear(4, 4)  # noqa: E731
    act = nn.LeakyReLU
    # eval-mode Dropout anywhere is the identity, as ever; its rates are known where one stands behind each hidden layer
    for layers in ([nn.Dropout(0.1), lin(), act(), lin()], [lin(), act(), nn.Dropout(0.1), nn.Dropout(0.2), lin()], [lin(), act(), lin(), nn.Dropout(0.3)],
                   [lin(), nn.Dropout(0.3), nn.BatchNorm1d(4), act(), lin()]):
        assert describe_guidance(nn.Sequential(*layers).eval())["dropout"] is None
    for layers in ([lin(), nn.RMSNorm(4), lin()], [nn.RMSNorm(5), lin()], [nn.RMSNorm(4), nn.RMSNorm(4), lin()], [lin(), act(), nn.RMSNorm(4)],
                   [lin(), act(), nn.RMSNorm(4), act(), lin()], [lin(), act(), nn.RMSNorm(4), nn.BatchNorm1d(4), lin()]):
        with pytest.raises(CardError):
            describe_guidance(nn.Sequential(*layers).eval())


@pytest.mark.parametrize("change,needle", [(dict(rows=-1), "rows"), (dict(n_z=0), "n_z"), (dict(f=None), "null handle"), (dict(rows=1 << 50, n_z=1 << 20), "63 bits")])
def test_fphi_forward_mc_refusals(change, needle):
    a = dict(f=P, rows=1, n_z=1)
    a.update(change)
    p = (C.c_double * 1)(0.5)
    assert _lib.lib().card_fphi_forward_mc(a["f"], P, a["rows"], a["n_z"], p, 1, 0, P, None) == E_INVALID and needle in msg(), msg()
