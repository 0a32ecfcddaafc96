"""The layer operators at the edges of their range.  Tolerances count roundings, as in test_gpu_layers.py."""
import pytest
import torch

import card_amd
from tests import layer_reference as ref
from tests.layer_reference import TINY, U, U32, assert_within
from tests.test_gpu_layers import TYPES, chain, ids, rand

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
