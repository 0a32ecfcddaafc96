"""The layer operators at the edges of their range.  Tolerances count roundings, as in test_gpu_layers.py."""
import pytest
import torch

import card_amd
from tests import layer_reference as ref
from tests.layer_reference import TINY, U, U32, assert_within
from tests.test_gpu_layers import DEV, TYPES, chain, ids, rand

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
