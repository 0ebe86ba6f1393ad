"""The feed-forward operators at the edges of what their documents allow. Bounds as in
test_gpu_blocks.py."""
import pytest
import torch

import brovisionml_b200 as bv
from test_gpu_blocks import BF16, E4M3, F32, quantized, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead", [(0,), (2, 0), (0, 3)])
def test_empty_batches_in_8_bits(lead):
    """The 8-bit chain on no rows: norm, gated product, product."""
    x = torch.empty(*lead, 64, device="cuda", dtype=BF16)
    q, scale = bv.rms_norm_e4m3(x, rnd(64))
    assert q.shape == x.shape and q.dtype == E4M3 and scale.shape == lead
    (w, ws), (v, vs) = quantized(40, 64, 0), quantized(40, 64, 1)
    h = bv.gated_linear(q, w, v, x_scale=scale, gate_scale=ws, up_scale=vs)
    assert h.shape == (*lead, 40) and h.dtype == BF16
    y, z = bv.linear(q, w, rnd(40), x_scale=scale, w_scale=ws, out_dtype=F32, save=True)
    assert y.shape == z.shape == (*lead, 40) and y.dtype == F32
