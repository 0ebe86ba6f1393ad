"""CPU tests of the feed-forward operators at the edges of what their documents allow."""
import ctypes

import pytest

from brovisionml_b200 import _blocks_capi as B
from test_blocks_api import BF16, E4M3, EINVAL, at, err, gated_args, linear_args


@pytest.mark.parametrize("x,x_scale", [(None, None), (at(0), at(5))])
def test_empty_batches_in_8_bits(x, x_scale):
    """T = 0 rows are fine in 8 bits too, their (empty) scales null or not; the weights'
    scales are needed all the same."""
    a = linear_args(T=0, x=x, y=None, in_type=E4M3, x_scale=x_scale, w_scale=at(6))
    assert B.blocks_lib.bvml_linear(ctypes.byref(a), None, 0, None) == 0, err()
    assert B.blocks_lib.bvml_linear_workspace_bytes(ctypes.byref(a)) == 0
    a = gated_args(T=0, x=x, h=None, in_type=E4M3, out_type=BF16, x_scale=x_scale,
                   gate_scale=at(6), up_scale=at(7))
    assert B.blocks_lib.bvml_gated_linear(ctypes.byref(a), None, 0, None) == 0, err()
    a = linear_args(T=0, x=x, y=None, in_type=E4M3, x_scale=x_scale)
    assert B.blocks_lib.bvml_linear(ctypes.byref(a), None, 0, None) == EINVAL
    assert "need their scales" in err()
    a = linear_args(T=1, in_type=E4M3, w_scale=at(6))
    assert B.blocks_lib.bvml_linear(ctypes.byref(a), None, 0, None) == EINVAL
    assert "need their scales" in err()
