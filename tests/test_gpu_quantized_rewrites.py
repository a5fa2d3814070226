"""ops.quantize_rows over rows that are dropped and written again, as a program that takes back tokens does, against the plain form."""

import pytest
import torch

from chunkkv_amd import ops
from tests import test_gpu_quantized_cache as Q

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("back", [100, 96, 64, 128])  # from the middle of a block, and from first rows of one
def test_dropped_rows_written_again(block, back):
    c = Q._new(2, 200, 64, block)
    ops.quantize_rows(c, Q._rows(2, 140, 64, BF, 1, 0.5), Q._rows(2, 140, 64, BF, 2, 0.5))
    big = 1000 * Q._rows(2, 1, 64, BF, 3, 0.0)
    ops.quantize_rows(c, big, big, 140)  # raises its block's scale, then is dropped
    k, v = Q._rows(2, 170 - back, 64, BF, 4, 0.5), Q._rows(2, 170 - back, 64, BF, 5, 0.5)
    want = Q._want(c, k, v, back)
    ops.quantize_rows(c, k, v, back)
    Q._check(c, want)
    fresh = Q._new(2, 200, 64, block, 1)
    first = (back + block - 1) // block  # blocks that hold new rows alone
    ops.quantize_rows(fresh, k[:, :, first * block - back :], v[:, :, first * block - back :], first * block)
    assert torch.equal(c.k_scale.view(torch.uint8)[:, :, first : -(-170 // block)], fresh.k_scale.view(torch.uint8)[:, :, first : -(-170 // block)])
