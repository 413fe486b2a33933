"""The 8-bit operators have no gradients: what they refuse of autograd's tensors, and what autograd learns of the tensors
that they write."""
import pytest
import torch
from torch.autograd import forward_ad

from elips_b200 import int8 as ops


def dual(*shape):
    return forward_ad.make_dual(torch.ones(shape), torch.ones(shape))


def codes(*shape):
    return torch.zeros(shape, dtype=torch.int8)


ONE, SLOTS = torch.ones(4), torch.zeros(2, dtype=torch.int64)
TABLE, OFFSETS = torch.zeros((2, 3), dtype=torch.int32), torch.tensor([0, 1, 2])
CACHE, SCALES, ROWS = codes(2, 3, 4, 2, 8), torch.zeros((2, 3, 4, 2)), torch.zeros((2, 2, 8))


@pytest.mark.parametrize("call", [
    lambda: ops.quantize_rows(dual(4, 8)),
    lambda: ops.linear_int8(dual(4, 8), codes(4, 8), ONE),
    lambda: ops.linear_int8(torch.ones((4, 8)), codes(4, 8), dual(4)),
    lambda: ops.linear_int8(torch.ones((4, 8)), codes(4, 8), ONE, dual(4)),
    lambda: ops.linear_int8(torch.ones((4, 8)), codes(4, 8), ONE, out=dual(4, 4)),
    lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), dual(4), ONE),
    lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE, dual(4)),
    lambda: ops.cache_write(CACHE, SCALES, (ROWS, dual(2, 2, 8)), SLOTS),
    lambda: ops.cache_write(CACHE, dual(2, 3, 4, 2), (ROWS, ROWS), SLOTS),
    lambda: ops.cache_read(CACHE, dual(2, 3, 4, 2), TABLE, OFFSETS, 2),
    lambda: ops.cache_read(CACHE, SCALES, TABLE, OFFSETS, 2, out=(dual(2, 2, 8), ROWS)),
])
@pytest.mark.parametrize("recorded", [True, False])
def test_tangents_refused(call, recorded):
    with forward_ad.dual_level(), torch.set_grad_enabled(recorded):
        with pytest.raises(ValueError, match="gradient"):
            call()


def test_tensors_without_tangents_go_on():
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="CUDA"):
            ops.quantize_rows(torch.ones((4, 8)))
        with pytest.raises(ValueError, match="CUDA"):
            ops.linear_int8(forward_ad.unpack_dual(dual(4, 8)).primal, codes(4, 8), ONE)
