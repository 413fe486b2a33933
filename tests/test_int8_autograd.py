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


def writes(t):
    """(what is written, the call) for every entry point that writes into tensors it is given."""
    x, w = torch.ones((t, 32), device="cuda"), torch.ones((16, 32), device="cuda")
    codes_x, sx = ops.quantize_rows(x)
    codes_w, sw = ops.quantize_rows(w)
    cache = torch.zeros((2, 4, 8, 1, 32), dtype=torch.int8, device="cuda")
    scales = torch.zeros((2, 4, 8, 1), device="cuda")
    slots, table = torch.arange(t, device="cuda"), torch.arange(4, device="cuda")[None]
    offsets = torch.tensor([0, t], device="cuda")
    out = torch.zeros((t, 16), device="cuda")
    read = tuple(torch.zeros((t, 1, 32), device="cuda") for _ in range(2))
    return [((out,), lambda: ops.gemm_int8(codes_x, codes_w, sx, sw, out=out)),
            ((out,), lambda: ops.linear_int8(x, codes_w, sw, out=out)),
            ((cache, scales), lambda: ops.cache_write(cache, scales, (x[:, None], x[:, None]), slots)),
            (read, lambda: ops.cache_read(cache, scales, table, offsets, t, out=read))]


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("mode", ["plain", "no_grad", "inference"])
def test_written_tensors_have_a_new_version(which, mode):
    written, call = writes(5)[which]
    before = [w._version for w in written]
    with {"no_grad": torch.no_grad, "inference": torch.inference_mode}.get(mode, torch.enable_grad)():
        call()
    assert [w._version for w in written] == [v + 1 for v in before]


@pytest.mark.gpu
def test_written_inference_tensors():
    """They have no version to raise."""
    with torch.inference_mode():
        for _, call in writes(5):
            call()


@pytest.mark.gpu
def test_backward_through_a_tensor_that_was_written():
    """What autograd saved for a product is no longer what the product read."""
    (out,), call = writes(5)[0]
    p = torch.ones((5, 16), device="cuda", requires_grad=True)
    y = (p * out).sum()
    call()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
