"""A wait that expires among the 8-bit operators' kernels is reported by device_error, and by nothing else: searches
neither fail for it nor clear it, and the context stays usable."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def search():
    from elips_b200 import ExactIndex
    g = np.random.default_rng(5)
    base = g.standard_normal((500, 32)).astype(np.float32)
    ix = ExactIndex("euclidean", 32)
    ix.add(base)
    _, rows = ix.search_batch(base[:7], 1)
    assert np.array_equal(rows[:, 0], np.arange(7))


def test_expired_wait_is_no_error_of_a_search():
    from elips_b200 import _capi, int8
    assert _capi.device_error(0) == 0
    assert _capi.LIB.elips_b200_int8_wait_selftest(0, 100_000) == _capi.OK
    search()
    assert _capi.LIB.elips_b200_wait_selftest(0, 100_000) == _capi.DEVICE_TIMEOUT    # clears its own word only
    search()
    assert _capi.device_error(0) != 0
    assert _capi.device_error(0) == 0
    a, s = int8.quantize_rows(torch.ones((200, 64), device="cuda"))
    assert (int8.gemm_int8(a, a, s, s, out_dtype=torch.float32) - 64).abs().max() < 1e-4
    assert _capi.device_error(0) == 0


def test_refused_budgets():
    from elips_b200 import _capi
    for cycles in (0, 1 << 40):
        assert _capi.LIB.elips_b200_int8_wait_selftest(0, cycles) == _capi.INVALID_ARGUMENT
    assert _capi.device_error(0) == 0
