"""Arguments the 8-bit row operators refuse, in Python and at the C ABI. No GPU is needed: every check of sizes,
types and strides comes before the device is touched."""
import ctypes

import pytest
import torch

from elips_b200 import DimensionMismatch, _capi
from elips_b200 import int8 as ops


def codes(m, k):
    return torch.zeros((m, k), dtype=torch.int8)


ONE = torch.ones(4)


@pytest.mark.parametrize("call,error", [
    (lambda: ops.quantize_rows(torch.zeros(4)), DimensionMismatch),
    (lambda: ops.quantize_rows(torch.zeros((4, 0))), DimensionMismatch),
    (lambda: ops.quantize_rows(torch.zeros((4, 4), dtype=torch.float64)), ValueError),
    (lambda: ops.quantize_rows(torch.zeros((4, 8)).t()), ValueError),
    (lambda: ops.quantize_rows(torch.zeros((4, 8), requires_grad=True)), ValueError),
    (lambda: ops.quantize_rows(torch.zeros((4, 8))), ValueError),                         # not on a CUDA device
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 9), ONE, ONE), DimensionMismatch),
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE[:3], ONE), DimensionMismatch),
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE, torch.ones(8)[::2]), ValueError),
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE, ONE.double()), ValueError),
    (lambda: ops.gemm_int8(codes(4, 8).float(), codes(4, 8), ONE, ONE), ValueError),
    (lambda: ops.gemm_int8(codes(4, 8), codes(8, 4).t(), ONE, ONE), ValueError),
    (lambda: ops.gemm_int8(codes(1, 8).expand(4, 8), codes(4, 8), ONE, ONE), ValueError),
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE, ONE, bias=torch.ones(5)), DimensionMismatch),
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE, ONE, bias=torch.ones(4, dtype=torch.int32)), ValueError),
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE, ONE, out_dtype=torch.int32), ValueError),
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE, ONE, out=torch.zeros((4, 5))), DimensionMismatch),
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE, ONE, out=torch.zeros((1, 4)).expand(4, 4)), ValueError),
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE.clone().requires_grad_(), ONE), ValueError),
    (lambda: ops.gemm_int8(codes(4, 8), codes(4, 8), ONE, ONE), ValueError),              # not on a CUDA device
    (lambda: ops.linear_int8(torch.zeros((4, 8), requires_grad=True), codes(4, 8), ONE), ValueError),
    (lambda: ops.linear_int8(torch.zeros((4, 0)), codes(4, 0), ONE), DimensionMismatch),
    (lambda: ops.linear_int8(torch.zeros((4, 7)), codes(4, 8), ONE), DimensionMismatch),
    (lambda: ops.linear_int8(torch.zeros((4, 8)), codes(4, 8), ONE), ValueError),         # not on a CUDA device
])
def test_products_and_rows_refused(call, error):
    with pytest.raises(error):
        call()


def cache(parts=2, pages=3, page=4, heads=2, dim=8):
    return torch.zeros((parts, pages, page, heads, dim), dtype=torch.int8), torch.zeros((parts, pages, page, heads))


def rows(t=2, heads=2, dim=8, parts=2):
    return tuple(torch.zeros((t, heads, dim)) for _ in range(parts))


SLOTS = torch.zeros(2, dtype=torch.int64)
TABLE = torch.zeros((2, 3), dtype=torch.int32)
OFFSETS = torch.tensor([0, 1, 2])


@pytest.mark.parametrize("call,error", [
    (lambda c, s: ops.cache_write(c, s, rows(parts=1), SLOTS), DimensionMismatch),
    (lambda c, s: ops.cache_write(c, s, rows(t=3), SLOTS), DimensionMismatch),
    (lambda c, s: ops.cache_write(c, s, rows(dim=7), SLOTS), DimensionMismatch),
    (lambda c, s: ops.cache_write(c, s, rows(), SLOTS.float()), ValueError),
    (lambda c, s: ops.cache_write(c, s, rows(), torch.zeros(4, dtype=torch.int64)[::2]), DimensionMismatch),
    (lambda c, s: ops.cache_write(c.int(), s, rows(), SLOTS), ValueError),
    (lambda c, s: ops.cache_write(c, s[:, :2], rows(), SLOTS), DimensionMismatch),
    (lambda c, s: ops.cache_write(c[:1].expand(2, 3, 4, 2, 8), s, rows(), SLOTS), ValueError),
    (lambda c, s: ops.cache_write(torch.cat([c, c]), torch.cat([s, s]), rows(parts=4), SLOTS), DimensionMismatch),
    (lambda c, s: ops.cache_write(c, s, (rows()[0], rows()[1].half()), SLOTS), ValueError),
    (lambda c, s: ops.cache_write(c, s, tuple(x.requires_grad_() for x in rows()), SLOTS), ValueError),
    (lambda c, s: ops.cache_write(c, s, rows(), SLOTS), ValueError),                      # not on a CUDA device
    (lambda c, s: ops.cache_read(c, s, TABLE, OFFSETS[:2], 2), DimensionMismatch),
    (lambda c, s: ops.cache_read(c, s, TABLE.float(), OFFSETS, 2), ValueError),
    (lambda c, s: ops.cache_read(c, s, torch.zeros((3, 2), dtype=torch.int32).t(), OFFSETS, 2), ValueError),
    (lambda c, s: ops.cache_read(c, s, TABLE, OFFSETS, -1), DimensionMismatch),
    (lambda c, s: ops.cache_read(c, s, TABLE, OFFSETS, 2, dtype=torch.int8), ValueError),
    (lambda c, s: ops.cache_read(c, s, TABLE, OFFSETS, 2, out=rows(parts=1)), DimensionMismatch),
    (lambda c, s: ops.cache_read(c, s, TABLE, OFFSETS, 3, out=rows()), DimensionMismatch),
    (lambda c, s: ops.cache_read(c, s, TABLE, OFFSETS, 2, out=tuple(x[:1].expand(2, 2, 8) for x in rows())), ValueError),
    (lambda c, s: ops.cache_read(c, s, TABLE, OFFSETS, 2), ValueError),                   # not on a CUDA device
])
def test_cache_refused(call, error):
    with pytest.raises(error):
        call(*cache())


def test_c_entry_points_refuse_before_the_device():
    lib, bad = _capi.LIB, _capi.INVALID_ARGUMENT
    f32, bf16, int8 = _capi.PRECISION_FP32, _capi.PRECISION_BF16, _capi.PRECISION_INT8
    p = 16  # stands for a device address: none of these calls reaches the device
    assert lib.elips_b200_quantize_rows(0, None, f32, 1, 8, 8, p, 16, p, None) == bad
    assert lib.elips_b200_quantize_rows(0, p, int8, 1, 8, 8, p, 16, p, None) == bad
    assert lib.elips_b200_quantize_rows(0, p, f32, 1, 0, 8, p, 16, p, None) == bad
    assert lib.elips_b200_quantize_rows(0, p, f32, 1, (1 << 24) + 1, 8, p, 1 << 25, p, None) == bad
    assert lib.elips_b200_quantize_rows(0, p, f32, 2, 8, 8, p, 7, p, None) == bad

    def gemm(**kw):
        d = dict(a=p, a_scales=p, b=p, b_scales=p, bias=None, out=p, m=4, n=4, k=16, a_stride=16, b_stride=16, out_stride=4,
                 a_type=int8, bias_type=0, out_type=f32, reserved=0) | kw
        return lib.elips_b200_gemm_int8(0, ctypes.byref(_capi.Gemm(*d.values())), None)
    assert lib.elips_b200_gemm_int8(0, None, None) == bad
    assert gemm(a=None) == bad
    assert gemm(b_scales=None) == bad
    assert gemm(a_scales=None) == bad
    assert gemm(a_stride=15) == bad
    assert gemm(b_stride=15) == bad
    assert gemm(out_stride=3) == bad
    assert gemm(out_type=int8) == bad
    assert gemm(a_type=7) == bad
    assert gemm(bias=p, bias_type=9) == bad
    assert gemm(k=1 << 17, a_stride=1 << 17, b_stride=1 << 17) == bad   # the int32 sum could pass 2^31
    assert gemm(m=1 << 32) == bad
    assert gemm(n=-1) == bad
    assert gemm(a_type=bf16, k=0) == bad
    assert gemm(m=0, a=None) == _capi.OK                                # nothing to do

    def described(**kw):
        d = dict(codes=p, scales=p, parts=1, pages=3, page_size=4, heads=2, dim=8) | kw
        return _capi.Cache(d["codes"], d["scales"], d["parts"], d["pages"], d["page_size"], d["heads"], d["dim"],
                           (0, 64, 16, 8), (0, 8, 2, 1))
    r = (_capi.Rows * 2)(_capi.Rows(p, 16, 8), _capi.Rows(None, 16, 8))

    def write(c, type=bf16, slots=p):
        return lib.elips_b200_cache_write(0, None if c is None else ctypes.byref(c), r, type, 2, slots, 1, None)

    def read(c, type=bf16, **kw):
        d = dict(page_table=p, offsets=p, table_stride=3, sequences=2, table_width=3, total=2, table_64bit=0,
                 offsets_64bit=0) | kw
        return lib.elips_b200_cache_read(0, None if c is None else ctypes.byref(c),
                                         ctypes.byref(_capi.Sequences(*d.values())), r, type, 1, None)
    for call in (write, read):
        assert call(None) == bad
        assert call(described(parts=3)) == bad
        assert call(described(parts=2)) == bad            # the second part's rows are missing
        assert call(described(dim=0)) == bad
        assert call(described(page_size=0)) == bad
        assert call(described(codes=None)) == bad
        assert call(described(pages=1 << 30, page_size=2)) == bad
        assert call(described(), type=int8) == bad
    assert write(described(), slots=None) == bad
    assert read(described(), page_table=None) == bad
    assert read(described(), total=-1) == bad
    assert read(described(), sequences=1 << 40) == bad
    assert lib.elips_b200_cache_read(0, ctypes.byref(described()), None, r, bf16, 1, None) == bad
    assert read(described(), offsets=None) == bad


@pytest.mark.parametrize("kind", [_capi.PRECISION_INT8, _capi.PRECISION_BF16])
def test_products_onto_their_inputs_refused(kind):
    """An output on any byte of an input, from either side of it. Every address is far from the others' unless named."""
    size = 1 if kind == _capi.PRECISION_INT8 else 2
    m, n, k, a, b, a_scales, b_scales, bias, out = 4, 8, 16, 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20, 6 << 20

    def status(**kw):
        d = dict(a=a, a_scales=a_scales, b=b, b_scales=b_scales, bias=bias, out=out, m=m, n=n, k=k, a_stride=k,
                 b_stride=k, out_stride=n, a_type=kind, bias_type=_capi.PRECISION_BF16, out_type=_capi.PRECISION_FP32,
                 reserved=0) | kw
        return _capi.LIB.elips_b200_gemm_int8(0, ctypes.byref(_capi.Gemm(*d.values())), None)
    out_bytes = 4 * m * n
    inputs = [(a, m * k * size), (b, n * k), (b_scales, 4 * n), (bias, 2 * n)]
    if kind == _capi.PRECISION_INT8:
        inputs.append((a_scales, 4 * m))
    for at, count in inputs:
        assert status(out=at) == _capi.INVALID_ARGUMENT
        assert status(out=at + count - 4) == _capi.INVALID_ARGUMENT
        assert status(out=at - out_bytes + 4) == _capi.INVALID_ARGUMENT
    # One column of the output lies on the rows' last one, in a buffer of 256 bytes a row.
    assert status(a_stride=256 // size, out_stride=64, out=a + k * size - 4) == _capi.INVALID_ARGUMENT
    # The output's last column reaches into the next row's first value.
    assert status(a_stride=256 // size, out_stride=64, out=a + 256 - 4 * n + 4) == _capi.INVALID_ARGUMENT


def test_rows_and_reads_onto_one_another_refused():
    lib, bad, f32 = _capi.LIB, _capi.INVALID_ARGUMENT, _capi.PRECISION_FP32
    x, codes_at, scales = 1 << 20, 2 << 20, 3 << 20
    assert lib.elips_b200_quantize_rows(0, x, f32, 4, 16, 16, x, 16, scales, None) == bad
    assert lib.elips_b200_quantize_rows(0, x, f32, 4, 16, 16, x + 255, 16, scales, None) == bad
    assert lib.elips_b200_quantize_rows(0, x, f32, 4, 16, 16, codes_at, 16, x + 16, None) == bad
    assert lib.elips_b200_quantize_rows(0, x, f32, 4, 16, 16, codes_at, 16, codes_at + 60, None) == bad
    c = _capi.Cache(x, scales, 2, 3, 4, 2, 8, (192, 64, 16, 8), (24, 8, 2, 1))
    r = (_capi.Rows * 2)(_capi.Rows(codes_at, 16, 8), _capi.Rows(codes_at, 16, 8))
    q = _capi.Sequences(4 << 20, 5 << 20, 3, 2, 3, 2, 0, 0)
    assert lib.elips_b200_cache_read(0, ctypes.byref(c), ctypes.byref(q), r, _capi.PRECISION_BF16, 1, None) == bad
