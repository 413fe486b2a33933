"""Every kernel form of the int8 product against the definition, in every output type, with and without a bias, into
plain and offset outputs. Which form a size takes is asked of the library, so that a size that no longer takes the form
it stands for fails here."""
import ctypes
import math

import numpy as np
import pytest
import torch

from elips_b200 import _capi
from tests import int8_oracle as R
from tests.test_gpu_int8 import FLOATS, f32, gemm_case

# (rows of a tile, CTAs that split k): 1 the kernel of a few rows, 0 the one of CTA pairs. One size each, then those
# whose persistent CTAs (two to an SM) or pairs take three tiles or more.
FORMS = [
    ((1, 1), (1, 3001, 1100)), ((1, 1), (2, 1000, 5000)), ((1, 1), (4, 515, 4100)), ((1, 1), (7, 300, 3000)),
    ((16, 1), (20, 70, 130)), ((16, 2), (9, 9000, 2048)), ((16, 4), (100, 300, 1024)), ((16, 8), (16, 130, 2050)),
    ((32, 1), (4096, 10, 70)), ((32, 2), (20, 9000, 2100)), ((32, 4), (65, 1000, 1024)), ((32, 8), (300, 10, 2049)),
    ((64, 1), (129, 4096, 300)), ((64, 2), (33, 9000, 4096)), ((64, 4), (1500, 10, 2048)), ((64, 8), (200, 300, 4100)),
    ((128, 1), (300, 4096, 700)), ((128, 2), (65, 9000, 8192)), ((128, 4), (2600, 10, 4096)), ((128, 8), (129, 1000, 8190)),
    ((0, 1), (2600, 1000, 64)), ((0, 1), (2600, 2600, 700)), ((0, 1), (1000, 4400, 1500)),
]
MANY_TILES = [((16, 1), (16, 120000, 64)), ((32, 1), (32, 120000, 100)), ((64, 1), (64, 120000, 128)),
              ((128, 1), (300, 40000, 1024)), ((0, 1), (4096, 4096, 260)), ((0, 1), (4000, 3900, 1000))]


def form(m, n, k, dtype, sms):
    rows, splits = ctypes.c_int(), ctypes.c_int()
    kind = {torch.float32: _capi.PRECISION_FP32, torch.float16: _capi.PRECISION_FP16, torch.bfloat16: _capi.PRECISION_BF16}
    _capi.check(_capi.LIB.elips_b200_gemm_int8_form(m, n, k, kind[dtype], sms, ctypes.byref(rows), ctypes.byref(splits)), "form")
    return rows.value, splits.value


@pytest.mark.parametrize("dtype", FLOATS)
def test_sizes_take_the_forms_they_stand_for(dtype):
    for want, size in FORMS + MANY_TILES:
        assert form(*size, dtype, 148) == want, size
    wide = {(r, s) for r in (16, 32, 64, 128) for s in (1, 2, 4, 8)}
    assert {f for f, _ in FORMS} == wide | {(0, 1), (1, 1)}
    for (rows, _), (m, n, _) in MANY_TILES:
        per = math.ceil(m / (rows or 256)) * math.ceil(n / (128 if rows else 256)) / (296 if rows else 74)
        assert per > 3, (m, n)


def test_form_refusals():
    a, b = ctypes.c_int(), ctypes.c_int()
    call = _capi.LIB.elips_b200_gemm_int8_form
    assert call(4, 4, 4, 0, 148, None, ctypes.byref(b)) == _capi.INVALID_ARGUMENT
    for m, n, k, kind, sms in ((0, 4, 4, 0, 148), (4, 0, 4, 0, 148), (4, 4, -1, 0, 148), (4, 4, 1 << 17, 0, 148),
                               (4, 4, 4, _capi.PRECISION_INT8, 148), (4, 4, 4, 0, 1), (1 << 32, 4, 4, 0, 148)):
        assert call(m, n, k, kind, sms, ctypes.byref(a), ctypes.byref(b)) == _capi.INVALID_ARGUMENT


def assert_product(c, a, b, sa, sb, bias, dtype):
    """Within gemm_bound's fp32 roundings and then one rounding to the type. That is relative, but for fp16 numbers below
    2^-14, whose step is 2^-24: up to 2^-25 on top of the fp32 error, which a bias that cancels most of the product leaves
    well above 2^-24 of the result. (E.g. 2.8161e-5, off by 2.1e-9 in fp32 and by 3.18e-8 > 2^-25 = 2.98e-8 after it.)"""
    v = R.gemm(a.cpu().numpy(), b.cpu().numpy(), f32(sa), f32(sb), None if bias is None else f32(bias))
    off = np.abs(c.double().cpu().numpy() - v)
    fp32 = R.gemm_bound(v, None if bias is None else f32(bias), 0.0)
    eps = torch.finfo(dtype).eps
    bound = fp32 + np.maximum(eps / 2 * (np.abs(v) + fp32), 2.0 ** -25 if dtype == torch.float16 else 0.0)
    if dtype == torch.float16:
        fits = np.abs(v) < 65000
        off, bound = off[fits], bound[fits]
    assert (off <= bound).all(), float((off / bound).max())


def run(want, size, dtype, bias, first):
    from elips_b200 import int8
    m, n, k = size
    assert form(m, n, k, dtype, torch.cuda.get_device_properties(0).multi_processor_count) == want
    a, b, sa, sb, bv = gemm_case(m, n, k, dtype, bias)
    wide = torch.full((m, n + 24), 7.0, dtype=dtype, device="cuda")
    out = wide[:, first:first + n]
    int8.gemm_int8(a, b, sa, sb, bv, out=out)
    assert (wide[:, :first] == 7).all() and (wide[:, first + n:] == 7).all()
    assert_product(out, a, b, sa, sb, bv, dtype)
    plain = int8.gemm_int8(a, b, sa, sb, bv, out_dtype=dtype)
    assert torch.equal(plain, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("bias,first", [(None, 0), (torch.float32, 3), (torch.bfloat16, 8)])
@pytest.mark.parametrize("want,size", FORMS)
def test_forms(want, size, dtype, bias, first):
    run(want, size, dtype, bias, first)


@pytest.mark.gpu
@pytest.mark.parametrize("want,size,dtype", [(w, s, d) for i, (w, s) in enumerate(MANY_TILES)
                                             for d in ([FLOATS[0], FLOATS[1 + i % 2]])])
def test_three_tiles_a_cta(want, size, dtype):
    run(want, size, dtype, torch.float16, 16)


@pytest.mark.parametrize("dtype", FLOATS)
def test_one_and_two_rows_against_many_channels(dtype):
    """The kernel of a few rows spends as much on four channels of 64 codes as of 512, so many narrow ones go to the
    tensor cores; single tokens through a layer do not."""
    for size in ((1, 10000, 768), (1, 4096, 4096), (1, 40000, 4096), (2, 4096, 4096), (2, 10000, 768), (4, 2048, 2048)):
        assert form(*size, dtype, 148) == (1, 1), size
    for size in ((1, 1000000, 128), (1, 100000, 128), (1, 200000, 384), (2, 100000, 768), (4, 100000, 64), (4, 4096, 4096)):
        assert form(*size, dtype, 148)[0] == 16, size


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(1, 200000, 64), (2, 50000, 100), (1, 60001, 384), (4, 100000, 70), (8, 9000, 64)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_few_rows_against_many_channels(size, dtype):
    from elips_b200 import int8
    m, n, k = size
    a, b, sa, sb, bv = gemm_case(m, n, k, dtype, torch.bfloat16)
    out = int8.gemm_int8(a, b, sa, sb, bv, out_dtype=dtype)
    assert_product(out, a, b, sa, sb, bv, dtype)
    x = torch.randn((m, k), generator=torch.Generator(device="cuda").manual_seed(m), device="cuda")
    codes, scales = int8.quantize_rows(x)
    assert torch.equal(int8.linear_int8(x, b, sb, bv, out_dtype=dtype), int8.gemm_int8(codes, b, scales, sb, bv, out_dtype=dtype))
