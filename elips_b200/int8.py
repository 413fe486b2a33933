"""8-bit row operators on one B200, for the models around an index.

One format: a row x is held as int8 codes q and one fp32 scale s with
s = max|x| / 127 and q the integers nearest to x / s (ties to even), so x is
s * q to within s / 2. It is what ExactIndex(precision="int8") takes as rows
and queries, and what every function here makes or reads:

  quantize_rows   rows -> codes, scales (activations per token, weights per
                  output channel)
  gemm_int8       codes x codes -> scaled products (a layer's output, or the
                  scores of queries against stored rows)
  linear_int8     rows x codes: quantize_rows and gemm_int8 in one call
  cache_write     rows quantised into the slots of a paged cache
  cache_read      sequences of pages back into packed rows

The reference has no such operators: its scalar quantiser has one affine scale
per dimension and scores by lookup (src/quant_engine/ScalarQuantizer.cpp:83-128).

Everything takes CUDA tensors, runs asynchronously on `stream` (default: the
current stream of the tensors' device) and can be captured into a CUDA graph.
With another stream the outputs belong to it and the inputs are held until its
work is done; ordering that work after the inputs are written is the caller's.
These are the serving forms: rounding has no gradient, so an input that
requires one is refused while gradients are recorded.

Rows that cannot be held: a row whose largest magnitude is below 127 * 2^-126
becomes zeros with scale 0; a row with an infinity or a NaN gets a scale that
is not finite and codes 0, reads back as NaN and gives NaN products, without
touching any other row.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _capi as capi
from .exact import DimensionMismatch

_LIB = capi.LIB
_TYPES = {torch.float32: capi.PRECISION_FP32, torch.float16: capi.PRECISION_FP16,
          torch.bfloat16: capi.PRECISION_BF16}
_INTS = (torch.int32, torch.int64)


def _device(first, *others) -> int:
    """The CUDA device all tensors are on."""
    dev = first.device
    if dev.type != "cuda":
        raise ValueError("tensors must be on a CUDA device")
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on {dev} and {t.device}")
    return dev.index


def _no_grad(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("8-bit operators have no gradient: detach the inputs or use torch.no_grad()")


def _float_type(dtype, what: str) -> int:
    if dtype not in _TYPES:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, not {dtype}")
    return _TYPES[dtype]


def _matrix(t, dtype, what: str) -> None:
    if t.dim() != 2:
        raise DimensionMismatch(f"{what} must have two axes")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, not {t.dtype}")
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{what} must have its last axis contiguous")


def _pitch(t) -> int:
    """Elements from one row to the next; the width where there is no next."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _scales(t, n: int, what: str) -> None:
    if t.dtype != torch.float32:
        raise ValueError(f"{what} must be float32, not {t.dtype}")
    if t.dim() != 1 or t.shape[0] != n:
        raise DimensionMismatch(f"{what} must have {n} entries")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{what} must be contiguous")


def _handle(stream) -> int:
    return stream if isinstance(stream, int) else stream.cuda_stream


@contextlib.contextmanager
def _using(stream, device: int, *tensors):
    """Makes `stream` current, so that what is allocated belongs to it, and
    keeps the tensors' memory until its work is done."""
    s = torch.cuda.ExternalStream(_handle(stream), device=device)
    with torch.cuda.stream(s):
        yield
    for t in tensors:
        if t is not None:
            t.record_stream(s)


def _run(fn, stream, device: int, *tensors):
    """fn(stream handle) on the caller's stream."""
    if stream is None:
        return fn(torch.cuda.current_stream(device).cuda_stream)
    with _using(stream, device, *tensors):
        return fn(_handle(stream))


def quantize_rows(x, stream=None):
    """(codes int8 [n, d], scales float32 [n]) of float rows x [n, d]. The rows
    of codes start on multiples of 16 bytes (codes is a view of wider rows
    where d is no such multiple): gemm_int8 reads them as they are."""
    _no_grad(x)
    kind = _float_type(x.dtype, "rows")
    _matrix(x, None, "rows")
    n, d = x.shape
    if d == 0:
        raise DimensionMismatch("rows must have at least one value")
    device = _device(x)

    def go(s):
        wide = -(-d // 16) * 16
        codes = torch.empty((n, wide), dtype=torch.int8, device=x.device)
        scales = torch.empty(n, dtype=torch.float32, device=x.device)
        capi.check(_LIB.elips_b200_quantize_rows(device, x.data_ptr(), kind, n, d, _pitch(x), codes.data_ptr(), wide,
                                                 scales.data_ptr(), s), "elips_b200_quantize_rows")
        return codes[:, :d], scales

    return _run(go, stream, device, x)


def _target(out, m: int, n: int) -> None:
    _matrix(out, None, "out")
    if out.shape != (m, n):
        raise DimensionMismatch(f"out must be {m} x {n}")
    if m > 1 and out.stride(0) < n:
        raise ValueError("rows of out overlap")


def _weight(b, b_scales, bias, k: int) -> int:
    """Checks the n x k operand, its scales and the bias; the bias type."""
    _matrix(b, torch.int8, "weight codes")
    if b.shape[1] != k:
        raise DimensionMismatch(f"rows of {k} and of {b.shape[1]} values")
    if b.shape[0] > 1 and b.stride(0) < k:
        raise ValueError("weight rows overlap")
    _scales(b_scales, b.shape[0], "weight scales")
    if bias is None:
        return 0
    kind = _float_type(bias.dtype, "bias")
    if bias.dim() != 1 or bias.shape[0] != b.shape[0]:
        raise DimensionMismatch(f"bias must have {b.shape[0]} entries")
    if bias.shape[0] > 1 and bias.stride(0) != 1:
        raise ValueError("bias must be contiguous")
    return kind


def gemm_int8(a, b, a_scales, b_scales, bias=None, out_dtype=torch.bfloat16, out=None, stream=None):
    """out[i, j] = (sum_l a[i, l] b[j, l]) * a_scales[i] * b_scales[j] + bias[j],
    the sum exact in int32 (so the width is below 2^17), rounded once.

    a [m, k] and b [n, k] are int8 with contiguous rows, as quantize_rows gives
    them: a activations and b a layer's weight with a scale per channel, or a
    queries and b stored rows. Operands whose rows start on multiples of 16
    bytes are read as they are, others are copied to such rows first. bias
    [n] may have another float type than out."""
    _no_grad(a_scales, b_scales, bias, out)
    kind = _float_type(out_dtype if out is None else out.dtype, "out")
    _matrix(a, torch.int8, "row codes")
    m, k = a.shape
    if m > 1 and a.stride(0) < k:
        raise ValueError("rows of codes overlap")
    _scales(a_scales, m, "row scales")
    bias_kind = _weight(b, b_scales, bias, k)
    n = b.shape[0]
    if out is not None:
        _target(out, m, n)
    device = _device(a, b, a_scales, b_scales, bias, out)

    def go(s):
        c = out if out is not None else torch.empty((m, n), dtype=out_dtype, device=a.device)
        capi.check(_LIB.elips_b200_gemm_int8(
            device, a.data_ptr(), _pitch(a), a_scales.data_ptr(), b.data_ptr(), _pitch(b), b_scales.data_ptr(),
            None if bias is None else bias.data_ptr(), bias_kind, m, n, k, c.data_ptr(), kind, _pitch(c), s),
            "elips_b200_gemm_int8")
        return c

    return _run(go, stream, device, a, b, a_scales, b_scales, bias, out)


def linear_int8(x, weight, weight_scales, bias=None, out_dtype=None, out=None, stream=None):
    """gemm_int8 over the rows of x [m, k], quantised on the way as
    quantize_rows quantises them; out_dtype defaults to x's type."""
    _no_grad(x, weight_scales, bias, out)
    kind = _float_type(x.dtype, "rows")
    _matrix(x, None, "rows")
    m, k = x.shape
    if k == 0:
        raise DimensionMismatch("rows must have at least one value")
    bias_kind = _weight(weight, weight_scales, bias, k)
    dtype = out.dtype if out is not None else out_dtype if out_dtype is not None else x.dtype
    out_kind = _float_type(dtype, "out")
    n = weight.shape[0]
    if out is not None:
        _target(out, m, n)
    device = _device(x, weight, weight_scales, bias, out)

    def go(s):
        c = out if out is not None else torch.empty((m, n), dtype=dtype, device=x.device)
        capi.check(_LIB.elips_b200_linear_int8(
            device, x.data_ptr(), kind, _pitch(x), weight.data_ptr(), _pitch(weight), weight_scales.data_ptr(),
            None if bias is None else bias.data_ptr(), bias_kind, m, n, k, c.data_ptr(), out_kind, _pitch(c), s),
            "elips_b200_linear_int8")
        return c

    return _run(go, stream, device, x, weight, weight_scales, bias, out)


def _cache(codes, scales):
    """The C description of a cache's two tensors."""
    if codes.dtype != torch.int8 or scales.dtype != torch.float32:
        raise ValueError("a cache has int8 codes and float32 scales")
    if codes.dim() != 5 or scales.shape != codes.shape[:4]:
        raise DimensionMismatch("codes must be [parts, pages, page, heads, dim] and scales [parts, pages, page, heads]")
    parts, pages, page, heads, dim = codes.shape
    if not 1 <= parts <= 2:
        raise DimensionMismatch("a cache has one or two parts")
    if page < 1 or heads < 1 or dim < 1:
        raise DimensionMismatch("pages, heads and rows must not be empty")
    st = codes.stride()
    if st[4] != 1 and dim > 1:
        raise ValueError("rows of codes must be contiguous")
    return capi.Cache(codes.data_ptr(), scales.data_ptr(), parts, pages, page, heads, dim, st[:4], scales.stride())


def _distinct(t, what: str) -> None:
    """Refuses a tensor to be written whose elements share memory by a stride of 0."""
    if 0 in t.stride() and any(st == 0 and n > 1 for st, n in zip(t.stride(), t.shape)):
        raise ValueError(f"{what} must not be an expanded tensor")


def _rows(tensors, count, heads: int, dim: int, dtype, what: str):
    """The C description of a part's rows [count, heads, dim], for each part."""
    for x in tensors:
        if x.dim() != 3 or x.shape[1] != heads or x.shape[2] != dim or x.shape[0] != count:
            raise DimensionMismatch(f"{what} must be [{count}, {heads}, {dim}], not {list(x.shape)}")
        if x.dtype != dtype:
            raise ValueError(f"{what} must be {dtype}, not {x.dtype}")
        if x.stride(2) != 1 and dim > 1:
            raise ValueError(f"{what} must have their last axis contiguous")
    return (capi.Rows * len(tensors))(*[(x.data_ptr(), x.stride(0), x.stride(1)) for x in tensors])


def cache_write(codes, scales, rows, slots, stream=None) -> None:
    """Quantises rows into the slots of a paged cache, in place.

    codes int8 [parts, pages, page, heads, dim] and scales float32 [parts,
    pages, page, heads] are the cache: one part holds one kind of row, two hold
    keys and values. rows is a tuple of one float tensor [t, heads, dim] per
    part; each of its rows gets a scale per head. Row i goes to slot slots[i]
    (int32 or int64): row s % page of page s // page. A slot below 0 or past
    the last one is skipped (padding); of a slot given twice the last row is
    kept. Slots that are not named stay as they are."""
    rows = tuple(rows)
    _no_grad(scales, *rows)
    c = _cache(codes, scales)
    _distinct(codes, "codes")
    _distinct(scales, "scales")
    if len(rows) != c.parts:
        raise DimensionMismatch(f"{len(rows)} tensors of rows for a cache of {c.parts} parts")
    if slots.dtype not in _INTS:
        raise ValueError(f"slots must be int32 or int64, not {slots.dtype}")
    if slots.dim() != 1 or (slots.shape[0] > 1 and slots.stride(0) != 1):
        raise DimensionMismatch("slots must be one contiguous axis")
    t = slots.shape[0]
    kind = _float_type(rows[0].dtype, "rows")
    r = _rows(rows, t, c.heads, c.dim, rows[0].dtype, "rows")
    device = _device(codes, scales, slots, *rows)

    def go(s):
        capi.check(_LIB.elips_b200_cache_write(device, ctypes.byref(c), r, kind, t, slots.data_ptr(),
                                               slots.dtype == torch.int64, s), "elips_b200_cache_write")

    _run(go, stream, device, codes, scales, slots, *rows)


def cache_read(codes, scales, page_table, offsets, total: int, dtype=torch.bfloat16, out=None, stream=None):
    """Sequences of cached rows, packed: a tuple of one tensor [total, heads,
    dim] per part.

    Sequence b is the output rows offsets[b] .. offsets[b + 1] (offsets
    ascending, one more entry than there are sequences, int32 or int64);
    position i of it is read from row i % page of page page_table[b, i // page]
    (int32 or int64 [sequences, width]). An entry that is no page of the cache,
    or lies past the table's width, reads as zeros, as do rows in front of
    offsets[0]. `total` is the number of
    output rows, offsets[-1] or more; rows behind the last sequence are zeros,
    or with `out` (a tuple of tensors like the result, of any strides but the
    last) stay as they are."""
    out = None if out is None else tuple(out)
    _no_grad(scales, *(out or ()))
    c = _cache(codes, scales)
    if page_table.dtype not in _INTS or offsets.dtype not in _INTS:
        raise ValueError("page_table and offsets must be int32 or int64")
    if page_table.dim() != 2 or offsets.dim() != 1 or offsets.shape[0] != page_table.shape[0] + 1:
        raise DimensionMismatch("offsets must have one entry more than page_table has rows")
    if (page_table.shape[1] > 1 and page_table.stride(1) != 1) or (offsets.shape[0] > 1 and offsets.stride(0) != 1):
        raise ValueError("page_table rows and offsets must be contiguous")
    total = int(total)
    if total < 0:
        raise DimensionMismatch("total must not be negative")
    if out is not None:
        if len(out) != c.parts:
            raise DimensionMismatch(f"{len(out)} outputs for a cache of {c.parts} parts")
        dtype = out[0].dtype
        for x in out:
            _distinct(x, "out")
        given = _rows(out, total, c.heads, c.dim, dtype, "out")
    kind = _float_type(dtype, "out")
    device = _device(codes, scales, page_table, offsets, *(out or ()))

    def go(s):
        if out is not None:
            res, r = out, given
        else:
            res = tuple(torch.empty((total, c.heads, c.dim), dtype=dtype, device=codes.device) for _ in range(c.parts))
            r = _rows(res, total, c.heads, c.dim, dtype, "out")
        capi.check(_LIB.elips_b200_cache_read(
            device, ctypes.byref(c), page_table.data_ptr(), page_table.dtype == torch.int64, page_table.stride(0),
            page_table.shape[0], page_table.shape[1], offsets.data_ptr(), offsets.dtype == torch.int64, total, r,
            kind, out is None, s), "elips_b200_cache_read")
        return res

    return _run(go, stream, device, codes, scales, page_table, offsets, *(out or ()))
