"""8-bit row operators on one B200, for the models around an index.

One format: a row x is held as int8 codes q and one fp32 scale s with
s = max|x| / 127 and q the integers nearest to x / s (ties to even), so x is
s * q to within s / 2. It is what every function here makes or reads:

  quantize_rows   rows -> codes, scales (activations per token, weights per
                  output channel)
  gemm_int8       codes x codes -> scaled products (a layer's output, or the
                  scores of queries against stored rows)
  linear_int8     rows x codes: quantize_rows and gemm_int8 in one call
  cache_write     rows quantised into the slots of a paged cache
  cache_read      sequences of pages back into packed rows

ExactIndex(precision="int8") ranks by the integer product of the codes alone. A
query's scale does not change its order, so quantize_rows makes its queries;
stored rows have to have one scale for all of them (round(x / s) for s the
largest magnitude of the whole base over 127). Rows with a scale each are scored
by gemm_int8 with those scales: without them they are ordered as if all had the
same largest value.

The reference has no such operators: its scalar quantiser has one affine scale
per dimension and scores by lookup (src/quant_engine/ScalarQuantizer.cpp:83-128).

Everything takes CUDA tensors, runs asynchronously on `stream` (default: the
current stream of the tensors' device) and can be captured into a CUDA graph.
With another stream the outputs belong to it and the inputs are held until its
work is done; ordering that work after the inputs are written is the caller's.
A product one of whose device-side waits expired (about a second; a lost load)
leaves its output unwritten without an error of its call: the next
elips_b200._capi.device_error(device) is not 0.
These are the serving forms: rounding has no gradient, so an input that
requires one is refused while gradients are recorded, and one with a tangent of
forward-mode differentiation always.

Rows that cannot be held: a row whose largest magnitude is below 127 * 2^-126
becomes zeros with scale 0; a row with an infinity or a NaN gets a scale that
is not finite and codes 0, reads back as NaN and gives NaN products, without
touching any other row.
"""
from __future__ import annotations

import contextlib
import struct

import torch
from torch.autograd import forward_ad as _forward
from torch.autograd.graph import increment_version as _increment_version  # a written tensor that autograd saved is stale

from . import _capi as capi
from ._device import as_stream
from .exact import DimensionMismatch

_LIB = capi.LIB
_TYPES = {torch.float32: capi.PRECISION_FP32, torch.float16: capi.PRECISION_FP16,
          torch.bfloat16: capi.PRECISION_BF16}
# The C structures, packed: on the host a small call costs little more than its
# launch, and ctypes structures or a dozen ctypes arguments would add to that.
_GEMM = struct.Struct("12q4i")
_CACHE = struct.Struct("15q")
_SEQUENCES = struct.Struct("6q2i")
_ROWS = (None, struct.Struct("3q"), struct.Struct("6q"))
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _refuse_grad() -> None:
    raise ValueError("8-bit operators have no gradient: detach the inputs or use torch.no_grad()")


def _refuse_tangents(*tensors) -> None:
    """Inside a level of forward-mode differentiation: refuses tensors with a tangent, which the result would lack.
    torch.no_grad() does not turn that mode off."""
    if any(t is not None and _forward.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("8-bit operators have no gradient: unpack the dual tensors first")


def _refuse_devices(*tensors) -> None:
    where = sorted({str(t.device) for t in tensors if t is not None})
    raise ValueError("tensors must be on one CUDA device, not on " + " and ".join(where))


def _float_type(dtype, what: str) -> int:
    kind = _TYPES.get(dtype)
    if kind is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, not {dtype}")
    return kind


def _pitch(t, what: str, apart: bool = True) -> int:
    """Checks a matrix with contiguous rows; elements from one row to the next
    (the width where there is no next). apart: rows must not overlap."""
    strides = t.stride()
    if len(strides) != 2:
        raise DimensionMismatch(f"{what} must have two axes")
    rows, width = t.shape
    pitch, step = strides
    if step != 1 and width > 1:
        raise ValueError(f"{what} must have contiguous rows")
    if rows < 2:
        return width or 1
    if apart and pitch < width:
        raise ValueError(f"rows of {what} overlap")
    return pitch


def _vector(t, n: int, what: str) -> int:
    """Checks n contiguous values; their address."""
    if t.shape != (n,):
        raise DimensionMismatch(f"{what} must have {n} entries")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return t.data_ptr()


@contextlib.contextmanager
def _using(stream, device: int, *tensors):
    """Makes `stream` current, so that what is allocated belongs to it, and
    keeps the tensors' memory until its work is done."""
    s = as_stream(stream, device)
    with torch.cuda.stream(s):
        yield
    for t in tensors:
        if t is not None:
            t.record_stream(s)


def quantize_rows(x, stream=None):
    """(codes int8 [n, d], scales float32 [n]) of float rows x [n, d]. The rows
    of codes start on multiples of 16 bytes (codes is a view of wider rows
    where d is no such multiple): gemm_int8 reads them as they are."""
    if x.requires_grad and torch.is_grad_enabled():
        _refuse_grad()
    if _forward._current_level >= 0:
        _refuse_tangents(x)
    kind = _float_type(x.dtype, "rows")
    pitch = _pitch(x, "rows", apart=False)
    n, d = x.shape
    if d == 0:
        raise DimensionMismatch("rows must have at least one value")
    device = x.get_device()
    if device < 0:
        _refuse_devices(x)
    if stream is not None:
        with _using(stream, device, x):
            return quantize_rows(x)
    wide = -(-d // 16) * 16
    codes = x.new_empty((n, wide), dtype=torch.int8)
    scales = x.new_empty(n, dtype=torch.float32)
    capi.check(_LIB.elips_b200_quantize_rows(device, x.data_ptr(), kind, n, d, pitch, codes.data_ptr(), wide,
                                             scales.data_ptr(), _raw_stream(device)), "elips_b200_quantize_rows")
    return (codes if wide == d else codes[:, :d]), scales


def _product(x, x_kind, x_scales, b, b_scales, bias, dtype, out, stream):
    """The product of rows x (codes with x_scales, or floats with None) with the
    n x k codes b: the checks, the output, the call."""
    codes = x_scales is not None
    pitch, b_pitch = _pitch(x, "rows", codes), _pitch(b, "weight codes")
    m, k = x.shape
    n, width = b.shape
    if width != k:
        raise DimensionMismatch(f"rows of {k} and of {width} values")
    if b.dtype is not torch.int8:
        raise ValueError(f"weight codes must be int8, not {b.dtype}")
    if b_scales.dtype is not torch.float32 or (codes and x_scales.dtype is not torch.float32):
        raise ValueError("scales must be float32")
    x_scales_at = _vector(x_scales, m, "row scales") if codes else 0
    b_scales_at = _vector(b_scales, n, "weight scales")
    bias_at = bias_kind = 0
    if bias is not None:
        bias_kind = _float_type(bias.dtype, "bias")
        bias_at = _vector(bias, n, "bias")
    if out is not None:
        dtype = out.dtype
        out_pitch = _pitch(out, "out")
        if out.shape != (m, n):
            raise DimensionMismatch(f"out must be {m} x {n}")
    kind = _TYPES.get(dtype)
    if kind is None:
        _float_type(dtype, "out")
    if torch.is_grad_enabled() and (b_scales.requires_grad or x.requires_grad or (codes and x_scales.requires_grad) or
                                    (bias is not None and bias.requires_grad) or (out is not None and out.requires_grad)):
        _refuse_grad()
    if _forward._current_level >= 0:
        _refuse_tangents(x, x_scales, b_scales, bias, out)
    device = x.get_device()
    if device < 0 or b.get_device() != device or b_scales.get_device() != device or \
            (codes and x_scales.get_device() != device) or \
            (bias is not None and bias.get_device() != device) or (out is not None and out.get_device() != device):
        _refuse_devices(x, b, x_scales, b_scales, bias, out)
    if stream is not None:
        with _using(stream, device, x, b, x_scales, b_scales, bias, out):
            return _product(x, x_kind, x_scales, b, b_scales, bias, dtype, out, None)
    fresh = out is None
    if fresh:
        out = x.new_empty((m, n), dtype=dtype)
        out_pitch = n or 1
    status = _LIB.elips_b200_gemm_int8(
        device, _GEMM.pack(x.data_ptr(), x_scales_at, b.data_ptr(), b_scales_at, bias_at, out.data_ptr(), m, n, k, pitch,
                           b_pitch, out_pitch, x_kind, bias_kind, kind, 0), _raw_stream(device))
    if status:
        capi.check(status, "elips_b200_gemm_int8")
    if not fresh:
        _increment_version(out)
    return out


def gemm_int8(a, b, a_scales, b_scales, bias=None, out_dtype=torch.bfloat16, out=None, stream=None):
    """out[i, j] = (sum_l a[i, l] b[j, l]) * a_scales[i] * b_scales[j] + bias[j],
    the sum exact in int32 (so the width is below 2^17). The sum's conversion to
    fp32, its product with a_scales, the fused b_scales and bias, and out's type
    round once each, in this order.

    a [m, k] and b [n, k] are int8 with contiguous rows, as quantize_rows gives
    them: a activations and b a layer's weight with a scale per channel, or a
    queries and b stored rows. Operands whose rows start on multiples of 16
    bytes are read as they are, others are copied to such rows first. bias
    [n] may have another float type than out. An out that shares memory with an
    input is refused (columns side by side in one buffer share none)."""
    if a.dtype is not torch.int8:
        raise ValueError(f"row codes must be int8, not {a.dtype}")
    return _product(a, capi.PRECISION_INT8, a_scales, b, b_scales, bias, out_dtype, out, stream)


def linear_int8(x, weight, weight_scales, bias=None, out_dtype=None, out=None, stream=None):
    """gemm_int8 over the rows of x [m, k], quantised on the way as
    quantize_rows quantises them; out_dtype defaults to x's type. x cannot be
    its own out."""
    dtype = x.dtype
    kind = _float_type(dtype, "rows")
    if x.numel() == 0 and x.shape[-1:] == (0,):
        raise DimensionMismatch("rows must have at least one value")
    return _product(x, kind, None, weight, weight_scales, bias, dtype if out_dtype is None else out_dtype, out, stream)


def _distinct(strides, shape, what: str) -> None:
    """Refuses a tensor to be written whose elements share memory by a stride of 0."""
    if 0 in strides and any(st == 0 and n > 1 for st, n in zip(strides, shape)):
        raise ValueError(f"{what} must not be an expanded tensor")


def _cache(codes, scales, written: bool):
    """The packed elips_b200_cache of a cache's two tensors, and its shape."""
    if codes.dtype is not torch.int8 or scales.dtype is not torch.float32:
        raise ValueError("a cache has int8 codes and float32 scales")
    shape, held = codes.shape, scales.shape
    if len(shape) != 5 or held != shape[:4]:
        raise DimensionMismatch("codes must be [parts, pages, page, heads, dim] and scales [parts, pages, page, heads]")
    parts, pages, page, heads, dim = shape
    if not 1 <= parts <= 2:
        raise DimensionMismatch("a cache has one or two parts")
    if page < 1 or heads < 1 or dim < 1:
        raise DimensionMismatch("pages, heads and rows must not be empty")
    s0, s1, s2, s3, s4 = strides = codes.stride()
    if s4 != 1 and dim > 1:
        raise ValueError("rows of codes must be contiguous")
    t0, t1, t2, t3 = scale_strides = scales.stride()
    if written:
        _distinct(strides, shape, "codes")
        _distinct(scale_strides, held, "scales")
    return _CACHE.pack(codes.data_ptr(), scales.data_ptr(), parts, pages, page, heads, dim, s0, s1, s2, s3, t0, t1, t2,
                       t3), parts, heads, dim


def _rows(tensors, count: int, heads: int, dim: int, dtype, what: str, written: bool):
    """The packed elips_b200_rows of a part's rows [count, heads, dim], for each part."""
    want, packed = (count, heads, dim), []
    for x in tensors:
        if x.shape != want:
            raise DimensionMismatch(f"{what} must be {list(want)}, not {list(x.shape)}")
        if x.dtype is not dtype:
            raise ValueError(f"{what} must be {dtype}, not {x.dtype}")
        s0, s1, s2 = strides = x.stride()
        if s2 != 1 and dim > 1:
            raise ValueError(f"{what} must have their last axis contiguous")
        if written:
            _distinct(strides, want, what)
        packed += (x.data_ptr(), s0, s1)
    return _ROWS[len(tensors)].pack(*packed)


def _indexes(t, what: str) -> int:
    """1 for int64, 0 for int32."""
    if t.dtype is torch.int64:
        return 1
    if t.dtype is not torch.int32:
        raise ValueError(f"{what} must be int32 or int64, not {t.dtype}")
    return 0


def cache_write(codes, scales, rows, slots, stream=None) -> None:
    """Quantises rows into the slots of a paged cache, in place.

    codes int8 [parts, pages, page, heads, dim] and scales float32 [parts,
    pages, page, heads] are the cache: one part holds one kind of row, two hold
    keys and values. rows is a tuple of one float tensor [t, heads, dim] per
    part; each of its rows gets a scale per head. Row i goes to slot slots[i]
    (int32 or int64): row s % page of page s // page. A slot below 0 or past
    the last one is skipped (padding); of a slot given twice the last row is
    kept. Slots that are not named stay as they are. A cache that shares memory
    with rows or slots is refused."""
    cache, parts, heads, dim = _cache(codes, scales, True)
    if len(rows) != parts:
        raise DimensionMismatch(f"{len(rows)} tensors of rows for a cache of {parts} parts")
    wide = _indexes(slots, "slots")
    if slots.dim() != 1 or not slots.is_contiguous():
        raise DimensionMismatch("slots must be one contiguous axis")
    t = slots.numel()
    dtype = rows[0].dtype
    kind = _float_type(dtype, "rows")
    packed = _rows(rows, t, heads, dim, dtype, "rows", False)
    if torch.is_grad_enabled() and (scales.requires_grad or rows[0].requires_grad or rows[-1].requires_grad):
        _refuse_grad()
    if _forward._current_level >= 0:
        _refuse_tangents(scales, *rows)
    device = codes.get_device()
    if device < 0 or scales.get_device() != device or slots.get_device() != device or \
            rows[0].get_device() != device or rows[-1].get_device() != device:
        _refuse_devices(codes, scales, slots, *rows)
    if stream is not None:
        with _using(stream, device, codes, scales, slots, *rows):
            return cache_write(codes, scales, rows, slots)
    status = _LIB.elips_b200_cache_write(device, cache, packed, kind, t, slots.data_ptr(), wide, _raw_stream(device))
    if status:
        capi.check(status, "elips_b200_cache_write")
    _increment_version((codes, scales))


def cache_read(codes, scales, page_table, offsets, total: int, dtype=torch.bfloat16, out=None, stream=None):
    """Sequences of cached rows, packed: a tuple of one tensor [total, heads,
    dim] per part.

    Sequence b is the output rows offsets[b] .. offsets[b + 1] (offsets
    ascending, one more entry than there are sequences, int32 or int64);
    position i of it is read from row i % page of page page_table[b, i // page]
    (int32 or int64 [sequences, width]). An entry that is no page of the cache,
    or lies past the table's width, reads as zeros, as do rows in front of
    offsets[0]. `total` is the number of output rows, offsets[-1] or more; rows
    behind the last sequence are zeros, or with `out` (a tuple of tensors like
    the result, of any strides but the last) stay as they are. Outputs that
    share memory with one another or with what is read are refused."""
    cache, parts, heads, dim = _cache(codes, scales, False)
    table_wide, offsets_wide = _indexes(page_table, "page_table"), _indexes(offsets, "offsets")
    shape = page_table.shape
    if len(shape) != 2 or offsets.shape != (shape[0] + 1,):
        raise DimensionMismatch("offsets must have one entry more than page_table has rows")
    sequences, width = shape
    table_stride, step = page_table.stride()
    if (width > 1 and step != 1) or not offsets.is_contiguous():
        raise ValueError("page_table rows and offsets must be contiguous")
    total = int(total)
    if total < 0:
        raise DimensionMismatch("total must not be negative")
    fresh = out is None
    if not fresh:
        out = tuple(out)
        if len(out) != parts:
            raise DimensionMismatch(f"{len(out)} outputs for a cache of {parts} parts")
        dtype = out[0].dtype
        packed = _rows(out, total, heads, dim, dtype, "out", True)
    kind = _float_type(dtype, "out")
    if torch.is_grad_enabled() and (scales.requires_grad or (not fresh and any(x.requires_grad for x in out))):
        _refuse_grad()
    if _forward._current_level >= 0:
        _refuse_tangents(scales, *(out or ()))
    device = codes.get_device()
    if device < 0 or scales.get_device() != device or page_table.get_device() != device or \
            offsets.get_device() != device or (not fresh and any(x.get_device() != device for x in out)):
        _refuse_devices(codes, scales, page_table, offsets, *(out or ()))
    if stream is not None:
        with _using(stream, device, codes, scales, page_table, offsets, *(out or ())):
            return cache_read(codes, scales, page_table, offsets, total, dtype, out)
    if fresh:
        size, row = (total, heads, dim), heads * dim
        first = codes.new_empty(size, dtype=dtype)
        if parts == 1:
            out = (first,)
            packed = _ROWS[1].pack(first.data_ptr(), row, dim)
        else:
            second = codes.new_empty(size, dtype=dtype)
            out = (first, second)
            packed = _ROWS[2].pack(first.data_ptr(), row, dim, second.data_ptr(), row, dim)
    seqs = _SEQUENCES.pack(page_table.data_ptr(), offsets.data_ptr(), table_stride, sequences, width, total, table_wide,
                           offsets_wide)
    status = _LIB.elips_b200_cache_read(device, cache, seqs, packed, kind, fresh, _raw_stream(device))
    if status:
        capi.check(status, "elips_b200_cache_read")
    if not fresh:
        _increment_version(out)
    return out
