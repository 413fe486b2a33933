"""CUDA tensors handed to the C ABI as bare addresses: what is checked before, and the streams they are used on."""
from __future__ import annotations


def as_stream(stream, device: int):
    """The torch stream of `stream` (a stream of torch's, an object with its handle as `cuda_stream`, or a handle) for
    work on `device`. The default stream's handle is 0, or 1 for the legacy one that it is; ExternalStream takes 0 for
    none given, and would make a new stream."""
    import torch
    if isinstance(stream, torch.cuda.Stream):
        if stream.device_index != device:
            raise ValueError(f"the stream is on cuda:{stream.device_index}, the tensors on cuda:{device}")
        return stream
    handle = stream if isinstance(stream, int) else stream.cuda_stream
    if handle in (0, 1):
        return torch.cuda.default_stream(device)
    return torch.cuda.ExternalStream(handle, device=device)


def device_rows(rows, dimension: int, dtype, device: int, what: str, stream=None):
    """`rows`, checked, as a tensor [n, dimension] of `dtype` on cuda:`device` whose rows follow one another: the entry points take
    an address and read n * dimension values from it. A view of other strides (rows of wider ones, such as the codes
    that quantize_rows gives; a broadcast row; a transpose) is copied, on `stream` where one is given."""
    import torch

    from .exact import DimensionMismatch
    if rows.dim() != 2 or rows.shape[1] != dimension:
        raise DimensionMismatch(f"{what} dimension does not match index")
    if rows.dtype is not dtype:
        raise ValueError(f"{what} rows must be {dtype}, not {rows.dtype}")
    if not rows.is_cuda or rows.get_device() != device:
        raise ValueError(f"{what} rows must be on cuda:{device}, the index's CUDA device, not on {rows.device}")
    if rows.is_contiguous():
        return rows
    if stream is None:
        return rows.contiguous()
    s = as_stream(stream, rows.get_device())
    with torch.cuda.stream(s):
        copy = rows.contiguous()
    rows.record_stream(s)
    return copy
