"""The cache operators where what is beside a row must not matter: scales that are not finite, words of an unwritten
cache that look like claims, and the memory around outputs."""
import numpy as np
import pytest
import torch

from tests import int8_oracle as R
from tests.test_gpu_int8 import FLOATS, activations, f32, filled, new_cache, rng

pytestmark = pytest.mark.gpu

# (parts, heads, dim): 16-byte stores, 8-byte, 4-byte and single ones, and the packed form of odd rows
SHAPES = [(2, 8, 128), (1, 3, 20), (2, 1, 66), (1, 5, 67), (2, 2, 9), (1, 1, 1537)]


def same(got, want, dtype):
    w = torch.from_numpy(want).to(dtype)
    return torch.equal(torch.isnan(got), torch.isnan(w)) and torch.equal(got.masked_fill(got.isnan(), 0), w.masked_fill(w.isnan(), 0))


@pytest.mark.parametrize("parts,heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("packed", [False, True])
def test_scales_that_are_not_finite(parts, heads, dim, dtype, packed):
    """Their rows are NaN where the code is 0 or the scale NaN and infinite elsewhere; the rows beside them are not
    touched. packed: into a fresh output, else into rows with room between them."""
    from elips_b200 import int8
    g = rng(parts, heads, dim, 21)
    codes, scales = filled(g, parts, 9, 4, heads, dim)
    codes[:, 2, 1] = 0
    at = torch.from_numpy(g.random(scales.shape)).cuda()
    for value, low in ((float("nan"), 0.0), (float("inf"), 0.1), (-float("inf"), 0.2), (0.0, 0.3)):
        scales[(at >= low) & (at < low + 0.1)] = value
    offsets, table = np.array([0, 11, 11, 30]), g.integers(0, 9, (3, 8))
    want = R.read_rows(codes.cpu().numpy(), scales.cpu().numpy(), table, offsets, 30, 4)
    td, od = torch.from_numpy(table).cuda().int(), torch.from_numpy(offsets).cuda()
    if packed:
        got = int8.cache_read(codes, scales, td, od, 30, dtype)
    else:
        out = tuple(torch.full((30, heads, dim + 5), 5.0, dtype=dtype, device="cuda")[..., 2:2 + dim] for _ in range(parts))
        got = int8.cache_read(codes, scales, td, od, 30, out=out)
    for p in range(parts):
        assert same(got[p].cpu(), want[p], dtype)


@pytest.mark.parametrize("t", [257, 300, 3000])
@pytest.mark.parametrize("heads,dim", [(2, 48), (1, 400), (1, 33)])
@pytest.mark.parametrize("words", ["any row", "own row", "next row", "last row", "past the rows"])
def test_unwritten_words_that_look_like_claims(t, heads, dim, words):
    """Scale words of a fresh buffer that hold just what a claim of some row of this call would be."""
    from elips_b200 import int8
    g = rng(t, heads, dim)
    slots = g.integers(-1, 90, t)
    slots[g.integers(0, t, 3)] = 96
    codes, scales = new_cache(2, 6, 16, heads, dim, fill=3)
    first = np.full(96, t - 1)                                     # each slot's first row, and what stands for it here
    for i in range(t - 1, -1, -1):
        if 0 <= slots[i] < 96:
            first[slots[i]] = i
    row = {"any row": g.integers(0, t, (2, 96, heads)), "own row": first[None, :, None], "next row": first[None, :, None] + 1,
           "last row": np.full((1, 1, 1), t - 1), "past the rows": np.full((1, 1, 1), t)}[words]
    held = (0x80000001 + np.broadcast_to(row, (2, 96, heads)).astype(np.int64)).astype(np.uint32).view(np.int32)
    scales.view(torch.int32).copy_(torch.from_numpy(held.copy()).view(2, 6, 16, heads))
    before = scales.clone()
    x = tuple(activations(g, (t, heads, dim), torch.bfloat16) for _ in range(2))
    int8.cache_write(codes, scales, x, torch.from_numpy(slots).cuda())
    last = {int(s): i for i, s in enumerate(slots) if 0 <= s < 96}
    q, s = np.full((2, 96, heads, dim), 3, np.int8), before.cpu().numpy().reshape(2, 96, heads).copy()
    for slot, i in last.items():
        for p in range(2):
            q[p, slot], s[p, slot] = R.quantize(f32(x[p][i]))
    assert np.array_equal(codes.cpu().numpy().reshape(q.shape), q)
    assert np.array_equal(scales.cpu().numpy().reshape(s.shape).view(np.int32), s.view(np.int32))


@pytest.mark.parametrize("parts,heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("total", [1, 9, 500])
def test_nothing_is_written_beside_outputs(parts, heads, dim, dtype, total):
    """Every value of the buffers that hold the outputs: rows with room between them, packed ones that start one value
    into the buffer or on 16 bytes, with rows behind the last sequence."""
    from elips_b200 import int8
    g = rng(parts, heads, dim, total)
    codes, scales = filled(g, parts, 9, 4, heads, dim)
    kept = total - total // 4
    offsets, table = np.array([0, kept // 3, kept]), g.integers(0, 9, (2, kept // 4 + 1))
    td, od = torch.from_numpy(table).cuda().int(), torch.from_numpy(offsets).cuda()
    want = R.read_rows(codes.cpu().numpy(), scales.cpu().numpy(), table, offsets, total, 4)
    for before, between in ((1, 3), (8, 8), (1, 0), (16, 0), (0, 0)):
        pitch = dim + between
        buffers = [torch.full((before + total * heads * pitch + 33,), 5.0, dtype=dtype, device="cuda") for _ in range(parts)]
        views = [b[before:before + total * heads * pitch].view(total, heads, pitch)[..., :dim] for b in buffers]
        int8.cache_read(codes, scales, td, od, total, out=tuple(views))
        for p in range(parts):
            expected = torch.full(buffers[p].shape, 5.0, dtype=dtype)
            expected[before:before + total * heads * pitch].view(total, heads, pitch)[:kept, :, :dim] = \
                torch.from_numpy(want[p][:kept]).to(dtype)
            assert torch.equal(buffers[p].cpu(), expected), (before, between, p)


@pytest.mark.parametrize("heads,dim", [(8, 128), (3, 67), (1, 200)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("t", [3, 300])
def test_nothing_is_written_beside_slots(heads, dim, dtype, t):
    """Codes and scales inside wider buffers, every other value of which stays."""
    from elips_b200 import int8
    g = rng(heads, dim, t, 5)
    pages, page = 50, 7
    for pad in (3, 16 + (-dim) % 16):
        store = torch.full((1, pages, page, heads, dim + 2 * pad), 77, dtype=torch.int8, device="cuda")
        held = torch.full((1, pages, page, heads + 2), 77.0, device="cuda")
        x = activations(g, (t, heads, dim), dtype)
        slots = g.permutation(pages * page)[:t]
        int8.cache_write(store[..., pad:pad + dim], held[..., 1:1 + heads], (x,), torch.from_numpy(slots).cuda())
        q, s = R.quantize(f32(x))
        want = np.full((pages * page, heads, dim + 2 * pad), 77, np.int8)
        want_held = np.full((pages * page, heads + 2), 77, np.float32)
        want[slots, :, pad:pad + dim] = q
        want_held[slots, 1:1 + heads] = s
        assert np.array_equal(store.cpu().numpy().reshape(want.shape), want)
        assert np.array_equal(held.cpu().numpy().reshape(want_held.shape), want_held)
