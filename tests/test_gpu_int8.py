"""The 8-bit row operators (elips_b200.int8) against numpy in 64 bits (tests/int8_oracle.py).

Codes and scales have to be equal; products are held to the roundings that their formula makes, each at most half a
step of its type, counted in int8_oracle.gemm_bound; cached rows read back as one fp32 product rounded once, equal."""
import numpy as np
import pytest
import torch

from tests import int8_oracle as R

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def rng(*seed):
    return np.random.default_rng([17, *seed])


def f32(t):
    return t.detach().float().cpu().numpy()


def activations(g, shape, dtype):
    """Normal values, a few channels far larger, rows of very different size; on the device in `dtype`."""
    x = g.standard_normal(shape).astype(np.float32)
    x *= np.where(g.random(shape[-1]) < 0.02, 30, 1).astype(np.float32)
    x *= np.exp(g.uniform(-8, 6, shape[:-1] + (1,))).astype(np.float32)
    return torch.from_numpy(x).cuda().to(dtype)


def assert_rows(codes, scales, x):
    q, s = R.quantize(f32(x))
    assert np.array_equal(scales.cpu().numpy(), s, equal_nan=True)
    assert np.array_equal(codes.cpu().numpy(), q)


# ------------------------------------------------------------------ quantize_rows

@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("n,d", [(1, 1), (3, 2), (1, 4096), (70, 7), (33, 16), (100, 64), (257, 100), (64, 127), (65, 128),
                                 (31, 256), (9, 768), (5, 1000), (200, 1024), (7, 4096), (3, 8193), (2, 40001),
                                 (20000, 24)])
def test_quantize_rows(n, d, dtype):
    from elips_b200 import int8
    x = activations(rng(n, d), (n, d), dtype)
    codes, scales = int8.quantize_rows(x)
    assert codes.stride(0) % 16 == 0 or n == 1
    assert_rows(codes, scales, x)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("first,step", [(0, 24), (1, 24), (4, 23), (8, 48)])
def test_quantize_rows_of_a_wider_matrix(first, step, dtype):
    """Rows inside wider ones, starting anywhere: 16-byte aligned and not."""
    from elips_b200 import int8
    wide = activations(rng(first, step), (40, 4 * step), dtype)
    x = wide[:, first:first + step]
    assert_rows(*int8.quantize_rows(x), x)
    assert_rows(*int8.quantize_rows(x[::3]), x[::3])
    row = x[5].expand(6, step)                      # a broadcast row
    assert_rows(*int8.quantize_rows(row), row)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("n,d", [(3, 1), (40, 3), (7, 30), (2000, 31), (5, 250), (3000, 500), (5, 2000), (1200, 3000),
                                 (2, 5001), (3, 9000), (2, 33001)])
def test_quantize_rows_beside_nan(n, d, dtype):
    """Rows that start anywhere in wider ones whose other values are NaN and infinities; nothing written beside them."""
    from elips_b200 import _capi, int8
    wide = torch.full((n, d + 11), float("nan"), dtype=dtype, device="cuda")
    wide[:, ::2] = float("inf")
    for first in range(0, 9, 2 if d > 1000 else 1):
        wide[:, first:first + d] = activations(rng(n, d, first), (n, d), dtype)
        x = wide[:, first:first + d]
        assert_rows(*int8.quantize_rows(x), x)
        codes, scales = torch.full((n, d + 40), 99, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
        pitch = d + 40 if (d + 40) % 8 == 0 else (d + 40) // 8 * 8
        _capi.check(_capi.LIB.elips_b200_quantize_rows(
            0, x.data_ptr(), int8._TYPES[dtype], n, d, x.stride(0), codes.data_ptr(), pitch, scales.data_ptr(),
            torch.cuda.current_stream().cuda_stream), "quantize")
        got = codes.flatten()[:n * pitch].view(n, pitch)
        assert_rows(got[:, :d], scales, x)
        assert (got[:, d:] == 99).all()
        wide[:, first:first + d] = float("nan")


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("d", [40, 64, 513])
def test_quantize_values_next_to_a_border(d, dtype):
    """Values that are halves of the scale exactly, and their neighbours on both sides: the nearest integer, ties to
    even."""
    from elips_b200 import int8
    g = rng(d)
    rows = []
    for top in (127.0, 254.0, 127.0 * 2.0 ** -20, 96.5, 3.1, 2e-36 if dtype != torch.float16 else 7e-6, 1e-30 if dtype != torch.float16 else 1e-3, 60000.0):
        top = float(torch.tensor(top).to(dtype))
        s = np.float32(top) / np.float32(127)
        half = torch.from_numpy(((g.integers(-127, 127, d) + 0.5) * np.float64(s)).astype(np.float32)).to(dtype)
        for x in (half, torch.nextafter(half, torch.full_like(half, 1e38 if dtype != torch.float16 else 6e4)),
                  torch.nextafter(half, torch.full_like(half, -1e38 if dtype != torch.float16 else -6e4))):
            x = x.clone().clamp_(-top, top)
            x[g.integers(d)] = top
            rows.append(x)
    x = torch.stack(rows).cuda()
    assert_rows(*int8.quantize_rows(x), x)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantize_every_value_of_a_16_bit_type(dtype):
    """Rows that hold every magnitude up to their largest: whichever side of a half the stored scale puts a value."""
    from elips_b200 import int8
    count = 0x7C00 if dtype == torch.float16 else 0x7F80        # finite magnitudes, in ascending order of their bits
    every = torch.arange(count, dtype=torch.int32, device="cuda").to(torch.int16).view(dtype)
    tops = torch.arange(11 if dtype == torch.float16 else 1200, count, 487, device="cuda")
    x = torch.where(torch.arange(count, device="cuda") <= tops[:, None], every, torch.zeros_like(every))
    x[:, ::2] *= -1
    codes, scales = int8.quantize_rows(x)
    assert_rows(codes, scales, x)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("d", [5, 32, 384])
def test_quantize_rows_that_cannot_be_held(d, dtype):
    """Zeros, values too small for a scale, the largest ones, infinities and NaN: each stays in its own row."""
    from elips_b200 import int8
    info = torch.finfo(dtype)
    x = torch.ones((9, d), dtype=dtype)
    x[1] = 0
    x[2] = info.max
    x[2, 0] = info.min
    x[3] = info.tiny
    x[4, d // 2] = float("inf")
    x[5, 0] = -float("inf")
    x[6, d - 1] = float("nan")
    x[7] = torch.tensor(-0.0, dtype=dtype)
    x[8] = info.smallest_normal if dtype == torch.float16 else info.tiny * 0.25
    codes, scales = int8.quantize_rows(x.cuda())
    q, s = R.quantize(f32(x))
    assert np.array_equal(codes.cpu().numpy(), q)
    assert np.array_equal(scales.cpu().numpy(), s, equal_nan=True)
    sc = scales.cpu()
    assert sc[1] == 0 and sc[7] == 0 and torch.isinf(sc[4]) and torch.isinf(sc[5]) and torch.isnan(sc[6])
    assert (codes.cpu()[4:7] == 0).all()
    back = codes.float() * scales[:, None]
    assert torch.isnan(back[4:7]).all() and torch.isfinite(back[[0, 1, 2, 3, 7, 8]]).all()


def test_quantize_no_rows():
    from elips_b200 import int8
    codes, scales = int8.quantize_rows(torch.empty((0, 64), device="cuda"))
    assert codes.shape == (0, 64) and scales.shape == (0,)


# ---------------------------------------------------------------------- gemm_int8

def operand(g, rows, k, pitch, full=False):
    """int8 codes [rows, k] whose rows are a multiple of `pitch` bytes apart (1: starting one byte off as well)."""
    wide = -(-k // pitch) * pitch
    c = g.integers(-128, 128, (rows, wide)) if full else np.clip(np.rint(g.standard_normal((rows, wide)) * 40), -127, 127)
    c = torch.from_numpy(c.astype(np.int8)).cuda()
    if pitch == 1:
        flat = torch.zeros(rows * wide + 1, dtype=torch.int8, device="cuda")
        flat[1:] = c.flatten()
        c = flat[1:].view(rows, wide)
    return c[:, :k]


def gemm_case(m, n, k, out, bias=None, pitch=16, full=False):
    g = rng(m, n, k)
    a, b = operand(g, m, k, pitch, full), operand(g, n, k, pitch, full)
    sa = torch.from_numpy(np.exp(g.uniform(-9, 3, m)).astype(np.float32)).cuda()
    sb = torch.from_numpy(np.exp(g.uniform(-9, 3, n)).astype(np.float32)).cuda()
    bv = None if bias is None else torch.from_numpy(g.standard_normal(n).astype(np.float32)).cuda().to(bias)
    return a, b, sa, sb, bv


def assert_product(c, a, b, sa, sb, bias, dtype):
    assert c.dtype == dtype
    v = R.gemm(a.cpu().numpy(), b.cpu().numpy(), f32(sa), f32(sb), None if bias is None else f32(bias))
    off = np.abs(c.double().cpu().numpy() - v)
    bound = R.gemm_bound(v, None if bias is None else f32(bias), torch.finfo(dtype).eps)
    if dtype == torch.float16:
        bound = np.maximum(bound, 2.0 ** -25)            # half a step of the type's smallest numbers
        fits = np.abs(v) < 65000
        off, bound = off[fits], bound[fits]
    assert (off <= bound).all(), float((off / bound).max())


SIZES = [(1, 1, 1), (1, 10, 33), (1, 128, 128), (1, 1000, 768), (2, 17, 4096), (3, 129, 640), (5, 4096, 129), (8, 300, 2048),
         (9, 257, 96), (16, 128, 4096), (17, 130, 127), (31, 999, 1025), (33, 64, 5000), (64, 1000, 384), (65, 65, 65),
         (100, 300, 16), (127, 127, 300), (128, 128, 128), (129, 257, 255), (200, 4100, 512), (255, 255, 2049),
         (256, 256, 256), (257, 513, 64), (300, 1001, 1111), (512, 512, 100), (700, 1, 700), (1000, 3, 70), (1025, 900, 320),
         (2000, 1300, 130), (4097, 260, 31), (64, 20000, 200), (20, 40001, 70), (512, 4096, 300), (2048, 2560, 260),
         (1500, 2050, 1500), (2600, 2600, 700), (130, 12000, 64)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("pitch", [16, 1])
def test_gemm_sizes(m, n, k, pitch):
    from elips_b200 import int8
    dtype = FLOATS[(m + n + k) % 3]
    a, b, sa, sb, _ = gemm_case(m, n, k, dtype, pitch=pitch)
    assert_product(int8.gemm_int8(a, b, sa, sb, out_dtype=dtype), a, b, sa, sb, None, dtype)


@pytest.mark.parametrize("m,n,k", [(1, 300, 500), (20, 77, 512), (150, 130, 200), (513, 1024, 1024)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("bias", [None, *FLOATS])
def test_gemm_types(m, n, k, dtype, bias):
    from elips_b200 import int8
    a, b, sa, sb, bv = gemm_case(m, n, k, dtype, bias, full=True)
    assert_product(int8.gemm_int8(a, b, sa, sb, bv, out_dtype=dtype), a, b, sa, sb, bv, dtype)


@pytest.mark.parametrize("m,n", [(1, 5), (20, 40), (140, 260)])
@pytest.mark.parametrize("k", [131071, 65537])
def test_gemm_largest_sums(m, n, k):
    """Every product 2^14 and k just below 2^17: the sum is 2^31 - 2^14, and with the other sign its negative."""
    from elips_b200 import int8
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    b[n // 2:] = 127
    one = torch.ones(max(m, n), device="cuda")
    c = int8.gemm_int8(a, b, one[:m], one[:n], out_dtype=torch.float32)
    assert_product(c, a, b, one[:m], one[:n], None, torch.float32)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_gemm_no_width_and_no_rows(m):
    from elips_b200 import int8
    empty = lambda r, k: torch.empty((r, k), dtype=torch.int8, device="cuda")  # noqa: E731
    s = torch.ones(m, device="cuda")
    bias = torch.arange(6, device="cuda").float()
    c = int8.gemm_int8(empty(m, 0), empty(6, 0), s, torch.ones(6, device="cuda"), bias, out_dtype=torch.float32)
    assert torch.equal(c, bias.expand(m, 6))
    none = torch.empty(0, device="cuda")
    assert int8.gemm_int8(empty(0, 32), empty(6, 32), none, torch.ones(6, device="cuda")).shape == (0, 6)
    assert int8.gemm_int8(empty(m, 32), empty(0, 32), s, none).shape == (m, 0)


@pytest.mark.parametrize("m,n,k", [(4, 70, 64), (30, 150, 640), (300, 500, 256)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("first", [0, 3])
def test_gemm_into_a_wider_matrix(m, n, k, dtype, first):
    """Only the named columns of `out` are written; NaN and infinite scales stay in their rows and columns."""
    from elips_b200 import int8
    a, b, sa, sb, _ = gemm_case(m, n, k, dtype)
    sa[m // 2], sb[n // 3] = float("nan"), float("inf")
    wide = torch.full((m, n + 11), 7.0, dtype=dtype, device="cuda")
    out = wide[:, first:first + n]
    assert int8.gemm_int8(a, b, sa, sb, out=out) is out
    assert (wide[:, :first] == 7).all() and (wide[:, first + n:] == 7).all()
    rows = [i for i in range(m) if i != m // 2]
    cols = [j for j in range(n) if j != n // 3]
    assert torch.isnan(out[m // 2]).all()
    acc = a.cpu().double() @ b.cpu().double().t()
    assert not torch.isfinite(out[rows, n // 3].cpu()[acc[rows, n // 3] != 0]).any()
    pick = lambda t: t[rows][:, cols]  # noqa: E731
    assert_product(pick(out), a[rows], b[cols], sa[rows], sb[cols], None, dtype)


def test_gemm_operand_views():
    """Rows of every second layer row, an operand that is a view with a large pitch, a single row of a matrix."""
    from elips_b200 import int8
    g = rng(5)
    big_a, big_b = operand(g, 80, 512, 16), operand(g, 500, 1024, 16)
    a, b = big_a[::2, 32:32 + 200], big_b[100:400:3, 16:216]
    sa, sb = torch.rand(40, device="cuda") + 0.1, torch.rand(100, device="cuda") + 0.1
    assert_product(int8.gemm_int8(a, b, sa, sb, out_dtype=torch.float32), a, b, sa, sb, None, torch.float32)
    a1 = a[7:8]
    assert_product(int8.gemm_int8(a1, b, sa[7:8], sb, out_dtype=torch.float32), a1, b, sa[7:8], sb, None, torch.float32)


def test_gemm_offsets_past_32_bits():
    """Operand and output rows that lie past 2^31 and 2^32 bytes."""
    from elips_b200 import int8
    m, k, n = 70000, 64, 9
    a = torch.zeros((m, 65536), dtype=torch.int8, device="cuda")[:, :k]
    rows = torch.tensor([0, 1, 32767, 32768, 65535, 65536, m - 1], device="cuda")
    g = rng(6)
    a[rows] = operand(g, rows.numel(), k, 16)
    b, sb = operand(g, n, k, 16), torch.rand(n, device="cuda") + 0.1
    sa = torch.rand(m, device="cuda") + 0.1
    c = int8.gemm_int8(a, b, sa, sb, out_dtype=torch.float32)
    assert_product(c[rows], a[rows], b, sa[rows], sb, None, torch.float32)
    out = torch.zeros((m, 32768), dtype=torch.float32, device="cuda")[:, :n]
    int8.gemm_int8(a, b, sa, sb, out=out)
    assert torch.equal(out, c)


# -------------------------------------------------------------------- linear_int8

@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 96, 768), (1, 1000, 4096), (2, 333, 1001), (4, 512, 2048), (7, 130, 128),
                                   (8, 64, 5000), (9, 200, 333), (24, 1536, 384), (130, 140, 150), (600, 300, 768)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_linear_is_quantize_then_gemm(m, n, k, dtype):
    from elips_b200 import int8
    g = rng(m, n, k)
    x = activations(g, (m, k), dtype)
    w, sw = operand(g, n, k, 16), torch.from_numpy(np.exp(g.uniform(-6, 0, n)).astype(np.float32)).cuda()
    bias = torch.from_numpy(g.standard_normal(n).astype(np.float32)).cuda().to(dtype)
    c = int8.linear_int8(x, w, sw, bias, out_dtype=torch.float32)
    q, s = R.quantize(f32(x))
    v = R.gemm(q, w.cpu().numpy(), s, f32(sw), f32(bias))
    off = np.abs(c.double().cpu().numpy() - v)
    assert (off <= R.gemm_bound(v, f32(bias), torch.finfo(torch.float32).eps)).all()
    assert torch.equal(c, int8.gemm_int8(*[t for t in (int8.quantize_rows(x)[0], w, int8.quantize_rows(x)[1], sw)], bias,
                                         out_dtype=torch.float32))
    assert int8.linear_int8(x, w, sw).dtype == dtype


@pytest.mark.parametrize("m", [1, 5, 40])
def test_linear_rows_that_cannot_be_held(m):
    """A NaN in one row of the batch: that row is NaN, the others as without it; a zero row gives the bias."""
    from elips_b200 import int8
    g = rng(m, 3)
    x = activations(g, (m + 2, 300), torch.bfloat16)
    w, sw = operand(g, 70, 300, 16), torch.rand(70, device="cuda") + 0.1
    bias = torch.rand(70, device="cuda")
    ref = int8.linear_int8(x, w, sw, bias, out_dtype=torch.float32)
    x[m, 17], x[m + 1] = float("nan"), 0
    c = int8.linear_int8(x, w, sw, bias, out_dtype=torch.float32)
    assert torch.equal(c[:m], ref[:m]) and torch.isnan(c[m]).all() and torch.equal(c[m + 1], bias)


@pytest.mark.parametrize("m", [1, 6, 40])
@pytest.mark.parametrize("first", [0, 1])
def test_linear_views(m, first):
    """Rows that are slices of wider ones, aligned and not; weight rows of any pitch."""
    from elips_b200 import int8
    g = rng(m, first)
    wide = activations(g, (m, 900), torch.float16)
    x = wide[:, first:first + 640]
    w = operand(g, 50, 640, 1 if first else 16)
    sw = torch.rand(50, device="cuda") + 0.1
    c = int8.linear_int8(x, w, sw, out_dtype=torch.float32)
    q, s = R.quantize(f32(x))
    v = R.gemm(q, w.cpu().numpy(), s, f32(sw))
    assert (np.abs(c.double().cpu().numpy() - v) <= R.gemm_bound(v, None, 2.0 ** -23)).all()


# -------------------------------------------------------------------------- cache

def new_cache(parts, pages, page, heads, dim, fill=0):
    wide = -(-dim // 16) * 16
    codes = torch.full((parts, pages, page, heads, wide), fill, dtype=torch.int8, device="cuda")[..., :dim]
    return codes, torch.full((parts, pages, page, heads), float(fill), device="cuda")


CACHES = [(1, 1, 64), (1, 1, 1), (1, 1, 768), (1, 3, 67), (2, 8, 128), (2, 2, 80), (2, 1, 576), (1, 5, 200), (2, 4, 256),
          (1, 1, 1537), (2, 16, 16)]


def assert_slots(codes, scales, want):
    """Every slot of the cache: `want` maps (part, slot) to float rows [heads, dim]; the others hold 3 / 3.0."""
    parts, pages, page, heads, dim = codes.shape
    q = np.full((parts, pages * page, heads, dim), 3, np.int8)
    s = np.full((parts, pages * page, heads), 3, np.float32)
    for (p, slot), x in want.items():
        q[p, slot], s[p, slot] = R.quantize(x)
    assert np.array_equal(codes.cpu().numpy().reshape(q.shape), q)
    assert np.array_equal(scales.cpu().numpy().reshape(s.shape), s, equal_nan=True)


@pytest.mark.parametrize("parts,heads,dim", CACHES)
@pytest.mark.parametrize("t", [1, 3, 41, 300])
@pytest.mark.parametrize("dtype", FLOATS)
def test_cache_write_slots(parts, heads, dim, t, dtype):
    """Each row in its slot, padding and slots outside the cache skipped, every other slot as it was."""
    from elips_b200 import int8
    g = rng(parts, heads, dim, t)
    page, pages = 7, 50
    codes, scales = new_cache(parts, pages, page, heads, dim, fill=3)
    x = tuple(activations(g, (t, heads, dim), dtype) for _ in range(parts))
    slots = g.permutation(pages * page)[:t].astype(np.int64)
    if t > 2:
        slots[g.integers(0, t, t // 4 + 1)] = -1
        slots[0] = pages * page
    kind = torch.int32 if t % 2 else torch.int64
    int8.cache_write(codes, scales, x, torch.from_numpy(slots).cuda().to(kind))
    assert_slots(codes, scales, {(p, int(s)): f32(x[p][i]) for p in range(parts) for i, s in enumerate(slots)
                                 if 0 <= s < pages * page})


@pytest.mark.parametrize("t", [2, 40, 200, 257, 2500])
@pytest.mark.parametrize("heads,dim", [(2, 48), (1, 400)])
def test_cache_write_slot_given_twice_keeps_the_last_row(t, heads, dim):
    from elips_b200 import int8
    g = rng(t, heads)
    codes, scales = new_cache(2, 3, 16, heads, dim, fill=3)
    scales.view(torch.int32).fill_(-1)               # whatever the scales held before
    scales[:] = 3
    scales[0, 0, 0] = -5.0
    x = tuple(activations(g, (t, heads, dim), torch.bfloat16) for _ in range(2))
    slots = g.integers(-2, 48, t)
    slots[-1] = 0
    int8.cache_write(codes, scales, x, torch.from_numpy(slots).cuda())
    assert_slots(codes, scales, {(p, int(s)): f32(x[p][i]) for p in range(2) for i, s in enumerate(slots) if s >= 0})


@pytest.mark.parametrize("fill", [float("nan"), -1.0, float("-inf"), -0.0])
@pytest.mark.parametrize("t", [5, 400])
def test_cache_write_over_any_scales(fill, t):
    """Scales that no write left behind (an uninitialised buffer) do not matter."""
    from elips_b200 import int8
    codes, scales = new_cache(1, 400, 1, 2, 32)
    scales.fill_(fill)
    x = activations(rng(t), (t, 2, 32), torch.float32)
    int8.cache_write(codes, scales, (x,), torch.arange(t, device="cuda"))
    q, s = R.quantize(f32(x))
    assert np.array_equal(codes[0, :t, 0].cpu().numpy(), q) and np.array_equal(scales[0, :t, 0].cpu().numpy(), s)


def test_cache_write_views():
    """Keys and values as slices of one projection's rows, into one layer of a cache of many layers."""
    from elips_b200 import int8
    g = rng(8)
    t, heads, dim = 37, 4, 64
    qkv = activations(g, (t, 3 * heads * dim + 8), torch.bfloat16)
    for first in (heads * dim, heads * dim + 3):     # 16-byte aligned rows and others
        k = qkv[:, first:first + heads * dim].view(t, heads, dim)
        v = qkv[:, first + heads * dim - 3:][:, :heads * dim].view(t, heads, dim)
        layers = torch.full((3, 2, 5, 8, heads, dim), 3, dtype=torch.int8, device="cuda")
        scales = torch.full((3, 2, 5, 8, heads), 3.0, device="cuda")
        slots = torch.from_numpy(g.permutation(40)[:t]).cuda()
        int8.cache_write(layers[1], scales[1], (k, v), slots)
        assert_slots(layers[1], scales[1], {(p, int(s)): f32(x[i]) for p, x in enumerate((k, v))
                                            for i, s in enumerate(slots.tolist())})
        assert (layers[[0, 2]] == 3).all() and (scales[[0, 2]] == 3).all()
    # heads before rows, and the cache's heads before its pages
    x = activations(g, (heads, t, dim), torch.float16).transpose(0, 1)
    store = torch.full((1, heads, 5, 8, dim), 3, dtype=torch.int8, device="cuda").permute(0, 2, 3, 1, 4)
    held = torch.full((1, heads, 5, 8), 3.0, device="cuda").permute(0, 2, 3, 1)
    int8.cache_write(store, held, (x,), slots)
    assert_slots(store, held, {(0, int(s)): f32(x[i]) for i, s in enumerate(slots.tolist())})


def test_cache_write_rows_that_cannot_be_held():
    from elips_b200 import int8
    codes, scales = new_cache(1, 4, 2, 2, 40, fill=3)
    x = activations(rng(9), (5, 2, 40), torch.float32)
    x[0, 0, 39], x[1, 1, 0], x[2] = float("nan"), float("inf"), 0
    x[3] = 1e-38
    int8.cache_write(codes, scales, (x,), torch.tensor([6, 0, 3, 1, 2], device="cuda"))
    assert_slots(codes, scales, {(0, s): f32(x[i]) for i, s in enumerate([6, 0, 3, 1, 2])})


def filled(g, parts, pages, page, heads, dim):
    codes, scales = new_cache(parts, pages, page, heads, dim)
    codes.copy_(torch.from_numpy(g.integers(-127, 128, codes.shape).astype(np.int8)))
    scales.copy_(torch.from_numpy(np.exp(g.uniform(-9, 3, scales.shape)).astype(np.float32)))
    return codes, scales


def assert_read(got, codes, scales, table, offsets, total, behind=0.0):
    want = R.read_rows(codes.cpu().numpy(), scales.cpu().numpy(), table, offsets, total, codes.shape[2])
    for p, x in enumerate(got):
        w = torch.from_numpy(want[p])
        end = int(offsets[-1])
        assert torch.equal(x[:end].cpu(), w[:end].to(x.dtype)), p
        assert (x[end:] == behind).all()


@pytest.mark.parametrize("parts,heads,dim", CACHES)
@pytest.mark.parametrize("page", [1, 16, 5])
@pytest.mark.parametrize("dtype", FLOATS)
def test_cache_read_sequences(parts, heads, dim, page, dtype):
    """Sequences of no, one and many rows, pages that end inside a sequence, a page used by two of them, rows behind."""
    from elips_b200 import int8
    g = rng(parts, heads, dim, page)
    lengths = [0, 1, 33, 0, page, page + 1, 70, 0]
    pages = 30
    codes, scales = filled(g, parts, pages, page, heads, dim)
    scales[0, 3] = 0
    scales[0, 4, 0, 0] = float("nan")
    scales[0, 5, 0, 0] = float("nan")
    scales.nan_to_num_(nan=0.25)
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    table = g.integers(0, pages, (len(lengths), 70))
    total = int(offsets[-1]) + 9
    idx = torch.int32 if page != 16 else torch.int64
    td, od = torch.from_numpy(table).cuda().to(idx), torch.from_numpy(offsets).cuda().to(idx)
    got = int8.cache_read(codes, scales, td, od, total, dtype)
    assert len(got) == parts
    assert_read(got, codes, scales, table, offsets, total)
    out = tuple(torch.full((total, heads, dim + 3), 5.0, dtype=dtype, device="cuda")[..., 1:1 + dim] for _ in range(parts))
    res = int8.cache_read(codes, scales, td, od, total, out=out)
    assert res[0] is out[0]
    assert_read(res, codes, scales, table, offsets, total, behind=5.0)


@pytest.mark.parametrize("parts,heads,dim", [(2, 3, 67), (1, 1, 251), (2, 1, 9), (1, 8, 129), (1, 2, 8), (1, 5, 3), (2, 1, 2049)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("total", [1, 7, 8, 9, 500])
def test_cache_read_runs_of_odd_rows(parts, heads, dim, dtype, total):
    """Widths that no store divides, packed: stores that span rows, heads, sequences, bad pages and the rows behind,
    which stay as they are."""
    from elips_b200 import int8
    g = rng(parts, heads, dim, total)
    codes, scales = filled(g, parts, 9, 4, heads, dim)
    kept = total - total // 5
    cut = np.sort(g.integers(0, kept + 1, 5))
    offsets = np.concatenate([[0], cut, [kept]])
    table = g.integers(-1, 10, (6, kept // 4 + 1))
    td, od = torch.from_numpy(table).cuda().int(), torch.from_numpy(offsets).cuda()
    assert_read(int8.cache_read(codes, scales, td, od, total, dtype), codes, scales, table, offsets, total)
    out = tuple(torch.full((total, heads, dim), 5.0, dtype=dtype, device="cuda") for _ in range(parts))
    assert_read(int8.cache_read(codes, scales, td, od, total, out=out), codes, scales, table, offsets, total, behind=5.0)
    # one value off 16 bytes, and codes without padding
    held = codes.contiguous()
    out = tuple(torch.full((total * heads * dim + 1,), 5.0, dtype=dtype, device="cuda")[1:].view(total, heads, dim)
                for _ in range(parts))
    assert_read(int8.cache_read(held, scales, td, od, total, out=out), held, scales, table, offsets, total, behind=5.0)
    assert_read(int8.cache_read(held, scales, td, od, total, dtype), held, scales, table, offsets, total)


@pytest.mark.parametrize("heads,dim", [(1, 96), (3, 20)])
def test_cache_read_bad_pages_are_zeros(heads, dim):
    """Table entries that are no page, sequences longer than the table is wide."""
    from elips_b200 import int8
    g = rng(heads)
    codes, scales = filled(g, 2, 6, 4, heads, dim)
    table = np.array([[0, -1, 6, 5], [2, 1 << 30, -(1 << 31), 3], [4, 4, 4, 4]])
    offsets = np.array([0, 16, 30, 50])
    got = int8.cache_read(codes, scales, torch.from_numpy(table).cuda().int(), torch.from_numpy(offsets).cuda(), 50)
    assert_read(got, codes, scales, table, offsets, 50)
    got = int8.cache_read(codes, scales, torch.from_numpy(table).cuda() << 20, torch.from_numpy(offsets).cuda().int(), 50)
    assert_read(got, codes, scales, table << 20, offsets, 50)


@pytest.mark.parametrize("sequences", [255, 256, 257, 3000, 70000])
def test_cache_read_many_sequences(sequences):
    """More sequences than one step of the search looks at, many of them empty, the first not at row 0."""
    from elips_b200 import int8
    g = rng(sequences)
    codes, scales = filled(g, 1, 40, 2, 1, 24)
    offsets = 3 + np.concatenate([[0], np.cumsum(g.integers(0, 3, sequences))])
    table = g.integers(0, 40, (sequences, 1))
    total = int(offsets[-1]) + 5
    got = int8.cache_read(codes, scales, torch.from_numpy(table).cuda().int(), torch.from_numpy(offsets).cuda(), total,
                          torch.float32)[0].cpu()
    seq = np.repeat(np.arange(sequences), np.diff(offsets))
    pos = np.arange(3, offsets[-1]) - offsets[seq]
    pg = torch.from_numpy(table[seq, 0])
    want = codes[0].cpu()[pg, pos].float() * scales[0].cpu()[pg, pos][..., None]
    assert torch.equal(got[3:-5], want) and (got[:3] == 0).all() and (got[-5:] == 0).all()


@pytest.mark.parametrize("offsets", [[0, -5, 9], [7, 3, 1], [0, 1 << 40, 4], [-(1 << 40), 5, 9], [-(1 << 31) - 3, -7, 9]])
def test_cache_read_offsets_that_do_not_ascend(offsets):
    """Whatever they hold, every row read is a row of the cache or zeros."""
    from elips_b200 import int8
    codes, scales = new_cache(1, 3, 4, 1, 16, fill=1)
    table = torch.tensor([[0, 1, 2], [2, 1, 0]], device="cuda")
    got = int8.cache_read(codes, scales, table, torch.tensor(offsets, device="cuda"), 9, torch.float32)[0]
    assert ((got == 1) | (got == 0)).all()


def test_cache_read_nothing():
    from elips_b200 import int8
    codes, scales = filled(rng(1), 1, 2, 4, 1, 16)
    none = torch.empty((0, 0), dtype=torch.int32, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert int8.cache_read(codes, scales, none, zero, 0)[0].shape == (0, 1, 16)
    assert (int8.cache_read(codes, scales, none, zero, 5)[0] == 0).all()
    assert int8.cache_write(codes, scales, (torch.empty((0, 1, 16), device="cuda"),), zero[:0]) is None
    empty = torch.empty((1, 0, 4, 1, 16), dtype=torch.int8, device="cuda"), torch.empty((1, 0, 4, 1), device="cuda")
    int8.cache_write(*empty, (torch.ones((3, 1, 16), device="cuda"),), torch.zeros(3, dtype=torch.int64, device="cuda"))
    got = int8.cache_read(*empty, torch.zeros((1, 4), dtype=torch.int32, device="cuda"),
                          torch.tensor([0, 3], device="cuda"), 3)
    assert (got[0] == 0).all()


def test_cache_offsets_past_32_bits():
    """Slots past 2^31 and 2^32 bytes of codes."""
    from elips_b200 import int8
    pages, page, heads, dim = 8400, 64, 8, 1024     # 4.4 GB of codes
    codes = torch.zeros((1, pages, page, heads, dim), dtype=torch.int8, device="cuda")
    scales = torch.zeros((1, pages, page, heads), device="cuda")
    last = pages * page - 1
    slots = torch.tensor([0, 262143, 262144, 524287, 524288, last], device="cuda")
    x = activations(rng(3), (6, heads, dim), torch.bfloat16)
    int8.cache_write(codes, scales, (x,), slots)
    q, s = R.quantize(f32(x))
    flat, held = codes.view(-1, heads, dim), scales.view(-1, heads)
    assert np.array_equal(flat[slots].cpu().numpy(), q) and np.array_equal(held[slots].cpu().numpy(), s)
    table = (slots // page)[:, None].int()
    offsets = torch.arange(7, device="cuda") * page
    got = int8.cache_read(codes, scales, table, offsets, 6 * page, torch.float32)[0]
    at = torch.arange(6, device="cuda") * page + slots % page
    assert torch.equal(got[at].cpu(), torch.from_numpy(q.astype(np.float32) * s[..., None]))


# --------------------------------------------------------- streams, graphs, together

def pass_of_all(st):
    """One step of a program that uses them together: tokens through a layer into the cache, the cache read back, and
    the tokens scored against the rows it gave."""
    from elips_b200 import int8
    kv = int8.linear_int8(st["x"], st["w"], st["sw"])
    t = kv.shape[0]
    k, v = kv[:, :128].view(t, 2, 64), kv[:, 128:].view(t, 2, 64)
    int8.cache_write(st["codes"], st["scales"], (k, v), st["slots"])
    keys, values = int8.cache_read(st["codes"], st["scales"], st["table"], st["offsets"], t, torch.bfloat16)
    rows, held = int8.quantize_rows(keys.view(t, 128))
    return keys, values, int8.gemm_int8(rows, rows, held, held, out_dtype=torch.float32)


def state(t, seed, k=96):
    g = rng(t, seed)
    codes, scales = new_cache(2, -(-t // 16) + 2, 16, 2, 64)
    order = g.permutation(codes.shape[1])[:-(-t // 16)]
    pos = np.arange(t)
    return {"x": activations(g, (t, k), torch.bfloat16), "w": operand(g, 256, k, 16), "sw": torch.from_numpy(g.random(256).astype(np.float32) + np.float32(0.1)).cuda(),
            "codes": codes, "scales": scales, "slots": torch.from_numpy(order[pos // 16] * 16 + pos % 16).cuda(),
            "table": torch.from_numpy(order[None].astype(np.int32)).cuda(),
            "offsets": torch.tensor([0, t], dtype=torch.int32, device="cuda")}


@pytest.mark.parametrize("t", [1, 6, 50, 300])
def test_together(t):
    """The whole pass equals the definitions, each step on what the one before gave."""
    from elips_b200 import ExactIndex, int8
    st = state(t, 1)
    keys, values, scores = pass_of_all(st)
    kv = int8.linear_int8(st["x"], st["w"], st["sw"])
    q, s = R.quantize(f32(kv).reshape(t, 2, 2, 64))
    back = torch.from_numpy(q.astype(np.float32) * s[..., None]).to(torch.bfloat16)
    assert torch.equal(keys.cpu(), back[:, 0]) and torch.equal(values.cpu(), back[:, 1])
    rows, held = int8.quantize_rows(keys.view(t, 128))
    assert_product(scores, rows, rows, held, held, None, torch.float32)
    # the codes are rows of the int8 index, whose distance is minus the integer product
    ix = ExactIndex("dot_product", 128, precision="int8")
    ix.add_device(rows)
    d, r = ix.search_batch(rows.cpu().numpy(), 1)
    ones = torch.ones(t, device="cuda")
    plain = int8.gemm_int8(rows, rows, ones, ones, out_dtype=torch.float32).cpu().numpy()
    assert np.array_equal(-d[:, 0], plain.max(1))


@pytest.mark.parametrize("t", [1, 6, 300])
def test_captured_and_replayed(t):
    """Two graphs of the same calls, replayed in turn and on different streams over new inputs."""
    a, b = state(t, 1), state(t, 2)
    fresh = [[y.clone() for y in pass_of_all(state(t, s))] for s in (1, 2, 3, 4)]
    graphs = []
    for st in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = pass_of_all(st)
        graphs.append((g, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for s, (g, _) in zip(streams, graphs):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for (g, out), want in zip(graphs, fresh[:2]):
        assert all(torch.equal(x, y) for x, y in zip(out, want))
    for st, seed in ((a, 3), (b, 4)):
        for key, v in state(t, seed).items():
            if key not in ("codes", "scales"):
                st[key].copy_(v)
    for _ in range(2):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for (g, out), want in zip(graphs, fresh[2:]):
        assert all(torch.equal(x, y) for x, y in zip(out, want))


@pytest.mark.parametrize("t", [3, 300])
def test_captured_over_two_streams(t):
    """A graph whose calls fork to a second stream and meet again, with copies and fills between them."""
    from elips_b200 import int8
    st = state(t, 5)
    w2 = operand(rng(t, 6), 200, 96, 16)
    sw2 = torch.rand(200, device="cuda")

    def step():
        main, side = torch.cuda.current_stream(), torch.cuda.Stream()
        x = st["x"].clone()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            right = int8.linear_int8(x, w2, sw2)
            int8.cache_write(st["codes"], st["scales"], (right[:, :128].view(t, 2, 64), right[:, 64:192].view(t, 2, 64)),
                             st["slots"])
        codes, scales = int8.quantize_rows(x)
        left = int8.gemm_int8(codes, w2, scales, sw2)
        main.wait_stream(side)
        keys, _ = int8.cache_read(st["codes"], st["scales"], st["table"], st["offsets"], t)
        again, held = int8.quantize_rows(keys.view(t, 128))
        out = torch.zeros((t, t), device="cuda")
        return left, right, keys, int8.gemm_int8(again, again, held, held, out=out)

    want = [y.clone() for y in step()]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(3):
        for y in got:
            y.fill_(1)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("as_handle", [False, True])
def test_on_another_stream(as_handle):
    """stream=: work is ordered on that stream, outputs belong to it, inputs may be dropped at once."""
    from elips_b200 import int8
    g = rng(4)
    s = torch.cuda.Stream()
    handle = s.cuda_stream if as_handle else s
    x = activations(g, (600, 512), torch.bfloat16)
    w, sw = operand(g, 400, 512, 16), torch.rand(400, device="cuda")
    want = int8.linear_int8(x, w, sw)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        y = x.clone()
    got = int8.linear_int8(y, w, sw, stream=handle)
    codes, held = int8.quantize_rows(y, stream=handle)
    scored = int8.gemm_int8(codes, w, held, sw, stream=handle)
    cache, scales = new_cache(1, 600, 1, 1, 512)
    slots = torch.arange(600, device="cuda")
    table, offsets = torch.arange(600, device="cuda")[None], torch.tensor([0, 600], device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    int8.cache_write(cache, scales, (y[:, None],), slots, stream=handle)
    back, = int8.cache_read(cache, scales, table, offsets, 600, torch.float32, stream=handle)
    del y, slots, table, offsets
    noise = [torch.randn((600, 512), device="cuda").bfloat16() for _ in range(4)]
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(scored, want) and len(noise) == 4
    assert torch.equal(back[:, 0], codes.float() * held[:, None])


def test_two_calls_at_once():
    """Writes of disjoint slots and products on two streams at the same time."""
    from elips_b200 import int8
    g = rng(7)
    codes, scales = new_cache(1, 2000, 1, 2, 64)
    x = activations(g, (2000, 2, 64), torch.bfloat16)
    order = torch.from_numpy(g.permutation(2000)).cuda()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for half, s in enumerate(streams):
        part = slice(half * 1000, (half + 1) * 1000)
        int8.cache_write(codes, scales, (x[part],), order[part], stream=s)
    torch.cuda.synchronize()
    q, held = R.quantize(f32(x))
    assert np.array_equal(codes[0, :, 0][order].cpu().numpy(), q)
    assert np.array_equal(scales[0, :, 0][order].cpu().numpy(), held)


def test_products_at_once():
    """Products of every form on two streams at the same time, over and over: the same bits as alone."""
    from elips_b200 import int8
    sizes = [(1500, 2050, 1500), (40, 4096, 4096), (1, 4096, 4096), (64, 20000, 200), (16, 1024, 2048), (512, 4096, 300)]
    calls = []
    for m, n, k in sizes:
        a, b, sa, sb, _ = gemm_case(m, n, k, torch.float32)
        x = activations(rng(m), (m, k), torch.bfloat16)
        calls.append((a, b, sa, sb, x))
    want = [(int8.gemm_int8(a, b, sa, sb), int8.linear_int8(x, b, sb)) for a, b, sa, sb, x in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(6):
        for half, s in enumerate(streams):
            with torch.cuda.stream(s):
                for a, b, sa, sb, x in (calls if half else calls[::-1]):
                    got.append((int8.gemm_int8(a, b, sa, sb), int8.linear_int8(x, b, sb), b))
    torch.cuda.synchronize()
    of = {b.data_ptr(): w for (_, b, _, _, _), w in zip(calls, want)}
    for c, d, b in got:
        assert torch.equal(c, of[b.data_ptr()][0]) and torch.equal(d, of[b.data_ptr()][1])


def test_inputs_that_require_gradients():
    from elips_b200 import int8
    x = torch.randn((3, 64), device="cuda", requires_grad=True)
    with pytest.raises(ValueError):
        int8.quantize_rows(x)
    with torch.no_grad():
        codes, _ = int8.quantize_rows(x)
    assert not codes.is_floating_point()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_a_device_that_is_not_current():
    from elips_b200 import int8
    x = torch.randn((30, 256), device="cuda:1")
    codes, scales = int8.quantize_rows(x)
    c = int8.gemm_int8(codes, codes, scales, scales, out_dtype=torch.float32)
    assert c.device.index == 1 and torch.cuda.current_device() == 0
    assert_product(c, codes, codes, scales, scales, None, torch.float32)


def test_errors_leave_no_device_error():
    from elips_b200 import _capi, int8
    a = torch.zeros((2, 1 << 17), dtype=torch.int8, device="cuda")
    one = torch.ones(2, device="cuda")
    with pytest.raises(_capi.ElipsB200Error) as e:
        int8.gemm_int8(a, a, one, one)
    assert e.value.status == _capi.INVALID_ARGUMENT
    assert _capi.device_error(0) == 0


@pytest.mark.parametrize("m", [1, 5, 40, 600])
def test_outputs_beside_and_on_their_inputs(m):
    """One buffer holds the rows and, in the columns next to them, the output; on the rows themselves it is refused
    (few rows are quantised by every block of the product, which would find some of them overwritten)."""
    from elips_b200 import ElipsB200Error, int8 as ops
    torch.manual_seed(m)
    n, k = 64, 96
    buffer = torch.randn((m, k + n), device="cuda", dtype=torch.bfloat16)
    weight, scales = ops.quantize_rows(torch.randn((n, k), device="cuda"))
    x = buffer[:, :k]
    want = ops.linear_int8(x.clone(), weight, scales)
    before = x.clone()
    assert torch.equal(ops.linear_int8(x, weight, scales, out=buffer[:, k:]), want)
    assert torch.equal(x, before)
    with pytest.raises(ElipsB200Error):
        ops.linear_int8(x, weight, scales, out=buffer[:, k - 1:-1])
    with pytest.raises(ElipsB200Error):
        ops.linear_int8(x, weight, scales, out=x[:, :n])
    assert torch.equal(x, before)
