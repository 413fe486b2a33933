"""The 8-bit row operators in numpy, from their definitions in 64 bits."""
import numpy as np

TINY = np.float32(2.0 ** -126)
LARGEST = np.float32(2.6793883890187504e+36)                   # the largest scale whose 127-fold is a finite fp32 number


def quantize(x):
    """(codes int8, scales float32) of rows x [..., d] given as float32. The quotient of two 24-bit numbers that is no
    tie is further from one than a 64-bit division rounds, so rint of it is the nearest integer, ties to even."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        top = np.abs(x).max(-1)                                # NaN where the row has one
        s = (top / np.float32(127)).astype(np.float32)         # numpy divides fp32 by fp32 correctly rounded
        s = np.where(np.isfinite(top) & (s > LARGEST), LARGEST, s)
        s = np.where(s < TINY, np.float32(0), s)
        held = np.isfinite(s) & (s > 0)
        div = np.where(held, s, 1).astype(np.float64)[..., None]
        q = np.rint(np.where(held[..., None], x, 0).astype(np.float64) / div)
    assert np.abs(q).max(initial=0) <= 127
    return q.astype(np.int8), s


def gemm(a, b, sa, sb, bias=None):
    """float64 products: the sums are whole numbers below 2^31, exact in 64 bits."""
    acc = a.astype(np.float64) @ b.astype(np.float64).T
    v = acc * sa.astype(np.float64)[:, None] * sb.astype(np.float64)
    return v if bias is None else v + bias.astype(np.float64)


def gemm_bound(v, bias, out_eps):
    """How far a result may be off v: the sum's conversion to fp32, the two scales and the bias each round by at most
    2^-24 of what they give (the bias may make that smaller than the products: their size is at most |v| + |bias|),
    then one rounding to the output's type."""
    big = np.abs(v) + (0 if bias is None else np.abs(bias.astype(np.float64)))
    fp32 = 4 * 2.0 ** -24 * (1 + 2.0 ** -20) * big
    return fp32 + out_eps / 2 * (np.abs(v) + fp32) + 2.0 ** -149


def read_rows(codes, scales, table, offsets, total, page):
    """[parts, total, heads, dim] float32 products code * scale (one fp32 rounding), NaN rows where nothing is read."""
    parts, pages, _, heads, dim = codes.shape
    out = np.full((parts, total, heads, dim), np.nan, np.float32)
    for b in range(len(offsets) - 1):
        for r in range(int(offsets[b]), min(int(offsets[b + 1]), total)):
            i = r - int(offsets[b])
            pg = int(table[b, i // page]) if i // page < table.shape[1] else -1
            if not 0 <= pg < pages:
                out[:, r] = 0
            else:
                out[:, r] = codes[:, pg, i % page].astype(np.float32) * scales[:, pg, i % page][..., None]
    return out
