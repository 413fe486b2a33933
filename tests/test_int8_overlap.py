"""Which calls of the 8-bit operators are refused because an output shares memory with an input or another output. The
addresses are made up and the device is one that no machine has: a call that passes the checks ends there."""
import ctypes
import itertools
import random

import pytest

from elips_b200 import _capi

LIB, BAD, NO_DEVICE = _capi.LIB, _capi.INVALID_ARGUMENT, 1 << 20
BF16, F32 = _capi.PRECISION_BF16, _capi.PRECISION_FP32


def verdict(status):
    """True where the call was refused for its arguments, False where it went on to the device."""
    assert status != _capi.OK
    return status == BAD


def nbytes(base, width, axes):
    """Every byte of runs of `width` bytes at each combination of the axes' (count, step)."""
    starts = [base + sum(i * s for i, (_, s) in zip(at, axes))
              for at in itertools.product(*(range(n) for n, _ in axes))]
    return {s + j for s in starts for j in range(width)}


class Call:
    """A cache of 3 pages of 4 slots with 2 heads of 8 codes, 5 rows written or read, everything far apart."""

    def __init__(self, **kw):
        self.parts, self.pages, self.page, self.heads, self.dim, self.t = 2, 3, 4, 2, 8, 5
        self.codes, self.scales, self.slots, self.table, self.offsets = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20
        self.rows = [6 << 20, 7 << 20]
        self.code_strides, self.scale_strides = [192, 64, 16, 8], [24, 8, 2, 1]
        self.row_strides = [[16, 8], [16, 8]]              # elements
        self.sequences, self.width, self.table_stride = 2, 3, 3
        self.__dict__.update(kw)

    def described(self):
        return _capi.Cache(self.codes, self.scales, self.parts, self.pages, self.page, self.heads, self.dim,
                           tuple(self.code_strides), tuple(self.scale_strides))

    def given(self):
        return (_capi.Rows * 2)(*[_capi.Rows(a, *s) for a, s in zip(self.rows, self.row_strides)])

    def write(self):
        c = self.described()
        return verdict(LIB.elips_b200_cache_write(NO_DEVICE, ctypes.byref(c), self.given(), BF16, self.t, self.slots, 1, None))

    def read(self):
        c = self.described()
        q = _capi.Sequences(self.table, self.offsets, self.table_stride, self.sequences, self.width, self.t, 0, 1)
        return verdict(LIB.elips_b200_cache_read(NO_DEVICE, ctypes.byref(c), ctypes.byref(q), self.given(), BF16, 1, None))

    def sets(self):
        axes = list(zip([self.parts, self.pages, self.page, self.heads], self.code_strides))
        scale_axes = list(zip([self.parts, self.pages, self.page, self.heads], [4 * s for s in self.scale_strides]))
        rows = [nbytes(a, 2 * self.dim, [(self.t, 2 * s[0]), (self.heads, 2 * s[1])])
                for a, s in zip(self.rows, self.row_strides)][:self.parts]
        return nbytes(self.codes, self.dim, axes), nbytes(self.scales, 4, scale_axes), rows


def test_far_apart_goes_on():
    assert not Call().write() and not Call().read()


@pytest.mark.parametrize("part", [0, 1])
@pytest.mark.parametrize("target", ["codes", "scales", "table", "offsets", "slots"])
@pytest.mark.parametrize("side", ["on", "end", "start"])
def test_rows_and_outputs_on_everything_else(target, part, side):
    size = {"codes": 384, "scales": 192, "table": 24, "offsets": 24, "slots": 40}[target]
    mine = 160                                             # bytes of 5 x 2 x 8 bf16 rows
    call = Call()
    at = getattr(call, target)
    call.rows[part] = {"on": at, "end": at + size - 2, "start": at - mine + 2}[side]
    beside = Call()
    beside.rows[part] = {"on": at + size, "end": at + size, "start": at - mine}[side]
    if target in ("codes", "scales"):
        assert call.write() and call.read()
    elif target == "slots":
        assert not call.write()                            # both are read
    else:
        assert call.read()
    assert not beside.write() and not beside.read()


def test_slots_and_the_cache():
    for at in (1 << 20, (1 << 20) + 376, 2 << 20, (2 << 20) + 184, (2 << 20) - 32):
        assert Call(slots=at).write()
    assert not Call(slots=(1 << 20) + 384).write()
    assert Call(scales=(1 << 20) + 380).write()            # codes that end in the first scale
    assert not Call(scales=(1 << 20) + 384).write()


def test_outputs_on_one_another():
    at = 6 << 20
    assert Call(rows=[at, at]).read()
    assert Call(rows=[at, at + 2]).read()
    assert Call(rows=[at, at + 158]).read()
    assert not Call(rows=[at, at + 160]).read()
    assert not Call(rows=[at, at]).write()                 # inputs may be one


def test_layouts_that_take_turns():
    at = 6 << 20
    # keys and values of a row side by side, of a head side by side, and one output's heads before its rows
    assert not Call(rows=[at, at + 32], row_strides=[[32, 8], [32, 8]]).read()
    assert not Call(rows=[at, at + 16], row_strides=[[32, 16], [32, 16]]).read()
    assert not Call(rows=[at, at + 80], row_strides=[[8, 80], [8, 80]]).read()
    assert Call(rows=[at, at + 14], row_strides=[[32, 16], [32, 16]]).read()
    # each page's codes, then its scales: 96 bytes a page, 288 a part
    packed = dict(codes=1 << 20, scales=(1 << 20) + 64, code_strides=[288, 96, 16, 8], scale_strides=[72, 24, 2, 1])
    assert not Call(**packed).write() and not Call(**packed).read()
    assert Call(**packed | {"scales": (1 << 20) + 60}).write()
    # pages outside parts
    packed = dict(codes=1 << 20, scales=(1 << 20) + 64, code_strides=[96, 192, 16, 8], scale_strides=[24, 48, 2, 1])
    assert not Call(**packed).write()
    # each row's codes, then its scale
    packed = dict(codes=1 << 20, scales=(1 << 20) + 8, code_strides=[288, 96, 24, 12], scale_strides=[72, 24, 6, 3])
    assert not Call(**packed).write()


def test_nothing_shared_is_ever_missed():
    """Random layouts in one small buffer: every call whose byte sets meet is refused."""
    g = random.Random(1)
    refused = went_on = 0
    for _ in range(3000):
        t, heads = g.randint(1, 4), g.randint(1, 3)
        call = Call(parts=g.randint(1, 2), pages=g.randint(1, 3), page=g.randint(1, 3), heads=heads, t=t,
                    codes=4096 + g.randint(0, 400), scales=4096 + 4 * g.randint(0, 100),
                    rows=[4096 + 2 * g.randint(0, 200), 4096 + 2 * g.randint(0, 200)],
                    code_strides=[g.choice([8, 16, 24, 48, 96, 192]) for _ in range(4)],
                    scale_strides=[g.choice([1, 2, 6, 12, 24]) for _ in range(4)],
                    row_strides=[[g.choice([8, 16, 24, 48]), g.choice([8, 16, 24])] for _ in range(2)])
        codes, scales, rows = call.sets()
        ins = codes & scales or any(r & codes or r & scales for r in rows)
        outs = any(r & codes or r & scales for r in rows) or (len(rows) == 2 and rows[0] & rows[1])
        for shared, said in ((ins, call.write()), (outs, call.read())):
            assert said or not shared
            refused += said
            went_on += not said
    assert refused > 300 and went_on > 300


def test_products_beside_their_inputs_at_other_pitches():
    """Rows of one pitch and outputs of twice that pitch in one buffer, their columns apart."""
    def status(**kw):
        d = dict(a=1 << 20, a_scales=2 << 20, b=3 << 20, b_scales=4 << 20, bias=None, out=(1 << 20) + 64, m=4, n=8, k=16,
                 a_stride=128, b_stride=16, out_stride=64, a_type=_capi.PRECISION_INT8, bias_type=0, out_type=F32,
                 reserved=0) | kw
        return verdict(LIB.elips_b200_gemm_int8(NO_DEVICE, ctypes.byref(_capi.Gemm(*d.values())), None))
    assert not status()
    assert status(out=(1 << 20) + 12)
    assert status(out=(1 << 20) + 128 - 28)
