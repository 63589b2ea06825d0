"""Microscaled 4-bit matrices: quantisation to the bit, values read back, and products against 64 bits on the host."""
import ctypes as C

import numpy as np
import pytest

import glm53h
from glm53h import DevBuf, check
from op_lib import BF16, F16, F32, HALF, TINY, Buf, Plan, close, dec, enc, routing, sorted_plan, swiglu
from test_gpu_parity import say

pytestmark = pytest.mark.gpu
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
LIMIT = 5.0


@pytest.fixture(scope="module")
def L():
    return glm53h.init(0)


def pack(lv):
    return (lv[..., 0::2] | (lv[..., 1::2] << 4)).astype(np.uint8)


def quant(x):
    """Levels [rows][cols] and scales [rows][cols / 32] of 64-bit values, from the definition."""
    v = x.reshape(x.shape[0], -1, 32)
    top = np.abs(v).max(2, keepdims=True)
    bad = ~np.isfinite(v).all(2, keepdims=True)
    with np.errstate(all="ignore"):
        e = np.where((top > 0) & ~bad, np.floor(np.log2(np.where(bad, 1, top))), -1000)
        # log2 near a power of two: the exact one by comparison
        e = np.where(np.ldexp(1.0, (e + 1).astype(int)) <= top, e + 1, e)
        e = np.where((np.ldexp(1.0, np.maximum(e, -1070).astype(int)) > top) & (top > 0), e - 1, e)
    b = np.maximum(e - 2, -127).astype(int)
    a = np.ldexp(np.where(bad, 0, np.abs(v)), -b)
    d = np.abs(a[..., None] - LEVELS)                        # the nearest level, ties to the even one
    lv = d.argmin(-1)
    tie = (lv < 7) & (np.take_along_axis(d, np.minimum(lv + 1, 7)[..., None], -1)[..., 0] == d.min(-1))
    lv = np.where(tie & (lv % 2 == 1), lv + 1, lv)
    lv = np.where(bad, 0, lv | (np.signbit(v) << 3))
    return lv.reshape(x.shape).astype(np.uint8), np.where(bad, 255, b + 127)[..., 0].astype(np.uint8)


def wide(lv, s):
    v = np.where(lv & 8, -1.0, 1.0) * LEVELS[lv & 7]
    return (np.ldexp(v.reshape(*s.shape, 32), s.astype(int)[..., None] - 127)).reshape(lv.shape)


class Mx4:
    """n stacked matrices of given levels and scales, on the host (wide) and on the device."""

    def __init__(self, lv, s, rows):
        self.w_d, self.s_d = Buf(pack(lv)), Buf(s)
        self.wide = wide(lv, s) if (s < 255).all() else None
        self.c = glm53h.G53hMx4(self.w_d.ptr, self.s_d.ptr, rows, lv.shape[1])

    @classmethod
    def random(cls, rng, rows, cols, n=1, low=124, high=130):
        return cls(rng.integers(0, 16, (n * rows, cols)).astype(np.uint8),
                   rng.integers(low, high + 1, (n * rows, cols // 32)).astype(np.uint8), rows)


def hard(rng, rows, cols, dt):
    """Values whose blocks hold ties between levels, powers of two and their neighbours, zeros, the smallest and the largest."""
    x = dec(enc(rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 12, (rows, 1))), dt), dt)
    v = x.reshape(rows, -1, 32)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, -0.25, -0.75, -1.25, -2.5, -3.5, -5, 4])
    pick = rng.integers(0, 6, v.shape[:2])
    v[..., :16][pick == 1] = ties * 0.125
    v[..., 16:][pick == 1] = 0.0
    v[pick == 2] = 0.0
    v[..., 0][pick == 2] = -0.0
    v[..., 5][pick == 3] = np.exp2(rng.integers(0, 9, (pick == 3).sum())) * 2
    big = {F32: 3.4e38, BF16: 3.38e38, F16: 65504.0}[dt]
    small = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}[dt]
    v[..., 3][pick == 4] = big
    v[pick == 5] = small * rng.integers(-40, 40, ((pick == 5).sum(), 32))
    return dec(enc(x, dt), dt)


@pytest.mark.parametrize("rows,cols,dt", [(1, 32, F32), (1, 4096, BF16), (3, 96, F16), (7, 2080, F32), (130, 160, BF16), (64, 1024, F16),
                                          (257, 32, F32)])
def test_quant(L, rows, cols, dt):
    say("quant", rows, cols, dt)
    rng = np.random.default_rng(rows + cols)
    x = hard(rng, rows, cols, dt)
    lv, s = quant(x)
    w_d, s_d = Buf.out((rows, cols // 2), np.uint8), Buf.out((rows, cols // 32), np.uint8)
    m = glm53h.G53hMx4(w_d.ptr, s_d.ptr, rows, cols)
    src = Buf(x, dt, shift=2 if dt != F32 else 4)
    check(L.g53h_mx4_quant(m, src.ptr, dt))
    assert np.array_equal(s_d.get(), s)
    got = w_d.get()
    assert np.array_equal(got, pack(lv)), np.argwhere(got != pack(lv))[:5]
    for out in (F32, BF16, F16):
        back = Buf.out((rows, cols), out, shift=2 if out != F32 else 4)
        check(L.g53h_mx4_dequant(back.ptr, out, m))
        with np.errstate(over="ignore"):
            want = dec(enc(wide(lv, s), out), out)           # below fp32's steps (2^-128) too: to nearest
        assert np.array_equal(back.val(), want)


def test_values_that_are_not_finite(L):
    say("quant, not finite")
    for dt in (F32, BF16, F16):
        x = np.ones((3, 96))
        x[0, 5], x[1, 40], x[2, 95] = np.inf, -np.inf, np.nan
        lv, s = quant(x)
        assert (s == 255).sum() == 3
        w_d, s_d, src = Buf.out((3, 48), np.uint8), Buf.out((3, 3), np.uint8), Buf(x, dt)
        m = glm53h.G53hMx4(w_d.ptr, s_d.ptr, 3, 96)
        check(L.g53h_mx4_quant(m, src.ptr, dt))
        assert np.array_equal(s_d.get(), s) and np.array_equal(w_d.get(), pack(lv))
        back = Buf.out((3, 96), dt)
        check(L.g53h_mx4_dequant(back.ptr, dt, m))
        assert np.array_equal(np.isnan(back.val()), np.repeat(s == 255, 32, 1))
        # a product: NaN where a block of 255 enters, the others as they are
        ones = Mx4(np.full((70, 96), 2, np.uint8), np.full((70, 3), 127, np.uint8), 70)
        y = Buf.out((3, 70), F32)
        check(L.g53h_mm_mx4(y.ptr, F32, m, ones.c, 0.0))
        assert np.isnan(y.val()).all()
        y = Buf.out((70, 3), F32)
        check(L.g53h_mm_mx4(y.ptr, F32, ones.c, m, 0.0))
        assert np.isnan(y.val()).all()
        s2 = s.copy()
        s2[1] = 127
        part = Mx4(np.full((3, 96), 2, np.uint8), s2, 3)
        y = Buf.out((70, 3), F32)
        check(L.g53h_mm_mx4(y.ptr, F32, ones.c, part.c, 0.0))
        assert np.isnan(y.val()[:, [0, 2]]).all() and (y.val()[:, 1] == 96).all()


def off(cols, size, y, dt, whole):
    """Sums of cols exact products in fp32: every addition off by at most 2^-23 of the sizes' sum, and the rounding."""
    return (0 if whole else (cols + 32) * 2.0 ** -23 * size) + HALF[dt] * np.abs(y) + TINY[dt]


def swiglu_off(gu, sums, dt):
    """Slopes of at most 1.1 and 1 times the other's limit; expf, the division and the products 4 steps; the rounding."""
    half, act = gu.shape[1] // 2, swiglu(gu, LIMIT)
    return (1.1 * LIMIT * (sums[:, :half] + sums[:, half:]) + (4 * 2.0 ** -23 + HALF[dt]) * np.abs(act) + TINY[dt]) * 1.01


@pytest.mark.parametrize("T,rows,cols,dt,sw", [(1, 1, 32, F32, 0), (1, 64, 512, BF16, 1), (2, 130, 96, F16, 0), (5, 300, 4128, F32, 1),
                                               (16, 66, 2048, BF16, 0), (17, 1001, 544, F16, 0), (64, 514, 800, F32, 1), (130, 258, 1056, BF16, 0),
                                               (300, 700, 256, F16, 1), (515, 34, 64, F32, 0)])
def test_dense(L, T, rows, cols, dt, sw):
    say("dense", T, rows, cols, dt, sw)
    rng = np.random.default_rng(rows)
    for whole in (True, False):
        # one scale: sums of multiples of a quarter, exact in fp32
        span = dict(low=127, high=127) if whole else dict(low=118, high=125)
        x, m = Mx4.random(rng, T, cols, **span), Mx4.random(rng, rows, cols, **span)
        ref, size = x.wide @ m.wide.T, np.abs(x.wide) @ np.abs(m.wide).T
        y = Buf.out((T, rows // 2 if sw else rows), dt, shift=2 if dt != F32 else 4)
        check(L.g53h_mm_mx4(y.ptr, dt, x.c, m.c, LIMIT if sw else 0.0))
        if sw:
            close(y.val(), swiglu(ref, LIMIT), swiglu_off(ref, off(cols, size, ref, F32, whole), dt), whole)
        else:
            with np.errstate(over="ignore"):
                close(y.val(), np.where(np.abs(ref) < 65519 if dt == F16 else True, ref, np.copysign(np.inf, ref)), off(cols, size, ref, dt, whole), whole)


@pytest.mark.parametrize("T,K,NE,rows,cols,dt,gather,sw", [
    (1, 1, 1, 2, 32, F32, 1, 0), (1, 4, 16, 128, 512, BF16, 1, 1), (5, 2, 3, 30, 64, F16, 0, 0), (33, 3, 7, 130, 1056, F32, 1, 1),
    (129, 2, 4, 136, 96, BF16, 1, 0), (64, 4, 300, 48, 160, F16, 0, 1), (300, 2, 2, 66, 352, BF16, 0, 0), (700, 1, 1, 300, 512, F16, 1, 0)])
def test_sorted(L, T, K, NE, rows, cols, dt, gather, sw):
    say("sorted", T, K, NE, rows, cols, dt, gather, sw)
    rng = np.random.default_rng(T + rows)
    idx = routing(rng, T, K, NE, 0.2)
    idx[rng.random((T, K)) < 0.1] = NE
    offsets, pair, _ = sorted_plan(idx, NE)
    n, used, plan = T * K, offsets[NE], Plan(idx, NE)
    for whole in (True, False):
        span = dict(low=126, high=126) if whole else dict(low=118, high=125)
        x, m = Mx4.random(rng, T if gather else n, cols, **span), Mx4.random(rng, rows, cols, NE, **span)
        ys = Buf.out((n, rows // 2 if sw else rows), dt)
        check(L.g53h_sorted_mm_mx4(ys.ptr, dt, x.c, gather, plan.c, m.c, LIMIT if sw else 0.0))
        ref, size = np.zeros((n, rows)), np.zeros((n, rows))
        for e in range(NE):
            r, w = slice(offsets[e], offsets[e + 1]), m.wide[e * rows:(e + 1) * rows]
            xe = x.wide[pair[r] // K] if gather else x.wide[r]
            ref[r], size[r] = xe @ w.T, np.abs(xe) @ np.abs(w).T
        sums = off(cols, size, ref, F32 if sw else dt, whole)
        want, tol = (swiglu(ref, LIMIT), swiglu_off(ref, sums, dt)) if sw else (ref, sums)
        want[used:], tol[used:] = 77.0, 0
        close(ys.val(), want, tol, whole)


def test_scales_far_apart(L):
    """Blocks of the smallest and the largest scales in one row, products from below fp32's steps to infinity."""
    say("scales")
    lv = np.full((2, 128), 2, np.uint8)                      # ones
    x = Mx4(lv, np.array([[0, 127, 127, 254], [127, 127, 127, 127]], np.uint8), 2)
    m = Mx4(lv, np.array([[0, 127, 127, 0], [127, 127, 127, 254]], np.uint8), 2)
    y = Buf.out((2, 2), F32)
    check(L.g53h_mm_mx4(y.ptr, F32, x.c, m.c, 0.0))
    got = y.val()
    assert got[0, 0] == 96 and got[0, 1] == np.inf and got[1, 0] == 64 and got[1, 1] == np.inf


def test_nothing_to_do(L):
    say("nothing")
    rng = np.random.default_rng(1)
    m, none = Mx4.random(rng, 8, 64, 4), glm53h.G53hMx4(None, None, 0, 64)
    check(L.g53h_mx4_quant(none, None, BF16))
    check(L.g53h_mx4_dequant(None, BF16, none))
    check(L.g53h_mm_mx4(None, BF16, none, m.c, 0.0))
    check(L.g53h_sorted_mm_mx4(None, BF16, none, 1, Plan(np.zeros((0, 2), np.int32), 4).c, m.c, 0.0))
    x, ys, plan = Mx4.random(rng, 3, 64), Buf.out((6, 8), BF16), Plan(np.full((3, 2), -1, np.int32), 4)
    check(L.g53h_sorted_mm_mx4(ys.ptr, BF16, x.c, 1, plan.c, m.c, 0.0))
    assert (ys.val() == 77).all()


def test_offsets_past_32_bits(L):
    say("large")
    rng = np.random.default_rng(4)
    # x: 3 million rows of 4096: 6.1 GB of levels; the last rows are whole numbers, the others zeros
    T, rows, cols, last = 3000000, 40, 4096, 20
    lv = rng.integers(0, 16, (last, cols)).astype(np.uint8)
    w, s = DevBuf(T * cols // 2), DevBuf(T * cols // 32)
    check(L.g53h_memset(w.ptr, 0, w.nbytes))
    check(L.g53h_memset(s.ptr, 127, s.nbytes))
    bits = pack(lv)
    check(L.g53h_h2d(w.ptr + (T - last) * cols // 2, bits.ctypes.data, bits.nbytes))
    m, x = Mx4.random(rng, rows, cols, low=127, high=127), glm53h.G53hMx4(w.ptr, s.ptr, T, cols)
    y = DevBuf(4 * T * rows)
    check(L.g53h_mm_mx4(y.ptr, F32, x, m.c, 0.0))
    got = y.download(np.float32, (last + 5) * rows, 4 * (T - last - 5) * rows).reshape(last + 5, rows)
    want = wide(lv, np.full((last, cols // 32), 127, np.uint8)) @ m.wide.T
    assert not got[:5].any() and np.array_equal(got[5:], want)
    # and quantised again from what it stands for, in fp32: 12e9 elements do not fit twice, the last 2^20 rows do
    part = 1 << 20
    xs = DevBuf(4 * part * cols)
    tail = glm53h.G53hMx4(w.ptr + (T - part) * cols // 2, s.ptr + (T - part) * cols // 32, part, cols)
    check(L.g53h_mx4_dequant(xs.ptr, F32, tail))
    w2, s2 = DevBuf(part * cols // 2), DevBuf(part * cols // 32)
    check(L.g53h_mx4_quant(glm53h.G53hMx4(w2.ptr, s2.ptr, part, cols), xs.ptr, F32))
    want_lv, want_s = quant(wide(lv, np.full((last, cols // 32), 127, np.uint8)))
    assert np.array_equal(w2.download(np.uint8, last * cols // 2, (part - last) * cols // 2).reshape(last, -1), pack(want_lv))
    assert np.array_equal(s2.download(np.uint8, last * cols // 32, (part - last) * cols // 32).reshape(last, -1), want_s)


# as many tiles as every form of the kernel takes, with ends of each
@pytest.mark.parametrize("T,NE,rows,cols", [(200, 0, 17000, 320), (300, 3, 11000, 96), (70, 0, 34000, 64), (20, 10, 7000, 544), (3, 3, 1000, 1088)])
def test_every_tile(L, T, NE, rows, cols):
    say("tiles", T, NE, rows, cols)
    rng = np.random.default_rng(rows)
    x, m = Mx4.random(rng, T, cols, low=127, high=128), Mx4.random(rng, rows, cols, max(NE, 1), low=125, high=126)
    y, act = Buf.out((T, rows), F32), Buf.out((T, rows // 2), BF16)
    if NE:
        idx = rng.integers(0, NE, (T, 1)).astype(np.int32)
        offsets, pair, _ = sorted_plan(idx, NE)
        plan = Plan(idx, NE)
        check(L.g53h_sorted_mm_mx4(y.ptr, F32, x.c, 1, plan.c, m.c, 0.0))
        check(L.g53h_sorted_mm_mx4(act.ptr, BF16, x.c, 1, plan.c, m.c, LIMIT))
        ref = np.concatenate([x.wide[pair[offsets[e]:offsets[e + 1]]] @ m.wide[e * rows:(e + 1) * rows].T for e in range(NE)])
    else:
        check(L.g53h_mm_mx4(y.ptr, F32, x.c, m.c, 0.0))
        check(L.g53h_mm_mx4(act.ptr, BF16, x.c, m.c, LIMIT))
        ref = x.wide @ m.wide.T
    assert np.array_equal(y.val(), ref)                      # multiples of 1 / 16 below 2^20: exact
    g, u = np.split(ref, 2, 1)
    with np.errstate(over="ignore"):
        want = swiglu(ref, LIMIT)
    # the hardware's exponential and reciprocal 2^-20; the exponential is zero where it lies below 2^-126
    deep = np.where(g < -87, 2.0 ** -126 * np.abs(g * np.clip(u, -LIMIT, LIMIT)), 0)
    close(act.val(), want, (2.0 ** -20 + HALF[BF16]) * np.abs(want) + TINY[BF16] + deep)


@pytest.mark.parametrize("rows,sw,sort", [((1 << 31) - 1, 0, 0), ((1 << 31) - 1, 0, 1), ((1 << 31) - 2, 1, 0)])
def test_as_many_rows_as_an_int_holds(L, rows, sw, sort):
    """Results of a matrix whose last tile ends behind row 2^31 - 1: its first, middle and last ones are right."""
    say("rows", rows, sw, sort)
    rng = np.random.default_rng(rows + sort)
    cols, half, some = 32, rows // 2 if sw else rows, 300
    # zeros but for `some` rows in a few places, of gate and of up with SwiGLU
    places = [0, 1 << 20, half // 2 + 5, half - some]
    w, s = DevBuf(rows * cols // 2), DevBuf(rows)
    check(L.g53h_memset(w.ptr, 0, w.nbytes))
    check(L.g53h_memset(s.ptr, 127, s.nbytes))
    x = Mx4.random(rng, 1, cols, low=127, high=127)
    y = DevBuf(2 * half)
    check(L.g53h_memset(y.ptr, 0x55, y.nbytes))
    want = []
    for at in places:
        y1 = []
        for part in range(2 if sw else 1):
            lv = rng.integers(0, 16, (some, cols)).astype(np.uint8)
            bits = pack(lv)
            check(L.g53h_h2d(w.ptr + (part * half + at) * cols // 2, bits.ctypes.data, bits.nbytes))
            y1.append(x.wide @ wide(lv, np.full((some, 1), 127, np.uint8)).T)
        want.append(np.concatenate(y1, 1))
    m = glm53h.G53hMx4(w.ptr, s.ptr, rows, cols)
    if sort:
        plan = Plan(np.zeros((1, 1), np.int32), 1)
        check(L.g53h_sorted_mm_mx4(y.ptr, F16, x.c, 1, plan.c, m, LIMIT if sw else 0.0))
    else:
        check(L.g53h_mm_mx4(y.ptr, F16, x.c, m, LIMIT if sw else 0.0))
    for at, v in zip(places, want):
        got = dec(y.download(np.float16, some, 2 * at), F16)
        if sw:                                               # sums are exact; see test_every_tile
            act = swiglu(v, LIMIT)[0]
            assert (np.abs(got - act) <= (2.0 ** -20 + HALF[F16]) * np.abs(act) + TINY[F16] + 2.0 ** -100).all(), at
        else:
            assert np.array_equal(got, dec(enc(v[0], F16), F16)), at
    # between them: products with zeros
    for at in (some, half // 3, half - some - 1000):
        assert not dec(y.download(np.float16, 900, 2 * at), F16).any(), at


def tile(cus, n, NE, rows):
    """The tile (rows of x, rows of the matrix) that the library takes for n rows, by its rule."""
    busy = min(NE, n) if NE else 1
    mean = -(-n // busy)
    count = lambda bm, bn: (n // bm + busy if NE else -(-n // bm)) * -(-rows // bn)     # noqa: E731
    if mean >= 32 and count(128, 256) >= 2 * cus:
        return 128, 256
    if mean >= 32 and count(128, 128) >= cus:
        return 128, 128
    return (64, 128) if mean > 1 and count(64, 128) >= 2 * cus else (32, 128)


# rows of x in every expert (one number: a single matrix), columns: one, two and three chunks, with scales to the end of a
# segment and not; the last tile of an expert has up to a quarter, a half and all of its rows
@pytest.mark.parametrize("counts,cols", [((300,), 352), ((140,), 96), ((148, 50, 102), 544), ((128, 0, 190), 512), ((33, 64, 97), 32)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_widest_tiles(L, counts, cols, dt):
    say("widest tiles", counts, cols, dt)
    rng = np.random.default_rng(sum(counts) + cols)
    used, NE, cus = sum(counts), len(counts) if len(counts) > 1 else 0, L.g53h_num_cus()
    n = used + 3 if NE else used                             # three tokens without an expert
    down = n // 128 + NE if NE else -(-n // 128)
    rows = 256 * (-(-2 * cus // down) + 1) - 150             # the last tile across: 106 rows
    assert tile(cus, n, NE, rows) == (128, 256)
    x, m = Mx4.random(rng, n, cols, low=127, high=128), Mx4.random(rng, rows, cols, max(NE, 1), low=125, high=126)
    idx = np.concatenate([np.repeat(np.arange(len(counts)), counts), np.full(n - used, -1)]).astype(np.int32)[:, None]
    rng.shuffle(idx)
    offsets, pair, _ = sorted_plan(idx, len(counts))
    plan = Plan(idx, len(counts))
    for sw in (0, 1):
        y = Buf.out((n, rows // 2 if sw else rows), dt, shift=2 if dt != F32 else 4)
        if NE:
            check(L.g53h_sorted_mm_mx4(y.ptr, dt, x.c, 1, plan.c, m.c, LIMIT if sw else 0.0))
            ref = np.concatenate([x.wide[pair[offsets[e]:offsets[e + 1]]] @ m.wide[e * rows:(e + 1) * rows].T for e in range(NE)])
        else:
            check(L.g53h_mm_mx4(y.ptr, dt, x.c, m.c, LIMIT if sw else 0.0))
            ref = x.wide @ m.wide.T
        got = y.val()
        assert (got[used:] == 77).all()
        if not sw:
            assert np.array_equal(got[:used], dec(enc(ref, dt), dt))       # sums are exact, see test_every_tile
            continue
        g, u = np.split(ref, 2, 1)
        with np.errstate(over="ignore"):
            want = swiglu(ref, LIMIT)
        deep = np.where(g < -87, 2.0 ** -126 * np.abs(g * np.clip(u, -LIMIT, LIMIT)), 0)
        # expf, a division and products: 4 steps; the hardware's exponential and reciprocal 2^-20, and half a step of what
        # the exponential is of, the gate by log2 e
        rel = 4 * 2.0 ** -23 if dt == F32 else 2.0 ** -20 + np.abs(np.minimum(g, 0)) * 2.0 ** -24
        close(got[:used], want, (rel + HALF[dt]) * np.abs(want) + TINY[dt] + deep)
