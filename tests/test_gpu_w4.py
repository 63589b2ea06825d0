"""Products with 4-bit levels and group scales (g53h_mm_w4, g53h_sorted_mm_w4) against 64-bit products
on the host. Tolerances are derived where the product is formed (op_lib.W4.product)."""
import ctypes as C

import numpy as np
import pytest

import glm53h
from glm53h import check
from op_lib import BF16, F16, F32, HALF, TINY, W4, Buf, Plan, close, dec, enc, routing, sorted_plan, swiglu
from test_gpu_parity import say

pytestmark = pytest.mark.gpu
LIMIT = 10.0


@pytest.fixture(scope="module")
def L():
    return glm53h.init(0)


def act_tol(y, tol, limit):
    """What an error of tol in gate and up sums makes of the SwiGLU: |silu'| <= 1.1, |silu(g)| <= |g| + 0.3, the
    clamps shrink distances; silu itself in fp32 is off by at most 8 roundings."""
    g, u = np.split(y, 2, -1)
    tg, tu = np.split(tol, 2, -1)
    gc, uc = np.abs(np.minimum(g, limit)), np.abs(np.clip(u, -limit, limit))
    return 1.1 * tg * (uc + tu) + (gc + 0.3) * tu + 8 * 2.0 ** -24 * (gc + 0.3) * uc


CASES = [  # T, rows, cols, group, s_dt, zeros, swiglu
    (1, 4096, 2048, 64, F32, False, False), (1, 1, 32, 32, F32, True, False), (2, 17, 64, 32, F16, True, False),
    (3, 33, 96, 64, BF16, False, False), (5, 100, 160, 128, F16, True, False), (8, 64, 4096, 4096, F32, False, True),
    (16, 1001, 2080, 32, F16, True, False), (17, 70, 480, 96, BF16, True, True), (24, 130, 1024, 128, F32, False, True),
    (31, 34, 2016, 32, F32, True, True), (33, 48, 288, 160, F32, True, False), (64, 66, 640, 256, BF16, False, True),
    (65, 20, 352, 64, F16, False, False), (130, 258, 224, 128, F32, True, True), (300, 40, 128, 1024, F32, True, False)]


@pytest.mark.parametrize("T,rows,cols,group,s_dt,zeros,sw", CASES)
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_product(L, T, rows, cols, group, s_dt, zeros, sw, dt):
    say("w4", T, rows, cols, group, s_dt, zeros, sw, dt)
    rng = np.random.default_rng(rows + cols + T)
    m = W4(rng, 1, rows, cols, group, s_dt, zeros)
    x, out = Buf(rng.standard_normal((T, cols)), dt), rows // 2 if sw else rows
    y = Buf.out((T, out), dt)
    check(L.g53h_mm_w4(y.ptr, x.ptr, dt, T, C.byref(m.c), LIMIT if sw else 0.0), "w4")
    want, tol = m.product(x.val())
    if sw:
        want, tol = swiglu(want, LIMIT), act_tol(want, tol, LIMIT)
    close(y.val(), want, HALF[dt] * np.abs(want) + TINY[dt] + tol)
    if dt == F32 and cols >= 1024 and not sw:
        # typical sums are far inside the worst case: 2^-16 of a value lost (a plane of x) would show here
        assert np.linalg.norm(y.val() - want) < 2e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("T,rows,cols,group,s_dt,zeros,sw", [c for c in CASES if not c[-1]])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_product_of_whole_numbers_is_exact(L, T, rows, cols, group, s_dt, zeros, sw, dt):
    """Small whole x and power-of-two scales: every partial sum fits 24 bits, so the result is the exact sum,
    rounded once, whatever the order."""
    say("w4, exact", T, rows, cols, group, s_dt, zeros, dt)
    rng = np.random.default_rng(rows + cols + T + 1)
    m = W4(rng, 1, rows, cols, group, s_dt, zeros, exact=True)
    xv = rng.integers(-8, 9, (T, cols)).astype(float)
    x, y = Buf(xv, dt), Buf.out((T, rows), dt)
    check(L.g53h_mm_w4(y.ptr, x.ptr, dt, T, C.byref(m.c), 0.0), "w4")
    with np.errstate(over="ignore"):
        assert np.array_equal(y.get(), enc(xv @ m.wide[0].T, dt))


@pytest.mark.parametrize("T", [1, 3, 12, 40])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (64, True), (96, True), (128, True), (192, False)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_matrices_of_many_rows_are_exact(L, T, group, zeros, dt):
    """A matrix that fills the card, whose waves take two row tiles and, for few tokens, whole lines: 16 copies of 1040
    rows, whole numbers as above."""
    say("w4, many rows", T, group, zeros, dt)
    rng = np.random.default_rng(group + T)
    rows, cols, n = 1040, 4096, 16
    m = W4(rng, 1, rows, cols, group, BF16, zeros, exact=True)
    parts = [glm53h.DevBuf(b.n * n) if b else None for b in (m.w_d, m.s_d, m.z_d)]
    for big, b in zip(parts, (m.w_d, m.s_d, m.z_d)):
        for k in range(n if b else 0):
            check(L.g53h_d2d(big.ptr + k * b.n, b.ptr, b.n), "d2d")
    c = glm53h.G53hW4(parts[0].ptr, parts[1].ptr, parts[2].ptr if zeros else None, rows * n, cols, group, BF16)
    xv = rng.integers(-2, 3, (T, cols)).astype(float)
    x, y = Buf(xv, dt), Buf.out((T, rows * n), dt)
    check(L.g53h_mm_w4(y.ptr, x.ptr, dt, T, C.byref(c), 0.0), "w4")
    with np.errstate(over="ignore"):
        assert np.array_equal(y.get(), np.tile(enc(xv @ m.wide[0].T, dt), (1, n)))


@pytest.mark.parametrize("T,rows,cols,group,zeros", [(2, 50, 2080, 32, True), (16, 34, 2112, 64, True), (5, 66, 2304, 96, False),
                                                     (9, 20, 4096, 192, True), (3, 130, 608, 64, False), (14, 36, 1600, 32, True)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_swiglu_of_few_tokens(L, T, rows, cols, group, zeros, dt):
    say("w4, swiglu", T, rows, cols, group, zeros, dt)
    rng = np.random.default_rng(rows + cols)
    m = W4(rng, 1, rows, cols, group, F16, zeros)
    x, y = Buf(rng.standard_normal((T, cols)), dt), Buf.out((T, rows // 2), dt)
    check(L.g53h_mm_w4(y.ptr, x.ptr, dt, T, C.byref(m.c), LIMIT), "w4")
    sums, tol = m.product(x.val())
    want, tol = swiglu(sums, LIMIT), act_tol(sums, tol, LIMIT)
    close(y.val(), want, HALF[dt] * np.abs(want) + TINY[dt] + tol)


def test_a_matrix_of_the_int4_experts(L):
    """A G53H_MAT_I4 matrix (quantised by the library) as it lies: against the engine's own product with it. Both are
    within the worst case of an fp32 sum of the 64-bit product: 512 products, group sums and their sum, each addition
    off by 2^-24 of at most 62 (levels as they enter) sum |x| s."""
    say("w4, int4 experts' format")
    rng = np.random.default_rng(21)
    rows, cols, T = 256, 512, 3
    codes = rng.integers(0, 256, (rows, cols)).astype(np.uint8)
    codes[(codes & 0x7f) == 0x7f] = 0                            # no NaN
    w, s = Buf(codes), Buf(rng.uniform(0.5, 1.5, (2, 4)), F32)
    q, steps = Buf(np.zeros((rows, cols // 2), np.uint8)), Buf(np.zeros((rows, cols // 64)), F32)
    f8 = glm53h.G53hMat(w.ptr, s.ptr, rows, cols, 128, 128, 4, 0)
    check(L.g53h_i4_from_f8(q.ptr, steps.ptr, C.byref(f8)), "g53h_i4_from_f8")
    i4 = glm53h.G53hMat(q.ptr, steps.ptr, rows, cols, 1, 64, cols // 64, 4)                # G53H_MAT_I4
    x, ya, yb = Buf(rng.standard_normal((T, cols)), F32), Buf.out((T, rows), F32), Buf.out((T, rows), F32)
    check(L.g53h_mm_f8(ya.ptr, x.ptr, T, C.byref(i4)), "g53h_mm_f8")
    check(L.g53h_mm_w4(yb.ptr, x.ptr, F32, T, C.byref(glm53h.G53hW4(q.ptr, steps.ptr, None, rows, cols, 64, F32)), 0.0), "w4")
    size = np.abs(x.val()) @ np.repeat(steps.val(), 64, 1).T
    close(yb.val(), ya.val(), 2 * (2 * 512 + 40) * 2.0 ** -24 * 62 * size)
    assert np.abs(ya.val()).max() > 0


@pytest.mark.parametrize("shift", [2, 4, 6, 14])
def test_rows_off_alignment(L, shift):
    say("w4, x and y off by", shift)
    rng = np.random.default_rng(shift)
    m = W4(rng, 1, 37, 96, 32, F32, True, exact=True)
    xv = rng.integers(-8, 9, (9, 96)).astype(float)
    for dt in (BF16, F32) if shift == 4 else (BF16,):
        x, y = Buf(xv, dt, shift), Buf.out((9, 37), dt, shift)
        check(L.g53h_mm_w4(y.ptr, x.ptr, dt, 9, C.byref(m.c), 0.0), "w4")
        assert np.array_equal(y.get(), enc(xv @ m.wide[0].T, dt))


def test_full_range_of_fp32(L):
    """fp32 activations from 2^-100 to 2^100: each is three planes exactly, so a column alone is off by the
    roundings of its own few sums."""
    say("w4, wide range")
    rng = np.random.default_rng(8)
    m = W4(rng, 1, 40, 64, 32, F32, True)
    xv = np.zeros((64, 64))
    xv[np.arange(64), np.arange(64)] = rng.uniform(1, 2, 64) * 2.0 ** rng.integers(-100, 100, 64)
    x, y = Buf(xv, F32), Buf.out((64, 40), F32)
    check(L.g53h_mm_w4(y.ptr, x.ptr, F32, 64, C.byref(m.c), 0.0), "w4")
    want, _ = m.product(x.val())
    # three planes of (16 + q) x and of x, the surplus, the scale: ten roundings of at most 62 |x| s
    close(y.val(), want, 10 * 2.0 ** -24 * 62 * (np.abs(x.val()) @ m.s[0].T))


def test_smallest_fp16_activations(L):
    """fp16 values below the normal range enter as they are: multiples of 2^-24, with sums that fit 24 bits, exactly."""
    say("w4, fp16 below its normal range")
    rng = np.random.default_rng(13)
    m = W4(rng, 1, 24, 96, 32, F32, True, exact=True)
    for T in (1, 20):
        xv = rng.integers(-8, 9, (T, 96)) * 2.0 ** -24
        x, y = Buf(xv, F16), Buf.out((T, 24), F16)
        assert np.array_equal(x.val(), xv)
        check(L.g53h_mm_w4(y.ptr, x.ptr, F16, T, C.byref(m.c), 0.0), "w4")
        assert np.array_equal(y.get(), enc(xv @ m.wide[0].T, F16))


@pytest.mark.parametrize("T", [1, 5, 6, 33])
def test_fp32_error_stays_that_of_one_sum(L, T):
    """fp32 products of short rows, in two groups of 128: x of size 1, levels even over 0..15, zero point 8. A group's D, the
    sum of (16 + level) x, has an rms of 24 sqrt(128) = 272 and is added up in 4 steps, each off by up to 2^-15 (a sum in
    [256, 512) that is cut, not rounded): 2^-15 / sqrt(3) rms. X, the sum of x, has 11.3 and counts 24 times: 24 x 2^-20 /
    sqrt(3). Together sqrt(4) sqrt(1.76e-5^2 + 1.32e-5^2) = 4.4e-5 of a group whose own rms is sqrt(128) x 4.6 = 52:
    8.5e-7, and the spread of a norm over 512 rows allows two fifths more. The lower planes add 2^-8 of it where their
    products have sums of their own; in one sum with the upper ones they would each be cut at its size: sqrt(3) as much."""
    say("w4, fp32 error", T)
    rng = np.random.default_rng(14 + T)
    m = W4(rng, 1, 512, 256, 128, F32, False)
    x, y = Buf(rng.standard_normal((T, 256)), F32), Buf.out((T, 512), F32)
    check(L.g53h_mm_w4(y.ptr, x.ptr, F32, T, C.byref(m.c), 0.0), "w4")
    want = x.val() @ m.wide[0].T
    assert np.linalg.norm(y.val() - want) < 1.2e-6 * np.linalg.norm(want)


def test_other_tokens_do_not_matter(L):
    """A token with an infinity or NaN spoils its own row only."""
    say("w4, not finite")
    rng = np.random.default_rng(9)
    m = W4(rng, 1, 50, 256, 64, F32, True)
    for dt in (F32, BF16, F16):
        xv = rng.standard_normal((6, 256))
        good = Buf(xv, dt)
        xv = xv.copy()
        xv[2, 100], xv[4, 0] = np.nan, np.inf
        bad = Buf(xv, dt)
        ya, yb = Buf.out((6, 50), dt), Buf.out((6, 50), dt)
        check(L.g53h_mm_w4(ya.ptr, good.ptr, dt, 6, C.byref(m.c), 0.0), "w4")
        check(L.g53h_mm_w4(yb.ptr, bad.ptr, dt, 6, C.byref(m.c), 0.0), "w4")
        assert np.isnan(yb.val()[[2, 4]]).all() and np.array_equal(ya.get()[[0, 1, 3, 5]], yb.get()[[0, 1, 3, 5]])


@pytest.mark.parametrize("T,K,NE,rows,cols,group,s_dt,zeros,sw,drop", [
    (1, 8, 288, 64, 256, 128, BF16, False, True, 0.0), (1, 1, 1, 5, 32, 32, F32, True, False, 0.0),
    (6, 4, 9, 40, 160, 64, F16, True, False, 0.2), (40, 6, 64, 34, 96, 32, F32, True, True, 0.1),
    (200, 8, 5, 24, 128, 128, F32, False, False, 0.0), (70, 3, 1000, 18, 64, 64, BF16, True, False, 0.4),
    (9, 2, 4, 10, 64, 64, F32, False, False, 1.0)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("gather", [1, 0])
def test_sorted_products(L, T, K, NE, rows, cols, group, s_dt, zeros, sw, drop, dt, gather):
    say("sorted w4", T, K, NE, rows, cols, group, s_dt, zeros, sw, drop, dt, gather)
    rng = np.random.default_rng(T + K + NE)
    idx = routing(rng, T, K, NE, drop)
    plan, (off, pair, _) = Plan(idx, NE), sorted_plan(idx, NE)
    n, out = off[NE], rows // 2 if sw else rows
    m = W4(rng, NE, rows, cols, group, s_dt, zeros)
    xv = rng.standard_normal((T if gather else T * K, cols))
    if not gather:
        xv[n:] = np.nan
    x, y = Buf(xv, dt), Buf.out((T * K, out), dt)
    check(L.g53h_sorted_mm_w4(y.ptr, x.ptr, dt, gather, plan.c, C.byref(m.c), LIMIT if sw else 0.0), "sorted w4")
    v, got = x.val(), y.val()
    for e in range(NE):
        a, b = off[e], off[e + 1]
        if a < b:
            want, tol = m.product(v[pair[a:b] // K] if gather else v[a:b], e)
            if sw:
                want, tol = swiglu(want, LIMIT), act_tol(want, tol, LIMIT)
            close(got[a:b], want, HALF[dt] * np.abs(want) + TINY[dt] + tol, e)
    assert (y.get()[n:] == enc([77.0], dt)).all()


@pytest.mark.parametrize("T,K,NE,expert,rows,cols", [(100, 2, 40, 39, 48, 256), (333, 1, 1000, 0, 40, 96), (70, 64, 64, 5, 16, 64),
                                                     (300, 3, 300, 299, 544, 2048)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_one_expert_takes_all(L, T, K, NE, expert, rows, cols, dt):
    """Every pair of every token the same expert, the others nothing: exact, whole numbers, and the same bits again."""
    say("sorted w4, one expert", T, K, NE, expert, rows, cols, dt)
    rng = np.random.default_rng(T)
    m = W4(rng, 1, rows, cols, 32, F32, True, exact=True)
    w, s, z = (glm53h.DevBuf(b.n * NE) for b in (m.w_d, m.s_d, m.z_d))
    for big, b in ((w, m.w_d), (s, m.s_d), (z, m.z_d)):
        check(L.g53h_memset(big.ptr, 0xff, b.n * NE), "memset")   # NaN scales elsewhere
        check(L.g53h_d2d(big.ptr + b.n * expert, b.ptr, b.n), "d2d")
    plan = Plan(np.full((T, K), expert, np.int32), NE)
    xv = rng.integers(-2, 3, (T, cols)).astype(float)
    x = Buf(xv, dt)
    c = glm53h.G53hW4(w.ptr, s.ptr, z.ptr, rows, cols, 32, F32)
    want = np.repeat(enc(xv @ m.wide[0].T, dt), K, 0)
    for _ in range(2):
        y = Buf.out((T * K, rows), dt)
        check(L.g53h_sorted_mm_w4(y.ptr, x.ptr, dt, 1, plan.c, C.byref(c), 0.0), "sorted w4")
        assert np.array_equal(y.get(), want)


def test_no_tokens(L):
    say("w4, no tokens")
    m = W4(np.random.default_rng(1), 1, 8, 32, 32, F32, False)
    assert L.g53h_mm_w4(None, None, BF16, 0, C.byref(m.c), 0.0) == 0
    off = Buf(np.zeros(2, np.int32))
    assert L.g53h_sorted_mm_w4(None, None, BF16, 0, glm53h.G53hSort(0, 1, 1, off.ptr, None, None), C.byref(m.c), 0.0) == 0


def test_matrix_past_2_gib(L):
    """Stacked matrices whose levels pass 2^31 bytes: the last expert's rows are its own."""
    say("w4, offsets past 32 bits")
    rows, cols, NE = 1024, 32768, 140
    one = rows * cols // 2
    assert one * NE > 1 << 31
    rng = np.random.default_rng(10)
    m = W4(rng, 1, rows, cols, 128, BF16, False, exact=True)
    w, s = glm53h.DevBuf(one * NE), glm53h.DevBuf(m.s_d.n * NE)
    check(L.g53h_memset(w.ptr, 0x88, one * NE), "memset")                    # every level 8: zero
    check(L.g53h_memset(s.ptr, 0x3f, m.s_d.n * NE), "memset")
    check(L.g53h_d2d(w.ptr + one * (NE - 1), m.w_d.ptr, one), "d2d")
    check(L.g53h_d2d(s.ptr + m.s_d.n * (NE - 1), m.s_d.ptr, m.s_d.n), "d2d")
    idx = np.array([[NE - 1, 3], [5, NE - 1]], np.int32)
    plan = Plan(idx, NE)
    xv = rng.integers(-2, 3, (2, cols)).astype(float)
    x, y = Buf(xv, BF16), Buf.out((4, rows), BF16)
    c = glm53h.G53hW4(w.ptr, s.ptr, None, rows, cols, 128, BF16)
    check(L.g53h_sorted_mm_w4(y.ptr, x.ptr, BF16, 1, plan.c, C.byref(c), 0.0), "sorted w4")
    got = y.get()
    assert (got[:2] == 0).all() and np.array_equal(got[2:], enc(xv @ m.wide[0].T, BF16))


def tight(m, x, dt, e=0):
    """x times matrix e, and what its sums may be off: a product is one of at most min(group, 128) of a partial sum, partial
    sums join the row's as often as the columns hold groups' pieces of 32 to 128, and then up to eight waves' and three
    planes' are added. Every addition is off by at most 2^-23 of the sum of its products' sizes (the matrix cores may cut
    what does not fit, which is a whole step). Levels enter as q - z, exactly; with bf16 as q, and z times the sum of x comes
    off: sizes are (q + z) |x| then."""
    depth = min(m.group, 128) + -(-x.shape[1] // min(m.group, 32 if m.group % 64 else 64 if m.group % 128 else 128)) + 16
    size = (m.lv[e] + m.z[e]) * m.s[e] if dt == BF16 else np.abs(m.wide[e])
    return x @ m.wide[e].T, depth * 2.0 ** -23 * (np.abs(x) @ size.T)


def centred(rng, m, zeros):
    """Levels as a quantiser makes them of N(0, 1) weights: the largest of a group 6 or 7 from its zero point, 6 to 9 or 8."""
    n, rows, cols = m.lv.shape
    gs = -(-cols // m.group)
    w = rng.standard_normal((n, rows, cols))
    top = np.repeat(np.abs(w).reshape(n, rows, gs, m.group).max(3), m.group, 2)
    if zeros:
        z = rng.integers(6, 10, (n, rows, gs + gs % 2)).astype(np.uint8)
        m.z = np.repeat(z[..., :gs], m.group, 2).astype(np.int64)
        m.z_d = Buf(z[..., 0::2] | (z[..., 1::2] << 4))
    levels(m, np.round(w / top * (6 if zeros else 7)).astype(np.int64) + m.z)


def levels(m, lv):
    m.lv, m.wide = lv, (lv - m.z) * m.s
    m.w_d = Buf((lv[..., 0::2] | (lv[..., 1::2] << 4)).astype(np.uint8))


def copies(L, m, n):
    """The arrays of n copies of m's rows below each other."""
    parts = [glm53h.DevBuf(b.n * n) if b else None for b in (m.w_d, m.s_d, m.z_d)]
    for big, b in zip(parts, (m.w_d, m.s_d, m.z_d)):
        for k in range(n if b else 0):
            check(L.g53h_d2d(big.ptr + k * b.n, b.ptr, b.n), "d2d")
    return parts


PATHS = [(1, 1), (5, 1), (6, 1), (24, 1), (1, 32), (5, 32), (12, 32), (40, 32)]   # tokens, copies of 520 rows


@pytest.mark.parametrize("T,n", PATHS)
@pytest.mark.parametrize("group,zeros", [(128, False), (128, True), (64, True), (32, True)])
@pytest.mark.parametrize("mean", [1.0, 10.0])
def test_fp32_error_whatever_the_mean(L, T, n, group, zeros, mean):
    """fp32 products of x = N(mean, 1) with weights around 0 are as near as a plain fp32 sum. Of 1024 columns a chunk of 128 is added in four
    steps, each off by at most a step (2^-23) of its partial sum, whose norm over the rows is at most sqrt(k / 4) of the
    chunk's at step k: 3.07 together; chunks' errors are independent, so the row's is 3.07 x 2^-23 = 3.7e-7 of its norm.
    Eight waves' sums and the chunks before them are added with half a step each of sqrt(j / 8): 5.9 x 2^-24 = 3.5e-7; a
    step's lower planes are 2^-8 of it. 7.2e-7 of the result's norm, and the spread of a norm over 512 rows makes 9e-7.
    (Groups of 32 and 64 trade steps of the first kind for as many of the second.)"""
    say("w4, fp32 error", T, n, group, zeros, mean)
    rng = np.random.default_rng(T + group)
    m = W4(rng, 1, 520, 1024, group, F32, zeros)
    centred(rng, m, zeros)
    parts = copies(L, m, n)
    x, y = Buf(rng.normal(mean, 1.0, (T, 1024)), F32), Buf.out((T, 520 * n), F32)
    c = glm53h.G53hW4(*[b.ptr if b else None for b in parts], 520 * n, 1024, group, F32)
    check(L.g53h_mm_w4(y.ptr, x.ptr, F32, T, C.byref(c), 0.0), "w4")
    want = x.val() @ m.wide[0].T
    got = y.val().reshape(T, n, 520)
    assert (got == got[:, :1]).all()
    off = np.linalg.norm(got[:, 0] - want) / np.linalg.norm(want)
    say("off by", off)
    assert off < 9e-7


@pytest.mark.parametrize("T,n", PATHS)
@pytest.mark.parametrize("group,zeros", [(128, False), (128, True), (96, True), (64, True), (32, False)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_a_large_value_that_a_level_makes_zero(L, T, n, group, zeros, dt):
    """One column of x is 2^13 to 2^30 times the others, and its levels are the zero point: it adds nothing, nor do its
    roundings in fp32 and fp16, where the bound is that of the other columns."""
    say("w4, large value", T, n, group, zeros, dt)
    rng = np.random.default_rng(T + group)
    m = W4(rng, 1, 520, 1024, group, F32, zeros)
    at = 700
    lv = m.lv.copy()
    lv[:, :, at] = m.z[:, :, at]
    levels(m, lv)
    parts = copies(L, m, n)
    xv = rng.standard_normal((T, 1024))
    xv[:, at] = {F32: 2.0 ** 30, F16: 2.0 ** 15, BF16: 2.0 ** 13}[dt]
    x, y = Buf(xv, dt), Buf.out((T, 520 * n), dt)
    c = glm53h.G53hW4(*[b.ptr if b else None for b in parts], 520 * n, 1024, group, F32)
    check(L.g53h_mm_w4(y.ptr, x.ptr, dt, T, C.byref(c), 0.0), "w4")
    want, tol = tight(m, x.val(), dt)
    got = y.val().reshape(T, n, 520)
    assert (got == got[:, :1]).all()
    close(got[:, 0], want, HALF[dt] * np.abs(want) + TINY[dt] + tol)


@pytest.mark.parametrize("T,n", PATHS)
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_a_value_that_is_not_finite_in_any_place(L, T, n, dt):
    """An infinity or NaN at any of 1024 columns makes all of its token's results NaN, and no other token's."""
    say("w4, not finite in any place", T, n, dt)
    rng = np.random.default_rng(T)
    m = W4(rng, 1, 520, 1024, 64, F32, True)
    parts = copies(L, m, n)
    c = glm53h.G53hW4(*[b.ptr if b else None for b in parts], 520 * n, 1024, 64, F32)
    xv = rng.standard_normal((T, 1024))
    x, ya, yb = Buf(xv, dt), Buf.out((T, 520 * n), dt), Buf.out((T, 520 * n), dt)
    check(L.g53h_mm_w4(ya.ptr, x.ptr, dt, T, C.byref(c), 0.0), "w4")
    good, size = ya.get(), x.n // x.shape[0] // 1024
    for k, (at, bad) in enumerate([(0, np.inf), (1, -np.inf), (6, np.nan), (39, -np.inf), (514, np.inf), (1023, np.inf)]):
        t = k % T
        one = Buf(np.array([bad]), dt)
        check(L.g53h_d2d(x.ptr + (t * 1024 + at) * size, one.ptr, size), "d2d")
        check(L.g53h_mm_w4(yb.ptr, x.ptr, dt, T, C.byref(c), 0.0), "w4")
        got = yb.val()
        assert np.isnan(got[t]).all(), (at, bad)
        rest = [i for i in range(T) if i != t]
        assert np.array_equal(yb.get()[rest], good[rest])
        one = Buf(xv[t, at:at + 1], dt)
        check(L.g53h_d2d(x.ptr + (t * 1024 + at) * size, one.ptr, size), "d2d")


@pytest.mark.parametrize("rows,limit", [((1 << 29) + 4096, 0.0), (1 << 30, 0.0), (1 << 30, LIMIT)])
def test_as_many_rows_as_there_may_be(L, rows, limit):
    """2^30 rows of 32 columns, 16 GiB of levels: copies of 4096 rows of whole numbers. (With SwiGLU: all copies alike, and
    the first one within its tolerance.)"""
    say("w4, many rows", rows, limit)
    rng = np.random.default_rng(17)
    m = W4(rng, 1, 4096, 32, 32, BF16, False, exact=True)
    parts = []
    for b in (m.w_d, m.s_d):
        big, have = glm53h.DevBuf(b.n // 4096 * rows), b.n
        check(L.g53h_d2d(big.ptr, b.ptr, b.n), "d2d")
        while have < big.nbytes:                                   # twice as much at a time
            more = min(have, big.nbytes - have)
            check(L.g53h_d2d(big.ptr + have, big.ptr, more), "d2d")
            have += more
        parts.append(big)
    c = glm53h.G53hW4(parts[0].ptr, parts[1].ptr, None, rows, 32, 32, BF16)
    x, out = Buf(rng.integers(-2, 3, (1, 32)).astype(float), BF16), rows // 2 if limit else rows
    y = glm53h.DevBuf(2 * out)
    check(L.g53h_memset(y.ptr, 0xff, 2 * out), "memset")           # NaN
    check(L.g53h_mm_w4(y.ptr, x.ptr, BF16, 1, C.byref(c), limit), "w4")
    got = y.download(np.uint16).reshape(-1, 4096)
    assert (got == got[0]).all()
    sums, tol = tight(m, x.val(), BF16)
    if limit:
        both, tol = np.concatenate((sums, sums), 1), np.concatenate((tol, tol), 1)    # gate and up rows are alike
        want, tol = swiglu(both, limit), act_tol(both, tol, limit)
        close(dec(got[:1], BF16), want, HALF[BF16] * np.abs(want) + TINY[BF16] + tol)
    else:
        assert np.array_equal(got[:1], enc(sums, BF16))


@pytest.mark.parametrize("T,rows,cols,group,s_dt,zeros,sw", CASES)
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_product_within_the_roundings_of_its_own_products(L, T, rows, cols, group, s_dt, zeros, sw, dt):
    """The bound counts |q - z| s |x| (bf16: q + z) and no more than 128 products a partial sum, so that a wrong wide group
    shows, with and without SwiGLU; and the whole is within half a step of the type and, for the sums, 2^-19."""
    say("w4, tight", T, rows, cols, group, s_dt, zeros, sw, dt)
    rng = np.random.default_rng(rows + cols + T + 2)
    m = W4(rng, 1, rows, cols, group, s_dt, zeros)
    x, out = Buf(rng.standard_normal((T, cols)), dt), rows // 2 if sw else rows
    y = Buf.out((T, out), dt)
    check(L.g53h_mm_w4(y.ptr, x.ptr, dt, T, C.byref(m.c), LIMIT if sw else 0.0), "w4")
    want, tol = tight(m, x.val(), dt)
    if sw:
        want, tol = swiglu(want, LIMIT), act_tol(want, tol, LIMIT)
    got = y.val()
    close(got, want, HALF[dt] * np.abs(want) + TINY[dt] + tol)
    if out * T >= 100:
        assert np.linalg.norm(got - want) <= (HALF[dt] + 2.0 ** -19) * np.linalg.norm(want)


class Stacked:
    """NE matrices of `n` copies of a tile of rows of their own: the tiles (W4) on the host, all of it on the device. With
    halves, gate over up: n copies of the tile's upper half of rows, then n of its lower half."""

    def __init__(self, L, rng, NE, tile, n, cols, group, s_dt, zeros, exact, halves=False):
        self.m = m = W4(rng, NE, tile, cols, group, s_dt, zeros, exact=exact)
        self.rows, parts = tile * n, []
        for b in (m.w_d, m.s_d, m.z_d):
            if b is None:
                parts.append(None)
                continue
            big, one = glm53h.DevBuf(b.n * n), b.n // NE                    # bytes of a tile
            piece = one // 2 if halves else one
            for e in range(NE):
                for h in range(2 if halves else 1):
                    for k in range(n):
                        check(L.g53h_d2d(big.ptr + (e * n * one) + (h * n + k) * piece, b.ptr + e * one + h * piece, piece), "d2d")
            parts.append(big)
        self.parts = parts
        self.c = glm53h.G53hW4(parts[0].ptr, parts[1].ptr, parts[2].ptr if zeros else None, tile * n, cols, group, s_dt)


@pytest.mark.parametrize("counts", [[40, 70, 0, 55, 33, 64, 47, 51], [1, 200, 0, 0, 31, 32, 33, 63]])
@pytest.mark.parametrize("gather", [1, 0])
@pytest.mark.parametrize("group,zeros,sw", [(128, True, False), (32, False, False), (64, True, True), (96, True, True)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_large_experts_of_many_rows(L, counts, gather, group, zeros, sw, dt):
    """A batch over eight large matrices, which go by 32 rows at a time: experts of uneven rows, some with none, some that end
    at a tile's end or one row behind it, tokens without an expert between them. Whole numbers are exact; with SwiGLU within
    the roundings of its sums."""
    say("sorted w4, large experts", counts, gather, group, zeros, sw, dt)
    rng = np.random.default_rng(group + sum(counts))
    NE, cols, tile, n = 8, 2112, 208, 20
    m = Stacked(L, rng, NE, tile, n, cols, group, BF16, zeros, not sw, halves=sw)
    flat = np.concatenate([np.full(k, e) for e, k in enumerate(counts)] + [np.full(9, -1)]).astype(np.int32)
    flat = rng.permutation(flat)
    K = 2 if len(flat) % 2 == 0 else 1
    idx = flat.reshape(-1, K)
    plan, (off, pair, _) = Plan(idx, NE), sorted_plan(idx, NE)
    last, out = off[NE], m.rows // 2 if sw else m.rows
    xv = rng.standard_normal((len(idx) if gather else flat.size, cols)) if sw else rng.integers(
        -2, 3, (len(idx) if gather else flat.size, cols)).astype(float)
    if not gather:
        xv[last:] = np.nan
    x, y = Buf(xv, dt), Buf.out((flat.size, out), dt)
    check(L.g53h_sorted_mm_w4(y.ptr, x.ptr, dt, gather, plan.c, C.byref(m.c), LIMIT if sw else 0.0), "sorted w4")
    v, got = x.val(), y.get()
    assert (got[last:] == enc([77.0], dt)).all()
    got = got[:last].reshape(last, n, -1)
    assert (got == got[:, :1]).all()                                        # copies alike
    for e in range(NE):
        a, b = off[e], off[e + 1]
        if a < b:
            want, tol = tight(m.m, v[pair[a:b] // K] if gather else v[a:b], dt, e)
            if sw:
                want, tol = swiglu(want, LIMIT), act_tol(want, tol, LIMIT)
                close(dec(got[a:b, 0], dt), want, HALF[dt] * np.abs(want) + TINY[dt] + tol, e)
            else:
                assert np.array_equal(got[a:b, 0], enc(want, dt)), e


@pytest.mark.parametrize("T", [33, 40, 64])
@pytest.mark.parametrize("group,zeros", [(128, True), (64, False), (32, True)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_swiglu_of_a_large_matrix_and_many_tokens(L, T, group, zeros, dt):
    say("w4, swiglu of a large matrix", T, group, zeros, dt)
    rng = np.random.default_rng(T + group)
    m = Stacked(L, rng, 1, 1040, 16, 4096, group, F16, zeros, False, halves=True)
    x, y = Buf(rng.standard_normal((T, 4096)), dt), Buf.out((T, 8320), dt)
    check(L.g53h_mm_w4(y.ptr, x.ptr, dt, T, C.byref(m.c), LIMIT), "w4")
    got = y.val().reshape(T, 16, 520)
    assert (got == got[:, :1]).all()
    sums, tol = tight(m.m, x.val(), dt)
    want, tol = swiglu(sums, LIMIT), act_tol(sums, tol, LIMIT)
    close(got[:, 0], want, HALF[dt] * np.abs(want) + TINY[dt] + tol)
    assert np.linalg.norm(got[:, 0] - want) <= (HALF[dt] + 2.0 ** -19) * np.linalg.norm(want)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_more_tokens_than_one_launch_takes(L, dt):
    """2^25 tokens and some, whose tiles are more than a launch's threads: copies of 4096 tokens of whole numbers."""
    say("w4, many tokens", dt)
    rng = np.random.default_rng(18)
    T, cols, rows = (1 << 25) + 3 * 4096, 32, 16
    m = W4(rng, 1, rows, cols, 32, F32, True, exact=True)
    one = Buf(rng.integers(-2, 3, (4096, cols)).astype(float), dt)
    x, have = glm53h.DevBuf(one.n // 4096 * T), one.n
    check(L.g53h_d2d(x.ptr, one.ptr, one.n), "d2d")
    while have < x.nbytes:
        more = min(have, x.nbytes - have)
        check(L.g53h_d2d(x.ptr + have, x.ptr, more), "d2d")
        have += more
    want = enc(one.val() @ m.wide[0].T, dt)
    y = glm53h.DevBuf(want.nbytes // 4096 * T)
    check(L.g53h_memset(y.ptr, 0xff, y.nbytes), "memset")                    # NaN
    check(L.g53h_mm_w4(y.ptr, x.ptr, dt, T, C.byref(m.c), 0.0), "w4")
    assert (y.download(want.dtype).reshape(-1, 4096, rows) == want).all()
