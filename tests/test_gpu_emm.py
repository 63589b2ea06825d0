"""Products of sorted rows with their experts' matrices, and their gradients, against 64 bits on the host: whole numbers,
whose sums are exact in fp32, to the bit, and normal values within the roundings of their sums."""
import numpy as np
import pytest

import glm53h
from glm53h import DevBuf, check
from op_lib import BF16, F16, F32, HALF, TINY, Buf, Plan, close, dec, enc, routing, sorted_plan, swiglu
from test_gpu_parity import say

pytestmark = pytest.mark.gpu
LIMIT = 2.0


@pytest.fixture(scope="module")
def L():
    return glm53h.init(0)


def rounded(a, dt):
    return dec(enc(a, dt), dt)


def values(rng, shape, dt, whole, scale=1.0):
    """Whole numbers of -3 to 3, or normal values of the type."""
    return rng.integers(-3, 4, shape).astype(np.float64) if whole else rounded(scale * rng.standard_normal(shape), dt)


def off(n, size, y, dt, whole, limit_slope=1.0):
    """What sums of n products in fp32, in any order, and the rounding to the type may be off by: every addition at
    most 2^-23 (a matrix core may cut instead of rounding) of the sum of the sizes; fp32 values' products 2^-24 each
    besides (2^-26 left out by the planes, doubled for the two roundings of planes)."""
    if whole:
        return HALF[dt] * np.abs(y) + TINY[dt]
    return limit_slope * (n + 32 + 6 * n / 32) * 2.0 ** -23 * size + HALF[dt] * np.abs(y) + TINY[dt]


# (T, K, NE, rows, cols): single tokens, tiles cut in every way, odd sizes, experts without rows, one that takes all
SIZES = [(1, 1, 1, 1, 1), (1, 4, 16, 64, 64), (5, 2, 3, 30, 40), (33, 3, 7, 130, 72), (70, 1, 1, 258, 200), (129, 2, 4, 136, 8),
         (64, 4, 300, 48, 96), (300, 2, 2, 66, 333), (17, 2, 5, 514, 301)]


def cases():
    for i, s in enumerate(SIZES):
        for dt in (BF16, F16, F32):
            yield s + (dt, i % 2, (i // 2 + dt) % 2, (i + dt) % 3 == 0)


@pytest.mark.parametrize("T,K,NE,rows,cols,dt,gather,sw,shifted", cases())
def test_forward(L, T, K, NE, rows, cols, dt, gather, sw, shifted):
    say("forward", T, K, NE, rows, cols, dt, gather, sw, shifted)
    rng = np.random.default_rng(T + rows)
    rows += rows % 2 if sw else 0
    idx = routing(rng, T, K, NE, 0.2)
    idx[rng.random((T, K)) < 0.1] = NE                       # outside
    offsets, pair, _ = sorted_plan(idx, NE)
    n, used, out = T * K, offsets[NE], rows // 2 if sw else rows
    shift = (2 if dt != F32 else 4) if shifted else 0
    plan = Plan(idx, NE)
    for whole in (True, False):
        xv = values(rng, (T if gather else n, cols), dt, whole)
        wv = values(rng, (NE, rows, cols), dt, whole, 0.1)
        x, w = Buf(xv, dt, shift), Buf(wv, dt, shift)
        ys, gu = Buf.out((n, out), dt, shift), Buf.out((n, rows), dt, shift)
        check(L.g53h_sorted_mm(ys.ptr, gu.ptr if sw else None, x.ptr, dt, gather, plan.c, w.ptr, rows, cols, LIMIT if sw else 0.0))
        ref, size, act = np.full((n, rows), 77.0), np.zeros((n, rows)), np.full((n, out), 77.0)
        for e in range(NE):
            r = slice(offsets[e], offsets[e + 1])
            xe = xv[pair[r] // K] if gather else xv[r]
            ref[r], size[r] = xe @ wv[e].T, np.abs(xe) @ np.abs(wv[e]).T
        tol = off(cols, size, ref, dt, whole)
        tol[used:] = 0
        if not sw:
            close(ys.val(), ref, tol, whole)
            continue
        close(gu.val(), ref, tol, ("gu", whole))
        act[:used] = swiglu(ref[:used], LIMIT)
        # |d silu| <= 1.1 and |up| <= limit, |silu| <= limit and slope 1: sums of both; expf and the division 4 steps
        sums = off(cols, size, ref, F32, whole)
        ta = np.zeros((n, out))
        ta[:used] = (1.1 * LIMIT * (sums[:used, :out] + sums[:used, out:]) + (4 * 2.0 ** -23 + HALF[dt]) * np.abs(act[:used]) + TINY[dt]) * 1.01
        close(ys.val(), act, ta, ("act", whole))


@pytest.mark.parametrize("T,K,NE,rows,cols,dt,gather,w32,shifted", cases())
def test_gradients(L, T, K, NE, rows, cols, dt, gather, w32, shifted):
    say("gradients", T, K, NE, rows, cols, dt, gather, w32, shifted)
    rng = np.random.default_rng(T + cols)
    idx = routing(rng, T, K, NE, 0.2)
    if NE > 1:
        idx[idx == 1] = -1                                   # an expert without rows
    offsets, pair, _ = sorted_plan(idx, NE)
    n, used, wt = T * K, offsets[NE], F32 if w32 else dt
    shift = (2 if dt != F32 else 4) if shifted else 0
    plan = Plan(idx, NE)
    for whole in (True, False):
        xv = values(rng, (T if gather else n, cols), dt, whole)
        wv, dv = values(rng, (NE, rows, cols), dt, whole, 0.1), values(rng, (n, rows), dt, whole)
        old = values(rng, (NE, rows, cols), wt, whole)
        x, w, d = Buf(xv, dt, shift), Buf(wv, dt, shift), Buf(dv, dt, shift)
        dx, dw, da = Buf.out((n, cols), dt, shift), Buf.out((NE, rows, cols), wt), Buf(old, wt)
        check(L.g53h_sorted_mm_grad(dx.ptr, dw.ptr, wt, 0, d.ptr, x.ptr, dt, gather, plan.c, w.ptr, rows, cols))
        check(L.g53h_sorted_mm_grad(None, da.ptr, wt, 1, d.ptr, x.ptr, dt, gather, plan.c, None, rows, cols))
        rx, sx = np.full((n, cols), 77.0), np.zeros((n, cols))
        rw, sz, many = np.zeros((NE, rows, cols)), np.zeros((NE, rows, cols)), np.zeros((NE, 1, 1))
        for e in range(NE):
            r = slice(offsets[e], offsets[e + 1])
            xe = xv[pair[r] // K] if gather else xv[r]
            rx[r], sx[r] = dv[r] @ wv[e], np.abs(dv[r]) @ np.abs(wv[e])
            rw[e], sz[e], many[e] = dv[r].T @ xe, np.abs(dv[r]).T @ np.abs(xe), r.stop - r.start
        tol = off(rows, sx, rx, dt, whole)
        tol[used:] = 0
        close(dx.val(), rx, tol, ("dx", whole))
        close(dw.val(), rw, off(many, sz, rw, wt, whole), ("dw", whole))
        close(da.val(), old + rw, off(many + 1, sz + np.abs(old), old + rw, wt, whole), ("added", whole))
        again = Buf.out((n, cols), dt, shift)
        check(L.g53h_sorted_mm_grad(again.ptr, None, wt, 0, d.ptr, None, dt, gather, plan.c, w.ptr, rows, cols))
        assert np.array_equal(again.get(), dx.get())


@pytest.mark.parametrize("T,K,inter,dt", [(1, 1, 1, F32), (5, 2, 33, BF16), (9, 3, 2056, F16), (30, 4, 128, F32), (7, 1, 4099, BF16)])
def test_swiglu_grad(L, T, K, inter, dt):
    say("swiglu_grad", T, K, inter, dt)
    rng = np.random.default_rng(inter)
    NE, n = 6, T * K
    idx = routing(rng, T, K, NE, 0.2)
    idx[0, 0] = 1
    used = sorted_plan(idx, NE)[0][NE]
    gv = rounded(2.0 * rng.standard_normal((n, 2 * inter)), dt)
    gv[0, :: max(1, inter // 7)] = LIMIT                     # at the limit: inside
    gv[n // 2, inter:] = -LIMIT
    gv[n - 1, 0] = -100.0                                    # exp of it overflows
    dv = rounded(rng.standard_normal((n, inter)), dt)
    gu, d, plan = Buf(gv, dt), Buf(dv, dt), Plan(idx, NE)
    out = Buf.out((n, 2 * inter), dt)
    check(L.g53h_sorted_swiglu_grad(out.ptr, d.ptr, gu.ptr, dt, inter, plan.c, LIMIT))
    g, u = gv[:, :inter], gv[:, inter:]
    gc, uc = np.minimum(g, LIMIT), np.clip(u, -LIMIT, LIMIT)
    s = 1.0 / (1.0 + np.exp(-gc))
    want = np.concatenate([np.where(g <= LIMIT, dv * uc * s * (1 + gc * (1 - s)), 0),
                           np.where(np.abs(u) <= LIMIT, dv * gc * s, 0)], 1)
    # ten operations of half a step each; 1 - s and 1 + gc (1 - s) are off by steps of their parts
    size = np.concatenate([np.abs(dv * uc) * s * (1 + np.abs(gc)), np.abs(dv * gc) * s], 1)
    # below 2^-126 fp32 has steps of 2^-149: s, formed by an exponential and a division, is off by half of one each, and
    # enters as s d u (1 + g) and s d g
    deep = 2.0 ** -149 * np.concatenate([np.abs(dv * uc) * (1 + np.abs(gc)), np.abs(dv * gc)], 1)
    tol = 16 * 2.0 ** -24 * size + deep + HALF[dt] * np.abs(want) + TINY[dt]
    want[used:], tol[used:] = 77.0, 0
    close(out.val(), want, tol)
    check(L.g53h_sorted_swiglu_grad(gu.ptr, d.ptr, gu.ptr, dt, inter, plan.c, LIMIT))      # in place
    assert np.array_equal(gu.get()[:used], out.get()[:used]) and np.array_equal(gu.get()[used:], enc(gv, dt)[used:])
    # against differences, away from the limits
    e = 1e-6
    f = lambda v: swiglu(v, LIMIT)                           # noqa: E731
    near = np.abs(np.abs(gv) - LIMIT) < 1e-4
    for half in (0, 1):
        step = np.zeros_like(gv)
        step[:, half * inter:(half + 1) * inter] = e
        diff = dv * (f(gv + step) - f(gv - step)) / (2 * e)
        part = slice(half * inter, (half + 1) * inter)
        ok = ~near[:used, part]
        assert (np.abs(diff[:used] - want[:used, part])[ok] <= 1e-8 * (1 + np.abs(dv[:used])[ok]) * 8).all()


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_values_that_are_not_finite_stay_in_their_rows(L, dt):
    say("not finite", dt)
    rng = np.random.default_rng(3)
    T, NE, rows, cols = 40, 3, 70, 96
    idx = routing(rng, T, 1, NE)
    offsets, pair, row = sorted_plan(idx, NE)
    xv, wv = values(rng, (T, cols), dt, True), values(rng, (NE, rows, cols), dt, True)
    dv = values(rng, (T, rows), dt, True)
    xv[7, 3], xv[20, 95], dv[row[7], 5] = np.inf, np.nan, np.nan
    x, w, d, plan = Buf(xv, dt), Buf(wv, dt), Buf(dv, dt), Plan(idx, NE)
    ys, dx = Buf.out((T, rows), dt), Buf.out((T, cols), dt)
    check(L.g53h_sorted_mm(ys.ptr, None, x.ptr, dt, 1, plan.c, w.ptr, rows, cols, 0.0))
    check(L.g53h_sorted_mm_grad(dx.ptr, None, dt, 0, d.ptr, None, dt, 1, plan.c, w.ptr, rows, cols))
    y, g = ys.val(), dx.val()
    for r in range(T):
        t = pair[r]
        e = idx[t, 0]
        if t in (7, 20):
            assert not np.isfinite(y[r][wv[e][:, 3 if t == 7 else 95] != 0]).any()
        else:
            assert np.array_equal(y[r], rounded(wv[e] @ xv[t], dt))
        if t == 7:
            assert np.isnan(g[r]).all()
        else:
            assert np.array_equal(g[r], rounded(dv[r] @ wv[e], dt))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_nothing_to_do(L, dt):
    say("nothing", dt)
    rows, cols, NE = 40, 24, 4
    w = Buf(np.ones((NE, rows, cols)), dt)
    dw = Buf.out((NE, rows, cols), dt)
    plan = Plan(np.full((3, 2), -1, np.int32), NE)           # no pair has an expert
    x, ys, d = Buf(np.full((3, cols), np.nan), dt), Buf.out((6, rows), dt), Buf(np.full((6, rows), np.nan), dt)
    dx = Buf.out((6, cols), dt)
    check(L.g53h_sorted_mm(ys.ptr, None, x.ptr, dt, 1, plan.c, w.ptr, rows, cols, 0.0))
    check(L.g53h_sorted_mm_grad(dx.ptr, dw.ptr, dt, 0, d.ptr, x.ptr, dt, 1, plan.c, w.ptr, rows, cols))
    assert (ys.val() == 77).all() and (dx.val() == 77).all() and (dw.val() == 0).all()
    none = Plan(np.zeros((0, 2), np.int32), NE)              # no tokens at all
    dw = Buf.out((NE, rows, cols), dt)
    check(L.g53h_sorted_mm(None, None, None, dt, 1, none.c, None, rows, cols, 0.0))
    check(L.g53h_sorted_swiglu_grad(None, None, None, dt, rows // 2, none.c, 1.0))
    check(L.g53h_sorted_mm_grad(None, dw.ptr, dt, 0, None, None, dt, 1, none.c, None, rows, cols))
    assert (dw.val() == 0).all()
    check(L.g53h_sorted_mm_grad(None, dw.ptr, dt, 1, None, None, dt, 1, none.c, None, rows, cols))
    assert (dw.val() == 0).all()


def test_offsets_past_32_bits(L):
    """Results and matrices whose bytes and elements pass 2^32: the last ones are right."""
    say("large")
    rng = np.random.default_rng(5)
    T, K, NE, rows, cols = 70000, 8, 2, 8000, 64             # ys: 4.48e9 elements
    n = T * K
    idx = np.tile(np.array([0, 0, 0, 0, 1, 1, 1, 1], np.int32), (T, 1))
    xv, wv = values(rng, (T, cols), BF16, True), values(rng, (NE, rows, cols), BF16, True)
    x, w, plan = Buf(xv, BF16), Buf(wv, BF16), Plan(idx, NE)
    ys = DevBuf(2 * n * rows)
    check(L.g53h_sorted_mm(ys.ptr, None, x.ptr, BF16, 1, plan.c, w.ptr, rows, cols, 0.0))
    offsets, pair, _ = sorted_plan(idx, NE)
    for r in (0, n // 2 - 1, n // 2, (1 << 32) // rows, (1 << 31) // rows, n - 1):
        got = dec(ys.download(np.uint16, rows, 2 * r * rows), BF16)
        assert np.array_equal(got, rounded(wv[int(r >= n // 2)] @ xv[pair[r] // K], BF16)), r
    # the rows' gradient reads them again: of the last rows, whole numbers once more
    last = values(rng, (8, rows), BF16, True)
    L.g53h_memset(ys.ptr, 0, ys.nbytes)
    bits = enc(last, BF16)
    check(L.g53h_h2d(ys.ptr + 2 * (n - 8) * rows, bits.ctypes.data, bits.nbytes))
    dx, dw = DevBuf(2 * n * cols), Buf.out((NE, rows, cols), F32)
    check(L.g53h_sorted_mm_grad(dx.ptr, dw.ptr, F32, 0, ys.ptr, x.ptr, BF16, 1, plan.c, w.ptr, rows, cols))
    got = dec(dx.download(np.uint16, 8 * cols, 2 * (n - 8) * cols), BF16).reshape(8, cols)
    assert np.array_equal(got, rounded(last @ wv[1], BF16))
    assert np.array_equal(dw.val()[1], last.T @ xv[pair[n - 8:] // K]) and not dw.val()[0].any()


def test_matrices_past_32_bits(L):
    say("large matrices")
    rng = np.random.default_rng(6)
    NE, rows, cols, T = 20, 8192, 16400, 3                   # 2.7e9 elements, 5.4e9 bytes
    one = values(rng, (rows, cols), F16, True)
    w = DevBuf(2 * NE * rows * cols)
    bits = enc(one, F16)
    check(L.g53h_h2d(w.ptr + 2 * (NE - 1) * rows * cols, bits.ctypes.data, bits.nbytes))
    idx = np.full((T, 1), NE - 1, np.int32)
    xv, dv, plan = values(rng, (T, cols), F16, True), values(rng, (T, rows), F16, True), Plan(idx, NE)
    x, d, ys, dx = Buf(xv, F16), Buf(dv, F16), Buf.out((T, rows), F16), Buf.out((T, cols), F16)
    check(L.g53h_sorted_mm(ys.ptr, None, x.ptr, F16, 1, plan.c, w.ptr, rows, cols, 0.0))
    check(L.g53h_sorted_mm_grad(dx.ptr, None, F16, 0, d.ptr, None, F16, 1, plan.c, w.ptr, rows, cols))
    assert np.array_equal(ys.val(), rounded(xv @ one.T, F16)) and np.array_equal(dx.val(), rounded(dv @ one, F16))
    check(L.g53h_sorted_mm_grad(None, w.ptr, F16, 0, d.ptr, x.ptr, F16, 1, plan.c, None, rows, cols))
    at = (NE - 1) * rows * cols
    assert np.array_equal(dec(w.download(np.float16, rows * cols, 2 * at), F16).reshape(rows, cols), dv.T @ xv)
    assert not w.download(np.uint16, 1 << 20, 2 * (at - (1 << 20))).any()


# (T, NE, N, K): as many tiles as every form of the kernel takes, with ends of each
@pytest.mark.parametrize("T,NE,N,K", [(300, 1, 33032, 72), (200, 3, 12296, 136), (300, 1, 22024, 64), (100, 2, 33800, 40), (40, 40, 1800, 88),
                                      (3, 3, 700, 520)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_every_tile(L, T, NE, N, K, dt):
    say("tiles", T, NE, N, K, dt)
    rng = np.random.default_rng(N)
    idx = rng.integers(0, NE, (T, 1)).astype(np.int32)
    offsets, pair, _ = sorted_plan(idx, NE)
    plan = Plan(idx, NE)
    xv, wv = values(rng, (T, K), dt, True), values(rng, (NE, N, K), dt, True)
    x, w, ys, gu = Buf(xv, dt), Buf(wv, dt), Buf.out((T, N), dt), Buf.out((T, N), dt)
    act = Buf.out((T, N // 2), dt)
    check(L.g53h_sorted_mm(ys.ptr, None, x.ptr, dt, 1, plan.c, w.ptr, N, K, 0.0))
    check(L.g53h_sorted_mm(act.ptr, gu.ptr, x.ptr, dt, 1, plan.c, w.ptr, N, K, LIMIT))
    ref = np.concatenate([xv[pair[offsets[e]:offsets[e + 1]]] @ wv[e].T for e in range(NE)])
    assert np.array_equal(ys.val(), rounded(ref, dt)) and np.array_equal(gu.val(), ys.val())
    want = swiglu(ref, LIMIT)
    # sums are exact; the hardware's exponential and reciprocal 2^-20, the products 2^-23; the exponential is zero where it
    # lies below 2^-126, which leaves out g u times as much
    g, u = np.split(ref, 2, 1)
    deep = np.where(g < -87, 2.0 ** -126 * np.abs(g * np.clip(u, -LIMIT, LIMIT)), 0)
    close(act.val(), want, (2.0 ** -20 + HALF[dt]) * np.abs(want) + TINY[dt] + deep)
    # the rows' gradient, of matrices the other way round: [K][N], dys [T][K]
    wt = np.ascontiguousarray(wv.transpose(0, 2, 1))
    w2, dx = Buf(wt, dt), Buf.out((T, N), dt)
    dy = Buf(xv[pair], dt)
    check(L.g53h_sorted_mm_grad(dx.ptr, None, dt, 0, dy.ptr, None, dt, 1, plan.c, w2.ptr, K, N))
    assert np.array_equal(dx.get(), ys.get())
    # the matrices' gradient [K][N] of the same rows and others
    zv = values(rng, (T, N), dt, True)
    z, dw = Buf(zv, dt), Buf.out((NE, K, N), F32)
    check(L.g53h_sorted_mm_grad(None, dw.ptr, F32, 0, dy.ptr, z.ptr, dt, 0, plan.c, None, K, N))
    for e in range(NE):
        r = slice(offsets[e], offsets[e + 1])
        assert np.array_equal(dw.val()[e], xv[pair[r]].T @ zv[r])


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("w32", [0, 1])
def test_results_at_any_element(L, dt, w32):
    """Operands at multiples of 16 bytes, results that start one element on, odd result columns among them."""
    say("results off", dt, w32)
    rng = np.random.default_rng(12)
    for T, NE, rows, cols in ((70, 2, 137, 64), (5, 3, 72, 136), (200, 2, 264, 72)):
        idx = rng.integers(0, NE, (T, 1)).astype(np.int32)
        offsets, pair, _ = sorted_plan(idx, NE)
        plan, wt = Plan(idx, NE), F32 if w32 else dt
        xv, wv, dv = values(rng, (T, cols), dt, True), values(rng, (NE, rows, cols), dt, True), values(rng, (T, rows), dt, True)
        x, w, d = Buf(xv, dt), Buf(wv, dt), Buf(dv, dt)
        one = 4 if dt == F32 else 2
        ys, dx, dw = Buf.out((T, rows), dt, one), Buf.out((T, cols), dt, one), Buf.out((NE, rows, cols), wt, 4 if wt == F32 else 2)
        check(L.g53h_sorted_mm(ys.ptr, None, x.ptr, dt, 1, plan.c, w.ptr, rows, cols, 0.0))
        check(L.g53h_sorted_mm_grad(dx.ptr, dw.ptr, wt, 0, d.ptr, x.ptr, dt, 1, plan.c, w.ptr, rows, cols))
        for e in range(NE):
            r = slice(offsets[e], offsets[e + 1])
            assert np.array_equal(ys.val()[r], rounded(xv[pair[r]] @ wv[e].T, dt))
            assert np.array_equal(dx.val()[r], rounded(dv[r] @ wv[e], dt))
            assert np.array_equal(dw.val()[e], rounded(dv[r].T @ xv[pair[r]], wt))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_swiglu_grad_of_deep_gates(L, dt):
    """Gates from -60 down to the type's lowest value and -inf, as a forward pass may store them: gradients that fade to
    zero; gates and ups above the clamps up to inf have none, NaN stays."""
    say("deep gates", dt)
    rng = np.random.default_rng(13)
    low = {F32: -3.4e38, BF16: -3.38e38, F16: -65504.0}[dt]
    gates = np.array([-60.0, -79.5, -80.5, -86.0, -88.0, -95.0, -103.0, -110.0, -200.0, -999.0, -1001.0, -5e4, low, -np.inf, np.inf, -0.0])
    T, inter = 9, gates.size
    plan = Plan(np.zeros((T, 1), np.int32), 1)
    gv = np.tile(gates, (T, 2))
    gv[:, inter:] = rounded(rng.standard_normal((T, inter)), dt)
    gv[1, inter:], gv[2, inter:] = np.inf, -np.inf
    gv = rounded(gv, dt)
    gv[3, 0], gv[3, inter + 1] = np.nan, np.nan
    dv = rounded(rng.standard_normal((T, inter)), dt)
    gu, d, out = Buf(gv, dt), Buf(dv, dt), Buf.out((T, 2 * inter), dt)
    check(L.g53h_sorted_swiglu_grad(out.ptr, d.ptr, gu.ptr, dt, inter, plan.c, LIMIT))
    g, u = gv[:, :inter], gv[:, inter:]
    gc, uc = np.maximum(np.minimum(g, LIMIT), -1000.0), np.clip(u, -LIMIT, LIMIT)     # at -1000 s is 0 in fp32
    with np.errstate(over="ignore"):
        s = 1.0 / (1.0 + np.exp(-gc))
    want = np.concatenate([np.where(g > LIMIT, 0, dv * uc * s * (1 + gc * (1 - s))), np.where(np.abs(u) > LIMIT, 0, dv * gc * s)], 1)
    # as in test_swiglu_grad, whose `deep` counts s below the normal range. The product d u s is rounded there too, to a
    # multiple of 2^-149, before it is multiplied by 1 + g (1 - s): 2^-150 (1 + |g|) however small d u is
    size = np.concatenate([np.abs(dv * uc) * s * (1 + np.abs(gc)), np.abs(dv * gc) * s], 1)
    deep = 2.0 ** -149 * np.concatenate([np.abs(dv * uc) * (1 + np.abs(gc)) + 0.5 * (1 + np.abs(gc)), np.abs(dv * gc)], 1)
    close(out.val(), want, 16 * 2.0 ** -24 * size + deep + HALF[dt] * np.abs(want) + TINY[dt])


def test_gates_past_fp16_forward_and_back(L):
    """A gate's sum that passes fp16: the activation is 0 or clamped, gate and up are kept as infinities, and no gradient that
    comes of them is one, or NaN."""
    say("gates past fp16")
    rng = np.random.default_rng(14)
    T, inter, cols = 12, 8, 16
    xv, wv = rng.integers(-3, 4, (T, cols)).astype(float), rng.integers(-3, 4, (1, 2 * inter, cols)).astype(float)
    xv[:, 0], wv[0, :, 0] = 300.0, 0.0
    wv[0, 0, 0], wv[0, 1, 0], wv[0, inter + 2, 0], wv[0, inter + 3, 0] = -300.0, 300.0, -300.0, 300.0
    x, w, plan = Buf(xv, F16), Buf(wv, F16), Plan(np.zeros((T, 1), np.int32), 1)
    act, gu = Buf.out((T, inter), F16), Buf.out((T, 2 * inter), F16)
    check(L.g53h_sorted_mm(act.ptr, gu.ptr, x.ptr, F16, 1, plan.c, w.ptr, 2 * inter, cols, LIMIT))
    kept = gu.val()
    assert (kept[:, [0, inter + 2]] == -np.inf).all() and (kept[:, [1, inter + 3]] == np.inf).all()
    assert np.isfinite(act.val()).all() and not act.val()[:, 0].any()
    dv = rng.integers(-3, 4, (T, inter)).astype(float)
    d, dgu, dx, dw = Buf(dv, F16), Buf.out((T, 2 * inter), F16), Buf.out((T, cols), F16), Buf.out((1, 2 * inter, cols), F32)
    check(L.g53h_sorted_swiglu_grad(dgu.ptr, d.ptr, gu.ptr, F16, inter, plan.c, LIMIT))
    check(L.g53h_sorted_mm_grad(dx.ptr, dw.ptr, F32, 0, dgu.ptr, x.ptr, F16, 1, plan.c, w.ptr, 2 * inter, cols))
    v = dgu.val()
    assert not v[:, [0, 1, inter, inter + 2, inter + 3]].any()           # the two gates, the deep gate's up, the two ups
    s = 1 / (1 + np.exp(-LIMIT))
    assert (np.abs(v[:, inter + 1] - np.where(np.abs(kept[:, inter + 1]) <= LIMIT, dv[:, 1] * LIMIT * s, 0)) <= 2.0 ** -10 * 8).all()
    assert np.isfinite(v).all() and np.isfinite(dx.val()).all() and np.isfinite(dw.val()).all() and not dw.val()[0, [0, inter]].any()


@pytest.mark.parametrize("n", [1, 300])
def test_products_whose_parts_are_largest(L, n):
    """fp32 values whose second and third bf16 parts are as large as they get, 2^-8 and 2^-17 of them, so that the products
    of parts that are left out come near their bound, 2^-24 of a product, and of one sign: sums of n."""
    say("largest parts", n)
    hard = np.array([float.fromhex(v) for v in ("0x1.00ff8p0", "0x1.01008p0", "0x1.00fe8p0", "0x1.20ff8p0")])
    T, N = 40, 70
    scale = np.exp2(np.arange(N) % 5 - 2.0)
    av = np.repeat(hard[np.arange(T) % 4][:, None], n, 1)                # [T][n]: a row's values alike
    bv = np.repeat((hard[np.arange(N) % 4] * scale)[:, None], n, 1)       # [N][n]
    want = av @ bv.T
    # besides: one product's parts are added in three steps of at most 2^-8 of it and one of its own size, each of 2^-23
    # (cut); sums of more add what test_forward's do
    tol = (2.0 ** -24 + 2.0 ** -23 + 3 * 2.0 ** -31) * want if n == 1 else off(n, want, want, F32, False) + 2.0 ** -24 * want
    plan = Plan(np.zeros((T, 1), np.int32), 1)
    x, w, ys = Buf(av, F32), Buf(bv[None], F32), Buf.out((T, N), F32)
    check(L.g53h_sorted_mm(ys.ptr, None, x.ptr, F32, 1, plan.c, w.ptr, N, n, 0.0))
    close(ys.val(), want, tol, "forward")
    wt, dx = Buf(np.ascontiguousarray(bv.T)[None], F32), Buf.out((T, N), F32)
    check(L.g53h_sorted_mm_grad(dx.ptr, None, F32, 0, x.ptr, None, F32, 1, plan.c, wt.ptr, n, N))
    close(dx.val(), want, tol, "rows")
    plan = Plan(np.zeros((n, 1), np.int32), 1)
    d, z, dw = Buf(np.ascontiguousarray(av.T), F32), Buf(np.ascontiguousarray(bv.T), F32), Buf.out((1, T, N), F32)
    check(L.g53h_sorted_mm_grad(None, dw.ptr, F32, 0, d.ptr, z.ptr, F32, 1, plan.c, None, T, N))
    close(dw.val()[0], want, tol, "matrices")


@pytest.mark.parametrize("what", ["small", "smaller", "large", "past"])
def test_fp32_at_the_ends_of_its_range(L, what):
    say("ends of fp32", what)
    rng = np.random.default_rng(15)
    T, N, K = 34, 66, 40
    one = 1.0 + rng.integers(0, 1 << 23, T) / 2.0 ** 23
    v = {"small": one * 2.0 ** -109, "smaller": one * np.exp2(-rng.integers(112, 127, T).astype(float)),
         "large": np.full(T, float.fromhex("0x1.fefffep127")), "past": np.full(T, float.fromhex("0x1.ffp127"))}[what]
    up = 2.0 ** (-120 if what in ("large", "past") else 100)
    xv, wv = np.zeros((T, K)), np.zeros((1, N, K))
    at = np.arange(T) % K
    xv[np.arange(T), at] = v
    xv[5] = 0.0                                              # a row of zeros among them
    wv[0] = up * np.exp2(np.arange(N) % 3)[:, None]
    want = xv @ wv[0].T
    plan = Plan(np.zeros((T, 1), np.int32), 1)
    x, w, ys = Buf(xv, F32), Buf(wv, F32), Buf.out((T, N), F32)
    check(L.g53h_sorted_mm(ys.ptr, None, x.ptr, F32, 1, plan.c, w.ptr, N, K, 0.0))
    wt, dx = Buf(np.ascontiguousarray(wv[0].T)[None], F32), Buf.out((T, N), F32)
    check(L.g53h_sorted_mm_grad(dx.ptr, None, F32, 0, x.ptr, None, F32, 1, plan.c, wt.ptr, K, N))
    dw = Buf.out((1, K, N), F32)
    ones = np.broadcast_to(wv[0, :, 0], (T, N))
    z = Buf(np.ascontiguousarray(ones), F32)
    check(L.g53h_sorted_mm_grad(None, dw.ptr, F32, 0, x.ptr, z.ptr, F32, 1, plan.c, None, K, N))
    wantw = xv.T @ ones
    for got, ref in ((ys.val(), want), (dx.val(), want), (dw.val()[0], wantw)):
        if what in ("small", "large"):                       # a value times a power of two: exact
            assert np.array_equal(got, ref)
        elif what == "smaller":                              # held to half of bf16's smallest step, 2^-133
            assert (np.abs(got - ref) <= 2.0 ** -134 * up * 4 + 2.0 ** -24 * np.abs(ref)).all()
        else:
            assert np.isnan(got[np.abs(ref).max(1) > 0]).all() and not got[np.abs(ref).max(1) == 0].any()


def tile(cus, op, dt, n, NE, rows, cols, whole):
    """The tile (rows, columns of the result) that the library takes for n rows, by its rule, or "stream" for the matrices'
    gradient in 16 bits; whole: operands of whole pieces of 16 bytes."""
    busy = min(NE, n)
    mean, size = -(-n // busy), rows if op == "forward" else cols
    count = lambda bm, bn: (n // bm + busy) * -(-size // bn)                         # noqa: E731
    few = NE * -(-rows // 128) * -(-cols // 128) < cus if op == "matrices" else mean <= 64
    if op == "rows" and few and count(32, 128) < cus and (dt == F32 or not whole):
        return 32, 64
    if dt == F32 or not whole:
        return (32, 128) if few else (128, 128)
    if op == "matrices":
        return "stream"
    if mean >= 64 and count(256, 256) >= cus:
        return 256, 256
    if mean >= 128 and count(128, 128) >= 2 * cus:
        return 128, 128
    if op == "rows" and mean > 1 and count(64, 256) >= 2 * cus:
        return 64, 256
    return (64, 128) if mean > 4 and count(64, 128) >= 2 * cus else (32, 128)


# rows of every expert, rows and columns of a matrix, bytes off a multiple of 16: the tiles that the other tests' sizes do not take,
# on 256 CUs, with ends of every kind
FORMS = [("rows", (64, 256), (BF16, F16), (70, 30), 72, 43768, 0), ("rows", (64, 256), (BF16, F16), (33, 0, 64, 16), 136, 33032, 0),
         ("rows", (64, 256), (BF16, F16), (48, 47), 40, 44032, 0),
         ("rows", (32, 128), (F32,), (33, 1, 0, 30), 132, 8196, 0), ("rows", (32, 128), (F32, BF16, F16), (33, 1, 0, 30), 131, 8193, 0),
         ("rows", (32, 128), (F32, BF16, F16), (40, 24), 64, 13000, 1),
         ("rows", (256, 256), (BF16, F16), (356, 40, 0, 204), 200, 13320, 0), ("forward", (256, 256), (BF16, F16), (356, 40, 0, 204), 13320, 200, 0),
         ("rows", (256, 256), (BF16, F16), (65, 384, 128), 136, 16648, 0), ("forward", (256, 256), (BF16, F16), (65, 384, 128), 16648, 136, 0),
         ("matrices", (128, 128), (F32,), (0, 33, 87), 1004, 1396, 0), ("matrices", (128, 128), (F32, BF16, F16), (1, 70, 128), 1001, 1399, 0),
         ("matrices", (128, 128), (F32, BF16, F16), (64, 0, 65), 1008, 1400, 1), ("matrices", (128, 128), (F32,), (300,), 2052, 2064, 0)]


@pytest.mark.parametrize("op,want_tile,dt,counts,rows,cols,shifted",
                         [(op, t, dt, *rest) for op, t, dts, *rest in FORMS for dt in dts])
def test_tiles_of_other_sizes(L, op, want_tile, dt, counts, rows, cols, shifted):
    say("tiles of other sizes", op, want_tile, dt, counts, rows, cols, shifted)
    rng = np.random.default_rng(sum(counts) + rows)
    NE, used, n = len(counts), sum(counts), sum(counts) + 3          # three tokens without an expert
    one = 4 if dt == F32 else 2
    whole = not shifted and cols * one % 16 == 0 and (op == "forward" or rows * one % 16 == 0)
    cus = L.g53h_num_cus()
    if cus == 256:
        assert tile(cus, op, dt, n, NE, rows, cols, whole) == want_tile
    idx = np.concatenate([np.repeat(np.arange(NE), counts), np.full(3, -1)]).astype(np.int32)[:, None]
    rng.shuffle(idx)
    offsets, pair, _ = sorted_plan(idx, NE)
    plan, shift = Plan(idx, NE), one if shifted else 0
    of = lambda e: slice(offsets[e], offsets[e + 1])                 # noqa: E731
    xv = values(rng, (n, cols), dt, True)
    if op == "matrices":
        dv = values(rng, (n, rows), dt, True)
        old = values(rng, (NE, rows, cols), dt, True)
        x, d, dw, da = Buf(xv, dt, shift), Buf(dv, dt, shift), Buf.out((NE, rows, cols), F32), Buf(old, dt, shift)
        check(L.g53h_sorted_mm_grad(None, dw.ptr, F32, 0, d.ptr, x.ptr, dt, 1, plan.c, None, rows, cols))
        check(L.g53h_sorted_mm_grad(None, da.ptr, dt, 1, d.ptr, x.ptr, dt, 1, plan.c, None, rows, cols))
        got, added = dw.val(), da.val()
        for e in range(NE):
            ref = dv[of(e)].T @ xv[pair[of(e)]]
            assert np.array_equal(got[e], ref) and np.array_equal(added[e], rounded(old[e] + ref, dt)), e
        return
    wv = values(rng, (NE, rows, cols), dt, True)
    w = Buf(wv, dt, shift)
    if op == "rows":
        dv = values(rng, (n, rows), dt, True)
        d, dx = Buf(dv, dt, shift), Buf.out((n, cols), dt, shift)
        check(L.g53h_sorted_mm_grad(dx.ptr, None, dt, 0, d.ptr, None, dt, 1, plan.c, w.ptr, rows, cols))
        ref = np.concatenate([dv[of(e)] @ wv[e] for e in range(NE)])
        assert np.array_equal(dx.val()[:used], rounded(ref, dt)) and (dx.val()[used:] == 77).all()
        return
    x, ys, gu, act = Buf(xv, dt, shift), Buf.out((n, rows), dt, shift), Buf.out((n, rows), dt, shift), Buf.out((n, rows // 2), dt, shift)
    check(L.g53h_sorted_mm(ys.ptr, None, x.ptr, dt, 1, plan.c, w.ptr, rows, cols, 0.0))
    check(L.g53h_sorted_mm(act.ptr, gu.ptr, x.ptr, dt, 1, plan.c, w.ptr, rows, cols, LIMIT))
    ref = np.concatenate([xv[pair[of(e)]] @ wv[e].T for e in range(NE)])
    assert np.array_equal(ys.val()[:used], rounded(ref, dt)) and np.array_equal(gu.val(), ys.val())
    assert (ys.val()[used:] == 77).all() and (act.val()[used:] == 77).all()
    with np.errstate(over="ignore"):
        want = swiglu(ref, LIMIT)
    g, u = np.split(ref, 2, 1)
    # as in test_every_tile, and half a step of what the exponential is of, the gate by log2 e
    deep = np.where(g < -87, 2.0 ** -126 * np.abs(g * np.clip(u, -LIMIT, LIMIT)), 0)
    rel = 2.0 ** -20 + np.abs(np.minimum(g, 0)) * 2.0 ** -24
    close(act.val()[:used], want, (rel + HALF[dt]) * np.abs(want) + TINY[dt] + deep)
