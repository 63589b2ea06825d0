"""The experts' own products run together: a MoE block's experts trained (forward, backward, gradients of the tokens, the
routing's weights and the matrices against differences in 64 bits), and the same experts quantised to microscaled 4 bits
and run; and calls as programs make them: many in a row without a wait, on one plan."""
import ctypes as C

import numpy as np
import pytest

import glm53h
from glm53h import check
from op_lib import BF16, F32, HALF, Buf, Plan, close, dec, enc, sorted_plan, swiglu
from test_gpu_mx4 import Mx4, quant, wide
from test_gpu_parity import say

pytestmark = pytest.mark.gpu
LIMIT = 3.0


@pytest.fixture(scope="module")
def L():
    return glm53h.init(0)


def experts(x, w, gu, down, idx):
    """out[t] = sum over j of w down . swiglu(gu . x[t]), in 64 bits."""
    out = np.zeros((x.shape[0], down.shape[1]))
    for t in range(x.shape[0]):
        for j, e in enumerate(idx[t]):
            if e >= 0:
                out[t] += w[t, j] * (down[e] @ swiglu(gu[e] @ x[t], LIMIT))
    return out


def test_training_step(L):
    say("experts' training step")
    rng = np.random.default_rng(8)
    T, H, inter, NE, K = 23, 72, 40, 5, 2
    idx = np.argsort(rng.random((T, NE - 1)), 1)[:, :K].astype(np.int32)          # the last expert has no rows
    idx[T - 2:] = -1
    n = T * K
    plan = Plan(idx, NE)
    f = lambda v: dec(enc(v, F32), F32)                                             # noqa: E731
    xv, wv, gv = f(rng.standard_normal((T, H))), f(rng.uniform(0.2, 1, (T, K))), f(rng.standard_normal((T, H)))
    uv, dv = f(0.3 * rng.standard_normal((NE, 2 * inter, H))), f(0.2 * rng.standard_normal((NE, H, inter)))
    x, w, g, up, down = (Buf(v, F32) for v in (xv, wv, gv, uv, dv))

    def step():
        z = lambda *s: Buf.out(s, F32, fill=0.0)                                    # noqa: E731
        gu, act, ys, out = z(n, 2 * inter), z(n, inter), z(n, H), z(T, H)
        check(L.g53h_sorted_mm(act.ptr, gu.ptr, x.ptr, F32, 1, plan.c, up.ptr, 2 * inter, H, LIMIT))
        check(L.g53h_sorted_mm(ys.ptr, None, act.ptr, F32, 0, plan.c, down.ptr, H, inter, 0.0))
        check(L.g53h_sorted_combine(out.ptr, ys.ptr, w.ptr, None, F32, H, plan.c))
        dys, dw, dact, ddown, dgu, dxs, dup, dx = z(n, H), z(T, K), z(n, inter), z(NE, H, inter), z(n, 2 * inter), z(n, H), z(NE, 2 * inter, H), z(T, H)
        check(L.g53h_sorted_combine_grad(dys.ptr, dw.ptr, g.ptr, ys.ptr, w.ptr, F32, H, plan.c))
        check(L.g53h_sorted_mm_grad(dact.ptr, ddown.ptr, F32, 0, dys.ptr, act.ptr, F32, 0, plan.c, down.ptr, H, inter))
        check(L.g53h_sorted_swiglu_grad(dgu.ptr, dact.ptr, gu.ptr, F32, inter, plan.c, LIMIT))
        check(L.g53h_sorted_mm_grad(dxs.ptr, dup.ptr, F32, 0, dgu.ptr, x.ptr, F32, 1, plan.c, up.ptr, 2 * inter, H))
        check(L.g53h_sorted_dispatch_grad(dx.ptr, dxs.ptr, F32, H, plan.c))
        # the second micro-batch's gradients join the first's
        check(L.g53h_sorted_mm_grad(None, dup.ptr, F32, 1, dgu.ptr, x.ptr, F32, 1, plan.c, None, 2 * inter, H))
        check(L.g53h_sync())
        return [b.get() for b in (out, dx, dw, dup, ddown)]

    first, again = step(), step()
    assert all(np.array_equal(a, b) for a, b in zip(first, again))
    out, dx, dw, dup, ddown = (v.astype(np.float64) for v in first)
    want = experts(xv, wv, uv, dv, idx)
    # sums of 72 and 40 fp32 products, sizes of order 10
    assert np.abs(out - want).max() < 1e-4
    assert not dup[NE - 1].any() and not ddown[NE - 1].any()
    at = [xv, wv, uv, dv]
    loss = lambda *a: (experts(*a, idx) * gv).sum()                                 # noqa: E731
    for i, grad in enumerate((dx, dw, dup / 2, ddown)):
        d, e = rng.standard_normal(at[i].shape), 1e-6
        hi, lo = ([v + s * e * d if k == i else v for k, v in enumerate(at)] for s in (1, -1))
        diff = (loss(*hi) - loss(*lo)) / (2 * e)
        # kinks at the clamps, passed within e, are off by e times their slopes; 64-bit rounding / e; fp32 gradients
        assert abs(diff - (grad * d).sum()) < 2e-4 * (1 + abs(diff)), i


def test_trained_then_served(L):
    """Experts in bf16, quantised by the library, run in 4 bits: the products are those of the quantised values."""
    say("experts quantised and run")
    rng = np.random.default_rng(9)
    T, H, inter, NE, K = 19, 160, 96, 6, 3
    idx = rng.integers(0, NE, (T, K)).astype(np.int32)
    offsets, pair, _ = sorted_plan(idx, NE)
    plan, n = Plan(idx, NE), T * K
    bf = lambda v: dec(enc(v, BF16), BF16)                                          # noqa: E731
    xv, uv, dv = bf(rng.standard_normal((T, H))), bf(0.1 * rng.standard_normal((NE * 2 * inter, H))), bf(0.1 * rng.standard_normal((NE * H, inter)))
    x, up, down = Buf(xv, BF16), Buf(uv, BF16), Buf(dv, BF16)
    new = lambda r, c: (Buf.out((r, c // 2), np.uint8), Buf.out((r, c // 32), np.uint8))        # noqa: E731
    mat = lambda b, r, c: glm53h.G53hMx4(b[0].ptr, b[1].ptr, r, c)                  # noqa: E731
    qx, qu, qd, qa = new(T, H), new(NE * 2 * inter, H), new(NE * H, inter), new(n, inter)
    act, ys = Buf.out((n, inter), BF16, fill=0.0), Buf.out((n, H), BF16)
    check(L.g53h_mx4_quant(mat(qu, NE * 2 * inter, H), up.ptr, BF16))
    check(L.g53h_mx4_quant(mat(qd, NE * H, inter), down.ptr, BF16))
    check(L.g53h_mx4_quant(mat(qx, T, H), x.ptr, BF16))
    check(L.g53h_sorted_mm_mx4(act.ptr, BF16, mat(qx, T, H), 1, plan.c, mat(qu, 2 * inter, H), LIMIT))
    check(L.g53h_mx4_quant(mat(qa, n, inter), act.ptr, BF16))
    check(L.g53h_sorted_mm_mx4(ys.ptr, BF16, mat(qa, n, inter), 0, plan.c, mat(qd, H, inter), 0.0))
    check(L.g53h_sync())
    val = lambda v: wide(*quant(v))                                                 # noqa: E731
    U, D, X = val(uv).reshape(NE, 2 * inter, H), val(dv).reshape(NE, H, inter), val(xv)
    e_of = np.repeat(np.arange(NE), np.diff(offsets))
    a = np.stack([swiglu(U[e] @ X[p // K], LIMIT) for e, p in zip(e_of, pair)])
    got = act.val()
    # sums of exact products; the SwiGLU's slopes and the hardware's exponential; half a step of bf16
    assert (np.abs(got - a) <= (HALF[BF16] + 2.0 ** -18) * np.abs(a) + 1e-5).all()
    A = val(got)
    y = np.stack([D[e] @ A[r] for r, e in enumerate(e_of)])
    size = np.stack([np.abs(D[e]) @ np.abs(A[r]) for r, e in enumerate(e_of)])
    close(ys.val(), y, HALF[BF16] * np.abs(y) + (inter + 32) * 2.0 ** -23 * size)


def test_many_in_a_row(L):
    """Forty calls of changing sizes on one stream without a wait: each like the first of its kind."""
    say("in a row")
    rng = np.random.default_rng(10)
    sets = []
    for T, K, NE, rows, cols, dt in ((3, 2, 4, 130, 64, BF16), (90, 2, 3, 66, 77, BF16), (40, 1, 2, 300, 136, F32), (257, 3, 9, 130, 200, BF16)):
        idx = rng.integers(0, NE, (T, K)).astype(np.int32)
        x, w = Buf(rng.standard_normal((T, cols)), dt), Buf(rng.standard_normal((NE, rows, cols)), dt)
        d = Buf(rng.standard_normal((T * K, rows)), dt)
        sets.append((T, K, NE, rows, cols, dt, Plan(idx, NE), x, w, d))
    first = None
    for _ in range(10):
        outs = []
        for T, K, NE, rows, cols, dt, plan, x, w, d in sets:
            o = [Buf.out((T * K, rows), dt), Buf.out((T * K, cols), dt), Buf.out((NE, rows, cols), F32)]
            check(L.g53h_sorted_mm(o[0].ptr, None, x.ptr, dt, 1, plan.c, w.ptr, rows, cols, 0.0))
            check(L.g53h_sorted_mm_grad(o[1].ptr, o[2].ptr, F32, 0, d.ptr, x.ptr, dt, 1, plan.c, w.ptr, rows, cols))
            outs += o
        got = [b.get() for b in outs]
        first = first or got
        assert all(np.array_equal(a, b) for a, b in zip(first, got))


@pytest.mark.parametrize("what", ["mm", "mx4"])
def test_rows_outside_a_tile_are_not_read(L, what):
    """NaN in rows behind the last sorted one, and in other experts' rows and matrices, reach nothing."""
    say("others' rows", what)
    rng = np.random.default_rng(11)
    T, NE, rows, cols = 37, 3, 70, 96
    idx = np.where(np.arange(T) % 3 == 0, -1, 2).astype(np.int32)[:, None]
    offsets, pair, _ = sorted_plan(idx, NE)
    used, plan = offsets[NE], Plan(idx, NE)
    if what == "mm":
        for dt in (BF16, F32):
            xv, wv = rng.integers(-3, 4, (T, cols)).astype(float), rng.integers(-3, 4, (NE, rows, cols)).astype(float)
            dv = rng.integers(-3, 4, (T, rows)).astype(float)
            want = xv[:used] @ wv[2].T
            dx, dw = dv[:used] @ wv[2], dv[:used].T @ xv[:used]
            xv[used:], wv[:2], dv[used:] = np.nan, np.nan, np.nan
            x, w, d = Buf(xv, dt), Buf(wv, dt), Buf(dv, dt)
            ys, gx, gw = Buf.out((T, rows), dt), Buf.out((T, cols), dt), Buf.out((NE, rows, cols), F32)
            check(L.g53h_sorted_mm(ys.ptr, None, x.ptr, dt, 0, plan.c, w.ptr, rows, cols, 0.0))
            check(L.g53h_sorted_mm_grad(gx.ptr, gw.ptr, F32, 0, d.ptr, x.ptr, dt, 0, plan.c, w.ptr, rows, cols))
            r = lambda v: dec(enc(v, dt), dt)                                       # noqa: E731
            assert np.array_equal(ys.val()[:used], r(want)) and np.array_equal(gx.val()[:used], r(dx))
            assert np.array_equal(gw.val()[2], dw) and not gw.val()[:2].any()
            assert (ys.val()[used:] == 77).all() and (gx.val()[used:] == 77).all()
    else:
        lv = lambda r: rng.integers(0, 16, (r, cols)).astype(np.uint8)              # noqa: E731
        sx, sm = np.full((T, cols // 32), 127, np.uint8), np.full((NE * rows, cols // 32), 126, np.uint8)
        lx, lm = lv(T), lv(NE * rows)
        want = wide(lx[:used], sx[:used]) @ wide(lm[2 * rows:], sm[2 * rows:]).T
        sx[used:], sm[:2 * rows] = 255, 255
        x, m, ys = Mx4(lx, sx, T), Mx4(lm, sm, rows), Buf.out((T, rows), F32)
        check(L.g53h_sorted_mm_mx4(ys.ptr, F32, C.byref(x.c), 0, plan.c, C.byref(m.c), 0.0))
        assert np.array_equal(ys.val()[:used], want) and (ys.val()[used:] == 77).all()
