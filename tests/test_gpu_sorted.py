"""Tokens sorted by expert and back (g53h_sort_tokens, g53h_sorted_dispatch, g53h_sorted_combine and
their gradients) against a stable sort and sums in 64 bits on the host.

Tolerances: a copy is exact. A sum of k products in fp32 is off by at most k 2^-24 of the sum of the
products' sizes (one rounding each, fused), and a result by half a step of its type more."""
import numpy as np
import pytest

import glm53h
from glm53h import check
from op_lib import BF16, F16, F32, HALF, TINY, Buf, Plan, close, dec, enc, routing, sorted_plan
from test_gpu_parity import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    return glm53h.init(0)


@pytest.mark.parametrize("T,K,NE", [(1, 8, 288), (1, 1, 1), (1, 64, 1024), (5, 3, 7), (64, 1, 2), (65, 8, 288), (127, 8, 16),
                                    (129, 8, 1024), (1024, 1, 63), (1025, 1, 64), (1024, 8, 65), (1025, 8, 288),
                                    (4096, 8, 288), (9000, 3, 1000), (40000, 8, 129), (140000, 8, 300)])
@pytest.mark.parametrize("drop", [0.0, 0.3])
def test_sort(L, T, K, NE, drop):
    say("sort", T, K, NE, drop)
    rng = np.random.default_rng(T * 31 + K + NE)
    idx = routing(rng, T, K, NE, drop)
    got = Plan(idx, NE).arrays()
    for g, w, name in zip(got, sorted_plan(idx, NE), ("offsets", "pair", "row")):
        assert np.array_equal(g, w), name


@pytest.mark.parametrize("T,K,NE,fill", [(300, 4, 288, 17), (2000, 8, 5, 4), (20000, 4, 288, 0), (300, 4, 9, -1),
                                         (20000, 4, 9, 9), (10, 4, 9, -2147483648), (10, 4, 9, 2147483647)])
def test_sort_one_expert_or_none(L, T, K, NE, fill):
    say("sort, all", fill, T, K, NE)
    idx = np.full((T, K), fill, np.int32)
    for g, w in zip(Plan(idx, NE).arrays(), sorted_plan(idx, NE)):
        assert np.array_equal(g, w)


@pytest.mark.parametrize("n", [63, 64, 65, 1023, 1024, 1025, 2048, 2049])
@pytest.mark.parametrize("NE", [1, 255, 256, 1024])
def test_sort_at_the_edges_of_its_kernels(L, n, NE):
    say("sort, edges", n, NE)
    rng = np.random.default_rng(n + NE)
    idx = routing(rng, n, 1, NE, 0.2)
    idx[-1] = NE - 1                                      # the last pair is there, and one just past the experts is not
    idx[0] = NE
    for g, w in zip(Plan(idx, NE).arrays(), sorted_plan(idx, NE)):
        assert np.array_equal(g, w)


def test_sort_no_tokens(L):
    say("sort, no tokens")
    off = Buf(np.full(10, -7, np.int32))
    check(L.g53h_sort_tokens(glm53h.G53hSort(0, 4, 9, off.ptr, None, None), None), "sort")
    assert (off.get() == 0).all()
    p = glm53h.G53hSort(0, 4, 9, off.ptr, None, None)
    assert L.g53h_sorted_dispatch(None, None, 0, 8, p) == 0 and L.g53h_sorted_combine(None, None, None, None, 0, 8, p) == 0
    assert L.g53h_sorted_combine_grad(None, None, None, None, None, 0, 8, p) == 0


SHAPES = [(1, 8, 288, 4096, 0.0, 0), (1, 1, 1, 1, 0.0, 0), (7, 3, 5, 9, 0.3, 0), (33, 8, 16, 1023, 0.1, 0),
          (12, 9, 40, 2049, 0.2, 2), (5, 64, 64, 100, 0.5, 4), (70, 2, 288, 4104, 0.0, 6), (9, 4, 6, 8191, 1.0, 0)]


@pytest.mark.parametrize("T,K,NE,H,drop,shift", SHAPES)
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_dispatch_and_its_gradient(L, T, K, NE, H, drop, shift, dt):
    say("dispatch", T, K, NE, H, drop, dt)
    shift = shift // 4 * 4 if dt == F32 else shift
    rng = np.random.default_rng(H + K)
    idx = routing(rng, T, K, NE, drop)
    plan, (off, pair, row) = Plan(idx, NE, given=True), sorted_plan(idx, NE)
    n = off[NE]
    x = Buf(rng.standard_normal((T, H)), dt, shift)
    xs = Buf.out((T * K, H), dt, shift)
    check(L.g53h_sorted_dispatch(xs.ptr, x.ptr, dt, H, plan.c), "dispatch")
    got = xs.get()
    assert np.array_equal(got[:n], x.get()[pair[:n] // K]) and (got[n:] == enc([77.0], dt)).all()
    dxs = Buf(rng.standard_normal((T * K, H)), dt, shift)
    dx = Buf.out((T, H), dt, shift)
    check(L.g53h_sorted_dispatch_grad(dx.ptr, dxs.ptr, dt, H, plan.c), "dispatch_grad")
    part = np.where(row.reshape(T, K, 1) >= 0, dxs.val()[row.reshape(T, K)], 0.0)
    want = part.sum(1)
    close(dx.val(), want, HALF[dt] * np.abs(want) + TINY[dt] + K * 2.0 ** -24 * np.abs(part).sum(1))


@pytest.mark.parametrize("T,K,NE,H,drop,shift", SHAPES)
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("add", [False, True])
def test_combine_and_its_gradient(L, T, K, NE, H, drop, shift, dt, add):
    say("combine", T, K, NE, H, drop, dt, add)
    shift = shift // 4 * 4 if dt == F32 else shift
    rng = np.random.default_rng(H * 3 + K)
    idx = routing(rng, T, K, NE, drop)
    plan, (off, pair, row) = Plan(idx, NE, given=True), sorted_plan(idx, NE)
    n, rows = off[NE], row.reshape(T, K)
    keep = rows >= 0
    ys_v = rng.standard_normal((T * K, H))
    ys_v[n:] = np.nan                                     # rows behind the last, and weights of pairs left out, are not read
    w_v = rng.uniform(-1, 2, (T, K)).astype(np.float32)
    w_v[~keep] = np.inf
    ys, w = Buf(ys_v, dt, shift), Buf(w_v)
    out = Buf(rng.standard_normal((T, H)), dt, shift) if add else Buf.out((T, H), dt, shift)
    a = out.val() if add else np.zeros((T, H))            # added in place
    check(L.g53h_sorted_combine(out.ptr, ys.ptr, w.ptr, out.ptr if add else None, dt, H, plan.c), "combine")
    y = np.where(keep[..., None], ys.val()[rows], 0.0)
    wv = np.where(keep, w_v, 0.0).astype(np.float64)
    want, size = a + (wv[..., None] * y).sum(1), np.abs(a) + (np.abs(wv)[..., None] * np.abs(y)).sum(1)
    close(out.val(), want, HALF[dt] * np.abs(want) + TINY[dt] + (K + 1) * 2.0 ** -24 * size, "out")

    dout, dw = Buf(rng.standard_normal((T, H)), dt, shift), Buf.out((T, K), F32)
    dys = Buf.out((T * K, H), dt, shift)
    check(L.g53h_sorted_combine_grad(dys.ptr, dw.ptr, dout.ptr, ys.ptr, w.ptr, dt, H, plan.c), "combine_grad")
    g = dout.val()
    got, want = dys.val(), wv.reshape(-1)[pair[:n]][:, None] * g[pair[:n] // K]
    close(got[:n], want, (HALF[dt] + 2.0 ** -24) * np.abs(want) + TINY[dt], "dys")
    assert (dys.get()[n:] == enc([77.0], dt)).all()
    depth = H // 512 + 12                                 # a lane's chain, 8 chains, 64 lanes
    close(dw.val(), np.where(keep, np.einsum("th,tkh->tk", g, y), 0.0),
          np.where(keep, depth * 2.0 ** -24 * np.einsum("th,tkh->tk", np.abs(g), np.abs(y)), 0.0), "dw")
    into = Buf(ys_v, dt, shift)                           # in place: the gradient over the rows
    dw2 = Buf.out((T, K), F32)
    check(L.g53h_sorted_combine_grad(into.ptr, dw2.ptr, dout.ptr, into.ptr, w.ptr, dt, H, plan.c), "combine_grad in place")
    assert np.array_equal(into.get()[:n], dys.get()[:n]) and np.array_equal(dw2.get(), dw.get())


def test_gradients_are_differences(L):
    """The gradients against differences of the product of the outputs with a fixed tensor, in 64 bits."""
    say("sorted, differences")
    rng = np.random.default_rng(5)
    T, K, NE, H = 6, 3, 4, 21
    idx = routing(rng, T, K, NE, 0.2)
    plan, (off, pair, row) = Plan(idx, NE, given=True), sorted_plan(idx, NE)
    rows = row.reshape(T, K)
    keep = rows >= 0
    x, ys, w, g, gs = (rng.standard_normal(s) for s in ((T, H), (T * K, H), (T, K), (T, H), (T * K, H)))
    x, ys, w, g, gs = (dec(enc(v, F32), F32) for v in (x, ys, w, g, gs))

    def loss(x, ys, w):
        out = np.where(keep[..., None], ys[rows] * w[..., None], 0.0).sum(1)
        return (out * g).sum() + (x[pair[:off[NE]] // K] * gs[:off[NE]]).sum()

    dys, dw, dx = Buf(np.zeros((T * K, H)), F32), Buf.out((T, K), F32), Buf.out((T, H), F32)
    wb, gb, gsb, yb = Buf(w, F32), Buf(g, F32), Buf(gs, F32), Buf(ys, F32)
    check(L.g53h_sorted_combine_grad(dys.ptr, dw.ptr, gb.ptr, yb.ptr, wb.ptr, F32, H, plan.c), "combine_grad")
    check(L.g53h_sorted_dispatch_grad(dx.ptr, gsb.ptr, F32, H, plan.c), "dispatch_grad")
    for _ in range(4):
        d = [rng.standard_normal(v.shape) for v in (x, ys, w)]
        e = 1e-4
        diff = (loss(x + e * d[0], ys + e * d[1], w + e * d[2]) - loss(x - e * d[0], ys - e * d[1], w - e * d[2])) / (2 * e)
        mine = (dx.val() * d[0]).sum() + (dys.val() * d[1]).sum() + (dw.val() * d[2]).sum()
        # the loss has degree 2: a central difference is exact; fp32 gradients, 600 terms
        assert abs(diff - mine) < 1e-5 * (1 + abs(diff))


def test_sum_order_and_weights_are_exact(L):
    """Whole numbers and powers of two: every sum fits 24 bits, so results are exact in any type that holds them."""
    say("combine, exact")
    rng = np.random.default_rng(6)
    T, K, NE, H = 50, 8, 12, 777
    idx = routing(rng, T, K, NE, 0.1)
    plan, (_, _, row) = Plan(idx, NE, given=True), sorted_plan(idx, NE)
    rows = row.reshape(T, K)
    ys, w = rng.integers(-9, 10, (T * K, H)).astype(float), 2.0 ** rng.integers(-1, 2, (T, K))
    y, wb, out = Buf(ys, BF16), Buf(w, F32), Buf.out((T, H), F16)
    check(L.g53h_sorted_combine(out.ptr, Buf(ys, F16).ptr, wb.ptr, None, F16, H, plan.c), "combine")
    want = np.where(rows[..., None] >= 0, ys[rows] * w[..., None], 0.0).sum(1)
    assert np.array_equal(out.val(), want)
    out2 = Buf.out((T, H), BF16)
    check(L.g53h_sorted_combine(out2.ptr, y.ptr, wb.ptr, None, BF16, H, plan.c), "combine")
    assert np.array_equal(out2.get(), enc(want, BF16))
