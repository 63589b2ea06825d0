"""The operators beside the layer run together, as a trunk runs a MoE block with 4-bit experts: norm,
router, sort, the experts' products over the sorted rows, the weighted sum with a shared expert's output,
and the norm after the block with its gate and residual; and a training step's gradients through all
but the products. All on the library's stream with one wait at the end, against 64 bits on the host."""
import ctypes as C

import numpy as np
import pytest

import glm53h
import glm53h.synth as S
from glm53h import DevBuf, check
from op_lib import BF16, F16, F32, HALF, W4, Buf, Plan, block, dec, enc, sorted_plan, swiglu
from test_gpu_grouped import run
from test_gpu_parity import say

pytestmark = pytest.mark.gpu
LIMIT, SCALE, EPS = 10.0, 0.5, 1e-6


@pytest.fixture(scope="module")
def L():
    return glm53h.init(0)


@pytest.mark.parametrize("T,H,inter,NE,K,dt", [(1, 256, 128, 16, 4, BF16), (7, 96, 64, 5, 2, F32), (70, 512, 160, 24, 3, F16),
                                               (33, 160, 96, 300, 6, BF16)])
def test_moe_block(L, T, H, inter, NE, K, dt):
    say("block", T, H, inter, NE, K, dt)
    rng = np.random.default_rng(H)
    h = Buf(rng.standard_normal((T, H)), dt)
    shared = Buf(0.1 * rng.standard_normal((T, H)), dt)
    gain, post, nxt = (Buf(rng.uniform(0.5, 1.5, H), F32) for _ in range(3))
    gate = Buf(rng.uniform(0.1, 1.0, H), F32)
    router, bias = Buf(rng.standard_normal((NE, H)) / np.sqrt(H), F32), Buf(0.1 * rng.standard_normal(NE), F32)
    up, down = W4(rng, NE, 2 * inter, H, 32, BF16, True), W4(rng, NE, H, inter, 32, F32, False)
    xn = Buf.out((T, H), dt)
    idx, w, flag = Buf.out((T, K), np.int32), Buf.out((T, K), F32), Buf.out(1, np.int32)
    plan = Plan(np.zeros((T, K), np.int32), NE, given=True)
    act, ys, out = Buf.out((T * K, inter), dt), Buf.out((T * K, H), dt), Buf.out((T, H), dt)
    h2, xn2 = Buf.out((T, H), dt), Buf.out((T, H), dt)
    b = glm53h.G53hBlockNorm(T, H, dt, 1, EPS, SCALE, post.ptr, nxt.ptr, gate.ptr)

    check(L.g53h_norm(xn.ptr, h.ptr, gain.ptr, dt, T, H, EPS), "norm")
    xf = xn if dt == F32 else Buf(xn.val(), F32)        # the router takes fp32
    check(L.g53h_router(idx.ptr, w.ptr, xf.ptr, T, router.ptr, 0, bias.ptr, NE, H, K, 1, 2.5, flag.ptr), "router")
    check(L.g53h_sort_tokens(plan.c, idx.ptr), "sort")
    check(L.g53h_sorted_mm_w4(act.ptr, xn.ptr, dt, 1, plan.c, C.byref(up.c), LIMIT), "gate and up")
    check(L.g53h_sorted_mm_w4(ys.ptr, act.ptr, dt, 0, plan.c, C.byref(down.c), 0.0), "down")
    check(L.g53h_sorted_combine(out.ptr, ys.ptr, w.ptr, shared.ptr, dt, H, plan.c), "combine")
    check(L.g53h_block_norm(h2.ptr, xn2.ptr, h.ptr, out.ptr, b), "block_norm")
    check(L.g53h_sync(), "sync")

    iv, wv, x = idx.get(), w.val(), xn.val()
    hv = h.val()
    want = hv / np.sqrt((hv * hv).mean(1, keepdims=True) + EPS) * gain.val()
    assert np.linalg.norm(x - want) <= 2 * (HALF[dt] + 1e-6) * np.linalg.norm(want)
    y, size = shared.val(), np.abs(shared.val())
    for t in range(T):
        for j in range(K):
            a, m = swiglu(x[t] @ up.wide[iv[t, j]].T, LIMIT), down.wide[iv[t, j]]
            y[t], size[t] = y[t] + wv[t, j] * (m @ a), size[t] + wv[t, j] * (np.abs(m) @ np.abs(a))
    # three roundings to the type on the way (act, ys, out), each at most half a step of what is summed; fp32 sums far less
    assert (np.abs(out.val() - y) <= (3 * HALF[dt] + 1e-5) * size).all()
    w2, wn = block(hv, out.val(), post.val(), nxt.val(), gate.val(), 1, SCALE, EPS)
    for got, ref in ((h2, w2), (xn2, wn)):
        assert np.linalg.norm(got.val() - ref) <= (HALF[dt] + 1e-5) * np.linalg.norm(ref)


def test_training_step(L):
    """Forward and backward of out = h + s gate norm(combine(expert rows of dispatch(norm(h)))) with the identity for the
    experts, in fp32, twice: the gradients of h and the weights against differences in 64 bits, and the same bits again."""
    say("training step")
    rng = np.random.default_rng(2)
    T, H, NE, K = 11, 72, 5, 2
    idx = rng.integers(0, NE, (T, K)).astype(np.int32)
    plan = Plan(idx, NE)
    hv, wv, gv = (dec(enc(v, F32), F32) for v in (rng.standard_normal((T, H)), rng.uniform(0.2, 1, (T, K)), rng.standard_normal((T, H))))
    h, w, g = Buf(hv, F32), Buf(wv, F32), Buf(gv, F32)
    gain, post, gate = (Buf(rng.uniform(0.5, 1.5, H), F32) for _ in range(3))
    b = glm53h.G53hBlockNorm(T, H, F32, 1, EPS, SCALE, post.ptr, None, gate.ptr)

    def step():
        n = lambda *s: Buf.out(s, F32)                                                  # noqa: E731
        xn, xs, y, h2 = n(T, H), n(T * K, H), n(T, H), n(T, H)
        check(L.g53h_norm(xn.ptr, h.ptr, gain.ptr, F32, T, H, EPS), "norm")
        check(L.g53h_sorted_dispatch(xs.ptr, xn.ptr, F32, H, plan.c), "dispatch")
        check(L.g53h_sorted_combine(y.ptr, xs.ptr, w.ptr, None, F32, H, plan.c), "combine")
        check(L.g53h_block_norm(h2.ptr, None, h.ptr, y.ptr, b), "block_norm")
        dh, dy, dgate, dpost, dxs, dw, dxn, dx, dgain = n(T, H), n(T, H), n(H), n(H), n(T * K, H), n(T, K), n(T, H), n(T, H), n(H)
        check(L.g53h_block_norm_grad(dh.ptr, dy.ptr, dgate.ptr, dpost.ptr, None, g.ptr, None, h.ptr, y.ptr, b), "block_norm_grad")
        check(L.g53h_sorted_combine_grad(dxs.ptr, dw.ptr, dy.ptr, xs.ptr, w.ptr, F32, H, plan.c), "combine_grad")
        check(L.g53h_sorted_dispatch_grad(dxn.ptr, dxs.ptr, F32, H, plan.c), "dispatch_grad")
        check(L.g53h_norm_grad(dx.ptr, dgain.ptr, dxn.ptr, h.ptr, gain.ptr, F32, T, H, EPS), "norm_grad")
        check(L.g53h_sync(), "sync")
        return [v.get() for v in (h2, dh, dx, dw, dgain, dpost, dgate)]

    def loss(h, w, gain, post, gate):
        x = h / np.sqrt((h * h).mean(1, keepdims=True) + EPS) * gain
        y = x * w.sum(1, keepdims=True)
        return (block(h, y, post, None, gate, 1, SCALE, EPS)[0] * gv).sum()

    first, again = step(), step()
    assert all(np.array_equal(a, b) for a, b in zip(first, again))
    _, dh, dx, dw, dgain, dpost, dgate = (v.astype(np.float64) for v in first)
    at = [hv, wv, gain.val(), post.val(), gate.val()]
    for i, grad in enumerate((dh + dx, dw, dgain, dpost, dgate)):
        d = rng.standard_normal(at[i].shape)
        e = 1e-5
        up, down = ([v + s * e * d if k == i else v for k, v in enumerate(at)] for s in (1, -1))
        diff = (loss(*up) - loss(*down)) / (2 * e)
        # e^2 of third derivatives of order one, 64-bit rounding / e, and fp32 gradients of some 800 terms
        assert abs(diff - (grad * d).sum()) < 1e-4 * (1 + abs(diff)), i


def test_between_the_phases_of_a_grouped_layer(L):
    """The operators have a workspace of their own: a grouped layer that is begun, with them in between, ends as without."""
    say("operators inside a grouped pass")
    sp = S.LayerSpec(E=512, I=512, NE=8, K=4, router_sigma=0.02)
    T = 700
    layer = S.DeviceLayer.build(sp)
    x = S.x_host(sp, T, batch=6)
    want, wi, ww = run(layer, x, 1, "g53h_moe_grouped")
    assert T <= L.g53h_grouped_max_tokens(C.byref(layer.layer))
    rng = np.random.default_rng(7)
    xd, od, id_, wd = DevBuf.from_array(x), DevBuf(x.nbytes), DevBuf.from_array(wi), DevBuf.from_array(ww)
    h, d, g = (Buf(rng.standard_normal(s), F32) for s in ((T, 512), (T, 512), (512,)))
    dx, dg = Buf.out((T, 512), F32), Buf.out(512, F32)

    def others():
        plan = Plan(np.repeat(wi, 8, 0), sp.NE)              # 22400 pairs: segments, whose counts lie in a workspace
        check(L.g53h_norm_grad(dx.ptr, dg.ptr, d.ptr, h.ptr, g.ptr, F32, T, 512, EPS), "norm_grad")
        return plan

    check(L.g53h_grouped_begin(xd.ptr, T, C.byref(layer.layer), id_.ptr), "begin")
    first = others()
    check(L.g53h_grouped_batch(C.byref(layer.layer)), "batch")
    second = others()
    check(L.g53h_grouped_end(od.ptr, wd.ptr), "end")
    assert L.g53h_grouped_errors() == 0
    assert np.array_equal(od.download(np.uint32).reshape(x.shape), want.view(np.uint32))
    for plan in (first, second):
        assert all(np.array_equal(a, b) for a, b in zip(plan.arrays(), sorted_plan(np.repeat(wi, 8, 0), sp.NE)))
