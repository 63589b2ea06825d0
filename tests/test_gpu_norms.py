"""The norms before and after a block (g53h_norm, g53h_block_norm) and their gradients against the
formulas in 64 bits, and the gradients against differences.

Tolerances: a row's sum of squares is a lane's chain of at most 32 fused additions, then 6 steps over the
lanes and 16 over the waves; with eps, division, square root and reciprocal 1 / sqrt(..) is off by at most
S = 40 roundings (2^-24) relative. Every further factor adds one."""
import numpy as np
import pytest

import glm53h
from glm53h import check
from op_lib import BF16, F16, F32, HALF, TINY, Buf, block, close
from test_gpu_parity import say

pytestmark = pytest.mark.gpu
R = 2.0 ** -24
S = 40 * R
WIDTHS = [1, 7, 8, 64, 511, 512, 513, 1000, 1024, 1030, 2048, 2055, 4096, 4104, 8191, 8192, 8200, 16384]


@pytest.fixture(scope="module")
def L():
    return glm53h.init(0)


def gate_of(rng, kind, T, H, dt):
    g = rng.uniform(0.1, 1.0, {0: 1, 1: H, 2: T, 3: (T, H)}[kind])
    return Buf(g, dt if kind == 3 else F32)


def setup(rng, T, H, dt, kind, post=True, scale=0.5, eps=1e-6, shift=0):
    h, y = Buf(rng.standard_normal((T, H)), dt, shift), Buf(0.7 * rng.standard_normal((T, H)), dt, shift)
    pb, nb = (Buf(rng.uniform(0.5, 1.5, H), F32) for _ in range(2))
    gb = gate_of(rng, kind, T, H, dt)
    c = glm53h.G53hBlockNorm(T, H, dt, kind, eps, scale, pb.ptr if post else None, nb.ptr, gb.ptr if kind else None)
    return h, y, pb, nb, gb, c


def forward_tol(h, y, pv, nv, gv, kind, scale, eps):
    h2, xn = block(h, y, pv, nv, gv, kind, scale, eps)
    t2 = (S + 5 * R) * np.abs(h2 - h) + R * np.abs(h2)               # of the fp32 h2
    rs = 1.0 / np.sqrt((h2 * h2).mean(1, keepdims=True) + eps)
    # an error t2 of h2 moves xn by next rs t2 itself, and rs by at most its root mean square times rs
    move = rs * (t2 + np.abs(h2) * rs * np.sqrt((t2 * t2).mean(1, keepdims=True)))
    return h2, xn, t2, np.abs(nv) * move + (S + 3 * R) * np.abs(xn)


@pytest.mark.parametrize("H", WIDTHS)
@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_norm(L, H, T, dt):
    say("norm", H, T, dt)
    rng = np.random.default_rng(H + T)
    x, g = Buf(rng.standard_normal((T, H)), dt), Buf(rng.uniform(0.5, 1.5, H), F32)
    o = Buf.out((T, H), dt)
    check(L.g53h_norm(o.ptr, x.ptr, g.ptr, dt, T, H, 1e-5), "norm")
    v = x.val()
    want = v / np.sqrt((v * v).mean(1, keepdims=True) + np.float32(1e-5)) * g.val()
    close(o.val(), want, (HALF[dt] + S + 2 * R) * np.abs(want) + TINY[dt])
    check(L.g53h_norm(x.ptr, x.ptr, g.ptr, dt, T, H, 1e-5), "norm in place")
    assert np.array_equal(x.get(), o.get())


@pytest.mark.parametrize("H", [1, 9, 512, 1000, 2049, 4096, 8191, 12000])
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("post", [True, False])
def test_block_norm(L, H, kind, dt, post):
    say("block norm", H, kind, dt, post)
    rng = np.random.default_rng(H * 5 + kind)
    T, shift = 6, 4 if H % 2 else 0
    h, y, pb, nb, gb, c = setup(rng, T, H, dt, kind, post, shift=shift)
    h2, xn = Buf.out((T, H), dt, shift), Buf.out((T, H), dt, shift)
    check(L.g53h_block_norm(h2.ptr, xn.ptr, h.ptr, y.ptr, c), "block_norm")
    w2, wn, t2, tn = forward_tol(h.val(), y.val(), pb.val() if post else None, nb.val(), gb.val(), kind, 0.5, c.eps)
    close(h2.val(), w2, HALF[dt] * np.abs(w2) + TINY[dt] + t2, "h2")
    close(xn.val(), wn, HALF[dt] * np.abs(wn) + TINY[dt] + tn, "xn")
    only = Buf.out((T, H), dt, shift)
    check(L.g53h_block_norm(only.ptr, None, h.ptr, y.ptr, c), "block_norm without xn")
    assert np.array_equal(only.get(), h2.get())
    check(L.g53h_block_norm(h.ptr, xn.ptr, h.ptr, y.ptr, c), "block_norm in place")
    assert np.array_equal(h.get(), h2.get())


def grads(h, y, pv, nv, gv, kind, scale, eps, dh2, dxn):
    """Gradients by the formulas in 64 bits: dh, dy, dgate (before its sum), dpost and dnext (before theirs)."""
    ry = 1.0 if pv is None else 1.0 / np.sqrt((y * y).mean(1, keepdims=True) + eps)
    yh, p = y * ry, 1.0 if pv is None else pv
    g = 1.0 if kind == 0 else gv[:, None] if kind == 2 else gv
    h2 = h + scale * g * yh * p
    rh = 1.0 / np.sqrt((h2 * h2).mean(1, keepdims=True) + eps)
    hh, v = h2 * rh, dxn * nv
    dh = dh2 + rh * (v - hh * (v * hh).mean(1, keepdims=True))
    du = scale * g * dh
    dv = du * p
    dy = dv if pv is None else ry * (dv - yh * (dv * yh).mean(1, keepdims=True))
    # sizes: what each is a sum of, for the tolerances. h2 = h + r is off by (S + 5 R) |r| + R |h2|, however small the
    # two leave h2: so hh = h2 rh is off by that times rh, at most S + 5 R of rh |r| + |hh|, and counts as that
    hb = np.abs(hh) + rh * np.abs(h2 - h)
    sh = np.abs(dh2) + rh * (np.abs(v) + hb * np.abs(v * hb).mean(1, keepdims=True))
    sv = np.abs(scale * g * p) * sh
    sy = sv if pv is None else ry * (sv + np.abs(yh) * (sv * np.abs(yh)).mean(1, keepdims=True))
    return dict(dh=(dh, sh), dy=(dy, sy), dgate=(scale * yh * p * dh, np.abs(scale * yh * p) * sh),
                dpost=(du * yh, np.abs(scale * g * yh) * sh), dnext=(dxn * hh, np.abs(dxn) * hb))


@pytest.mark.parametrize("T,H", [(1, 1), (3, 9), (300, 100), (7, 512), (1030, 520), (5, 1000), (270, 2048), (9, 4096), (600, 4095),
                                 (3, 8192), (2, 12000), (4, 16384)])
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("post,which", [(True, "both"), (False, "both"), (True, "dh2"), (True, "dxn")])
def test_block_norm_grad(L, T, H, kind, dt, post, which):
    if (T > 100 or H > 5000) and not (post and which == "both"):
        pytest.skip("the smaller sizes cover these")
    say("block norm grad", T, H, kind, dt, post, which)
    rng = np.random.default_rng(H + T + kind)
    shift = 4 if H % 2 else 0
    h, y, pb, nb, gb, c = setup(rng, T, H, dt, kind, post, shift=shift)
    dh2, dxn = Buf(rng.standard_normal((T, H)), dt, shift), Buf(rng.standard_normal((T, H)), dt, shift)
    dh, dy, dpost, dnext = Buf.out((T, H), dt, shift), Buf.out((T, H), dt, shift), Buf.out(H, F32), Buf.out(H, F32)
    dgate = Buf.out(gb.shape, gb.dt)
    a, b = dh2.ptr if which != "dxn" else None, dxn.ptr if which != "dh2" else None
    check(L.g53h_block_norm_grad(dh.ptr, dy.ptr, dgate.ptr, dpost.ptr, dnext.ptr, a, b, h.ptr, y.ptr, c), "grad")
    want = grads(h.val(), y.val(), pb.val() if post else None, nb.val(), gb.val(), kind, 0.5, c.eps,
                 dh2.val() if a else np.zeros((T, H)), dxn.val() if b else np.zeros((T, H)))
    # both reciprocal roots, the means (each a sum like a row's squares) and some twenty factors: 4 S relative to the sizes;
    # h2's own error moves rs and h2 / rms by the same share
    tol = 4 * S
    for name, buf in (("dh", dh), ("dy", dy)):
        w, s = want[name]
        close(buf.val(), w, HALF[dt] * np.abs(w) + TINY[dt] + tol * s, name)
    n = T / 256 + 40                                                  # additions over the tokens
    for name, buf in (("dpost", dpost), ("dnext", dnext)):
        w, s = want[name]
        if name == "dpost" and not post:
            continue
        close(buf.val(), w.sum(0), (tol + n * R) * s.sum(0) + TINY[F32], name)
    if kind:
        w, s = want["dgate"]
        ax = {1: 0, 2: 1}.get(kind)
        w, s = (w, s) if ax is None else (w.sum(ax), s.sum(ax))
        close(dgate.val(), w, (HALF[dt] * np.abs(w) + TINY[dt] if kind == 3 else 0) + (tol + (n + 32) * R) * s + TINY[F32], "dgate")
    first = [v.get() for v in (dh, dy, dpost, dnext, dgate)]
    check(L.g53h_block_norm_grad(dh2.ptr if a else dh.ptr, dy.ptr, dgate.ptr, dpost.ptr, dnext.ptr, a, b, h.ptr, y.ptr, c),
          "grad in place")
    assert np.array_equal((dh2 if a else dh).get(), first[0])
    assert all(np.array_equal(v.get(), f) for v, f in zip((dy, dpost, dnext, dgate), first[1:])), "another run, other bits"


@pytest.mark.parametrize("T,H", [(1, 1), (5, 100), (700, 1024), (3, 4097), (2, 16384)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_norm_grad(L, T, H, dt):
    say("norm grad", T, H, dt)
    rng = np.random.default_rng(H)
    x, dxn, g = Buf(rng.standard_normal((T, H)), dt), Buf(rng.standard_normal((T, H)), dt), Buf(rng.uniform(0.5, 1.5, H), F32)
    dx, dg = Buf.out((T, H), dt), Buf.out(H, F32)
    check(L.g53h_norm_grad(dx.ptr, dg.ptr, dxn.ptr, x.ptr, g.ptr, dt, T, H, 1e-6), "norm_grad")
    v, d = x.val(), dxn.val()
    rs = 1.0 / np.sqrt((v * v).mean(1, keepdims=True) + np.float32(1e-6))
    vh, w = v * rs, d * g.val()
    want, size = rs * (w - vh * (w * vh).mean(1, keepdims=True)), rs * (np.abs(w) + np.abs(vh) * np.abs(w * vh).mean(1, keepdims=True))
    close(dx.val(), want, HALF[dt] * np.abs(want) + TINY[dt] + 4 * S * size, "dx")
    close(dg.val(), (d * vh).sum(0), (4 * S + (T / 256 + 40) * R) * np.abs(d * vh).sum(0), "dgain")
    check(L.g53h_norm_grad(dxn.ptr, None, dxn.ptr, x.ptr, g.ptr, dt, T, H, 1e-6), "in place, without dgain")
    assert np.array_equal(dxn.get(), dx.get())


@pytest.mark.parametrize("kind", [0, 1, 2, 3])
def test_gradients_are_differences(L, kind):
    say("norm grad, differences", kind)
    rng = np.random.default_rng(3)
    T, H, eps, scale = 4, 50, 1e-6, 0.5
    h, y, pb, nb, gb, c = setup(rng, T, H, F32, kind)
    dh2, dxn = Buf(rng.standard_normal((T, H)), F32), Buf(rng.standard_normal((T, H)), F32)
    outs = [Buf.out((T, H), F32), Buf.out((T, H), F32), Buf.out(gb.shape, F32), Buf.out(H, F32), Buf.out(H, F32)]
    check(L.g53h_block_norm_grad(*[o.ptr for o in outs], dh2.ptr, dxn.ptr, h.ptr, y.ptr, c), "grad")
    at = [h.val(), y.val(), gb.val(), pb.val(), nb.val()]

    def loss(h, y, g, p, n):
        h2, xn = block(h, y, p, n, g, kind, scale, eps)
        return (h2 * dh2.val()).sum() + (xn * dxn.val()).sum()

    for i in range(5):
        if i == 2 and kind == 0:
            continue
        d = rng.standard_normal(at[i].shape)
        e = 1e-5
        up, down = ([v + s * e * d if k == i else v for k, v in enumerate(at)] for s in (1, -1))
        diff = (loss(*up) - loss(*down)) / (2 * e)
        # third derivatives of order one: e^2 = 1e-10 of the value; 64-bit rounding / e about 1e-10; fp32 gradients 1e-5
        assert abs(diff - (outs[i].val() * d).sum()) < 1e-4 * (1 + abs(diff)), i


def test_zero_rows_and_no_tokens(L):
    say("norm, zero rows")
    z, g = Buf(np.zeros((3, 100)), BF16), Buf(np.ones(100), F32)
    o = Buf.out((3, 100), BF16)
    check(L.g53h_norm(o.ptr, z.ptr, g.ptr, BF16, 3, 100, 1e-6), "norm")
    assert (o.get() == 0).all()
    assert L.g53h_norm(None, None, None, BF16, 0, 100, 1e-6) == 0
    dg = Buf.out(100, F32)
    check(L.g53h_norm_grad(None, dg.ptr, None, None, None, BF16, 0, 100, 1e-6), "norm_grad of no tokens")
    assert (dg.get() == 0).all()
    d = [Buf.out(100, F32) for _ in range(3)]
    c = glm53h.G53hBlockNorm(0, 100, BF16, 1, 1e-6, 1.0, g.ptr, g.ptr, g.ptr)
    check(L.g53h_block_norm_grad(None, None, *[b.ptr for b in d], None, None, None, None, c), "block_norm_grad of no tokens")
    assert all((b.get() == 0).all() for b in d)


def test_a_row_that_is_not_finite_stays_alone(L):
    say("norm, not finite")
    rng = np.random.default_rng(4)
    h, y, pb, nb, gb, c = setup(rng, 6, 300, F32, 1)
    a, b = Buf.out((6, 300), F32), Buf.out((6, 300), F32)
    check(L.g53h_block_norm(a.ptr, b.ptr, h.ptr, y.ptr, c), "block_norm")
    yv = y.val()
    yv[2, 7], yv[4, 0] = np.nan, np.inf
    bad = Buf(yv, F32)
    a2, b2 = Buf.out((6, 300), F32), Buf.out((6, 300), F32)
    check(L.g53h_block_norm(a2.ptr, b2.ptr, h.ptr, bad.ptr, c), "block_norm")
    rest = [0, 1, 3, 5]
    assert np.array_equal(a.get()[rest], a2.get()[rest]) and np.array_equal(b.get()[rest], b2.get()[rest])
    assert np.isnan(b2.get()[2]).all()
