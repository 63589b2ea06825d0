"""The norms' gradients in rows above 4096, which other code takes than narrower ones (inputs kept as they came, and above
8192 sums over tokens in LDS): several tokens a workgroup, with and without a post norm and either incoming gradient.
Tolerances are those of test_gpu_norms.py, where they are derived."""
import numpy as np
import pytest

import glm53h
from glm53h import check
from op_lib import BF16, F16, F32, HALF, TINY, Buf, close
from test_gpu_norms import R, S, grads, setup
from test_gpu_parity import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    return glm53h.init(0)


def run(L, T, H, dt, kind, post, which):
    rng = np.random.default_rng(H + T + kind)
    shift = 4 if H % 2 else 0
    h, y, pb, nb, gb, c = setup(rng, T, H, dt, kind, post, shift=shift)
    dh2, dxn = Buf(rng.standard_normal((T, H)), dt, shift), Buf(rng.standard_normal((T, H)), dt, shift)
    dh, dy, dpost, dnext = Buf.out((T, H), dt, shift), Buf.out((T, H), dt, shift), Buf.out(H, F32), Buf.out(H, F32)
    dgate = Buf.out(gb.shape, gb.dt)
    a, b = dh2.ptr if which != "dxn" else None, dxn.ptr if which != "dh2" else None
    outs = [o.ptr for o in (dh, dy, dgate, dpost, dnext)]
    check(L.g53h_block_norm_grad(*outs, a, b, h.ptr, y.ptr, c), "grad")
    want = grads(h.val(), y.val(), pb.val() if post else None, nb.val(), gb.val(), kind, 0.5, c.eps,
                 dh2.val() if a else np.zeros((T, H)), dxn.val() if b else np.zeros((T, H)))
    tol, n = 4 * S, T / 256 + 40
    for name, buf in (("dh", dh), ("dy", dy)):
        w, s = want[name]
        close(buf.val(), w, HALF[dt] * np.abs(w) + TINY[dt] + tol * s, name)
    for name, buf in (("dpost", dpost), ("dnext", dnext)):
        w, s = want[name]
        if name == "dnext" or post:
            close(buf.val(), w.sum(0), (tol + n * R) * s.sum(0) + TINY[F32], name)
    if kind:
        w, s = want["dgate"]
        if kind < 3:
            w, s = w.sum(kind - 1), s.sum(kind - 1)
        close(dgate.val(), w, (HALF[dt] * np.abs(w) + TINY[dt] if kind == 3 else 0) + (tol + (n + 32) * R) * s + TINY[F32], "dgate")
    first = [v.get() for v in (dh, dy, dpost, dnext, dgate)]
    outs[0] = dh2.ptr if a else dh.ptr
    check(L.g53h_block_norm_grad(*outs, a, b, h.ptr, y.ptr, c), "grad in place")
    again = [v.get() for v in (dh2 if a else dh, dy, dpost, dnext, dgate)]
    assert all(np.array_equal(p, q) for p, q in zip(again, first)), "another run, other bits"


@pytest.mark.parametrize("T,H", [(530, 4104), (300, 8192), (259, 6001), (530, 8200), (300, 16384), (513, 9001)])
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_several_tokens_a_workgroup(L, T, H, kind, dt):
    say("block norm grad, wide, several tokens", T, H, kind, dt)
    run(L, T, H, dt, kind, True, "both")


@pytest.mark.parametrize("T,H,dt", [(T, H, dt) for T, H in ((3, 4104), (5, 8192), (2, 8200), (4, 16384)) for dt in (F32, BF16, F16)]
                         + [(T, H, dt) for T, H in ((300, 5001), (290, 9001)) for dt in (F32, BF16)])
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("post,which", [(False, "both"), (True, "dh2"), (True, "dxn"), (False, "dxn"), (False, "dh2")])
def test_without_a_post_norm_or_one_of_the_gradients(L, T, H, kind, dt, post, which):
    say("block norm grad, wide", T, H, kind, dt, post, which)
    run(L, T, H, dt, kind, post, which)


@pytest.mark.parametrize("T,H", [(1030, 520), (270, 2048), (600, 4095)])
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("post,which", [(False, "both"), (True, "dh2"), (True, "dxn")])
def test_many_narrow_rows_without_them(L, T, H, kind, post, which):
    say("block norm grad, many rows", T, H, kind, post, which)
    run(L, T, H, BF16, kind, post, which)


@pytest.mark.parametrize("T,H", [(530, 4104), (300, 8192), (530, 8200), (300, 16384)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_the_norm_alone(L, T, H, dt):
    say("norm grad, wide, several tokens", T, H, dt)
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
