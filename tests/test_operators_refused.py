"""Calls that the operators beside the layer refuse, before anything touches a device: an error that
says why, on any machine. Pointers here are never followed."""
import ctypes as C

import pytest

import glm53h

P = 4096                                     # some address, aligned


@pytest.fixture(scope="module")
def L():
    return glm53h.lib()


def refused(L, rc, *words):
    msg = L.g53h_error().decode()
    assert rc == -1 and all(w in msg for w in words), msg


def plan(T=4, topk=2, NE=8, offsets=P, pair=P, row=P):
    return C.byref(glm53h.G53hSort(T, topk, NE, offsets, pair, row))


@pytest.mark.parametrize("bad", [dict(T=-1), dict(topk=0), dict(topk=65), dict(NE=0), dict(NE=1025),
                                 dict(T=1 << 28, topk=8), dict(offsets=None), dict(pair=None), dict(row=None)])
def test_plans(L, bad):
    refused(L, L.g53h_sort_tokens(plan(**bad), P), "g53h_sort_tokens")
    refused(L, L.g53h_sorted_dispatch(P, P, 0, 16, plan(**bad)), "g53h_sorted_dispatch")
    refused(L, L.g53h_sorted_dispatch_grad(P, P, 0, 16, plan(**bad)), "g53h_sorted_dispatch_grad")
    refused(L, L.g53h_sorted_combine(P, P, P, None, 0, 16, plan(**bad)), "g53h_sorted_combine")
    refused(L, L.g53h_sorted_combine_grad(P, P, P, P, P, 0, 16, plan(**bad)), "g53h_sorted_combine_grad")


def test_rows_and_types(L):
    refused(L, L.g53h_sort_tokens(None, P), "no plan")
    refused(L, L.g53h_sort_tokens(plan(), None), "no routing")
    for dt in (-1, 3):
        refused(L, L.g53h_sorted_dispatch(P, P, dt, 16, plan()), "element type")
        refused(L, L.g53h_sorted_combine(P, P, P, None, dt, 16, plan()), "element type")
    refused(L, L.g53h_sorted_dispatch(P, P, 0, 0, plan()), "hidden 0")
    refused(L, L.g53h_sorted_dispatch(None, P, 0, 16, plan()), "no rows")
    refused(L, L.g53h_sorted_dispatch_grad(P, None, 0, 16, plan()), "no rows")
    refused(L, L.g53h_sorted_combine(P, P, None, None, 0, 16, plan()), "no weights")
    refused(L, L.g53h_sorted_combine_grad(P, None, P, P, P, 0, 16, plan()), "no rows")


def w4(w=P, s=P, z=None, rows=64, cols=128, group=64, s_dt=0):
    return C.byref(glm53h.G53hW4(w, s, z, rows, cols, group, s_dt))


@pytest.mark.parametrize("bad,word", [
    (dict(w=None), "unbound"), (dict(s=None), "unbound"), (dict(rows=0), "levels"), (dict(cols=0), "levels"),
    (dict(cols=100), "levels"), (dict(group=0), "levels"), (dict(group=48), "levels"), (dict(s_dt=3), "levels"),
    (dict(w=P + 8), "multiple of 16"), (dict(s=P + 2), "multiple of 16")])
def test_matrices(L, bad, word):
    refused(L, L.g53h_mm_w4(P, P, 1, 1, w4(**bad), 0.0), word)
    refused(L, L.g53h_sorted_mm_w4(P, P, 1, 0, plan(), w4(**bad), 0.0), word)


def test_products(L):
    refused(L, L.g53h_mm_w4(P, P, 1, 1, None, 0.0), "unbound")
    refused(L, L.g53h_mm_w4(P, P, 7, 1, w4(), 0.0), "element type")
    refused(L, L.g53h_mm_w4(P, P, 1, -1, w4(), 0.0), "tokens")
    refused(L, L.g53h_mm_w4(None, P, 1, 1, w4(), 0.0), "no tokens")
    refused(L, L.g53h_mm_w4(P, P, 1, 1, w4(rows=63), 10.0), "SwiGLU")
    for limit in (-1.0, float("nan"), float("inf")):
        refused(L, L.g53h_mm_w4(P, P, 1, 1, w4(), limit), "SwiGLU")
    refused(L, L.g53h_sorted_mm_w4(P, P, 1, 0, None, w4(), 0.0), "no plan")
    refused(L, L.g53h_sorted_mm_w4(P, P, 1, 0, plan(pair=None), w4(), 0.0), "no plan")
    refused(L, L.g53h_sorted_mm_w4(P, None, 1, 0, plan(), w4(), 0.0), "no rows")


def norm(T=2, hidden=64, dt=1, gate_kind=0, eps=1e-6, scale=1.0, post=P, next=P, gate=P):
    return C.byref(glm53h.G53hBlockNorm(T, hidden, dt, gate_kind, eps, scale, post, next, gate))


@pytest.mark.parametrize("bad", [dict(T=-1), dict(hidden=0), dict(hidden=16385), dict(dt=3), dict(eps=0.0), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(eps=float("inf")), dict(gate_kind=-1), dict(gate_kind=4),
                                 dict(gate_kind=1, gate=None), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(next=None)])
def test_norms(L, bad):
    refused(L, L.g53h_block_norm(P, P, P, P, norm(**bad)), "g53h_block_norm")
    refused(L, L.g53h_block_norm_grad(P, P, P, P, P, P, P, P, P, norm(**bad)), "g53h_block_norm_grad")
    if not set(bad) & {"gate_kind", "scale", "next"}:
        a = dict(dict(dt=1, T=2, hidden=64, eps=1e-6), **bad)
        refused(L, L.g53h_norm(P, P, P, a["dt"], a["T"], a["hidden"], a["eps"]), "g53h_norm")
        refused(L, L.g53h_norm_grad(P, P, P, P, P, a["dt"], a["T"], a["hidden"], a["eps"]), "g53h_norm_grad")


def test_norms_without_rows(L):
    refused(L, L.g53h_norm(None, P, P, 1, 2, 64, 1e-6), "no rows")
    refused(L, L.g53h_norm(P, P, None, 1, 2, 64, 1e-6), "no gain")
    refused(L, L.g53h_norm_grad(P, None, P, P, None, 1, 2, 64, 1e-6), "no gain")
    refused(L, L.g53h_block_norm(P, P, P, P, None), "no parameters")
    refused(L, L.g53h_block_norm(None, P, P, P, norm()), "no rows")
    refused(L, L.g53h_block_norm_grad(P, None, P, P, P, P, P, P, P, norm()), "no rows")
    refused(L, L.g53h_block_norm_grad(P, P, P, P, P, None, None, P, P, norm()), "neither")


def test_sizes_past_the_limits(L):
    for d in (dict(rows=(1 << 30) + 1), dict(cols=(1 << 24) + 32), dict(rows=-64), dict(cols=-128), dict(group=-32)):
        refused(L, L.g53h_mm_w4(P, P, 1, 1, w4(**d), 0.0), "levels")
        refused(L, L.g53h_sorted_mm_w4(P, P, 1, 0, plan(), w4(**d), 0.0), "levels")
    refused(L, L.g53h_sorted_dispatch(P, P, 0, (1 << 30) + 1, plan()), "hidden")
    refused(L, L.g53h_sorted_combine(P, P, P, None, 0, (1 << 30) + 1, plan()), "hidden")
    for eps in (9e-31, 2e30):
        refused(L, L.g53h_norm(P, P, P, 1, 2, 64, eps), "eps")
        refused(L, L.g53h_block_norm(P, P, P, P, norm(eps=eps)), "eps")


def test_struct_sizes():
    assert C.sizeof(glm53h.G53hSort) == 40
    assert C.sizeof(glm53h.G53hW4) == 40
    assert C.sizeof(glm53h.G53hBlockNorm) == 48


@pytest.mark.parametrize("bad", [dict(T=-1), dict(topk=0), dict(topk=65), dict(NE=0), dict(NE=1025), dict(T=1 << 28, topk=8),
                                 dict(offsets=None), dict(pair=None)])
def test_expert_products_plans(L, bad):
    refused(L, L.g53h_sorted_mm(P, None, P, 1, 0, plan(**bad), P, 8, 8, 0.0), "g53h_sorted_mm", "plan")
    refused(L, L.g53h_sorted_mm_grad(P, P, 0, 0, P, P, 1, 0, plan(**bad), P, 8, 8), "g53h_sorted_mm_grad", "plan")
    refused(L, L.g53h_sorted_swiglu_grad(P, P, P, 1, 8, plan(**bad), 1.0), "g53h_sorted_swiglu_grad", "plan")


def test_expert_products(L):
    for dt in (-1, 3):
        refused(L, L.g53h_sorted_mm(P, None, P, dt, 0, plan(), P, 8, 8, 0.0), "element type")
        refused(L, L.g53h_sorted_mm_grad(P, P, 0, 0, P, P, dt, 0, plan(), P, 8, 8), "element type")
        refused(L, L.g53h_sorted_swiglu_grad(P, P, P, dt, 8, plan(), 1.0), "element type")
    for rows, cols in ((0, 8), (8, 0), (-8, 8), ((1 << 24) + 1, 8), (8, (1 << 24) + 1)):
        refused(L, L.g53h_sorted_mm(P, None, P, 1, 0, plan(), P, rows, cols, 0.0), "matrices")
        refused(L, L.g53h_sorted_mm_grad(P, P, 0, 0, P, P, 1, 0, plan(), P, rows, cols), "matrices")
    for limit in (-1.0, float("nan"), float("inf")):
        refused(L, L.g53h_sorted_mm(P, None, P, 1, 0, plan(), P, 8, 8, limit), "limit")
        refused(L, L.g53h_sorted_swiglu_grad(P, P, P, 1, 8, plan(), limit), "limit")
    refused(L, L.g53h_sorted_swiglu_grad(P, P, P, 1, 8, plan(), 0.0), "limit")
    refused(L, L.g53h_sorted_swiglu_grad(P, P, P, 1, 0, plan(), 1.0), "matrices")
    refused(L, L.g53h_sorted_mm(P, None, P, 1, 0, plan(), P, 7, 8, 1.0), "SwiGLU")
    refused(L, L.g53h_sorted_mm(P, P, P, 1, 0, plan(), P, 8, 8, 0.0), "without SwiGLU")
    refused(L, L.g53h_sorted_mm(None, None, P, 1, 0, plan(), P, 8, 8, 0.0), "no rows")
    refused(L, L.g53h_sorted_mm(P, None, P, 1, 0, plan(), None, 8, 8, 0.0), "no matrices")
    refused(L, L.g53h_sorted_mm(P, None, P + 1, 1, 0, plan(), P, 8, 8, 0.0), "multiples of an element")
    refused(L, L.g53h_sorted_mm_grad(None, None, 0, 0, P, P, 1, 0, plan(), P, 8, 8), "neither")
    refused(L, L.g53h_sorted_mm_grad(P, P, 2, 0, P, P, 1, 0, plan(), P, 8, 8), "of type 2")
    refused(L, L.g53h_sorted_mm_grad(P, None, 0, 0, None, P, 1, 0, plan(), P, 8, 8), "no rows")
    refused(L, L.g53h_sorted_mm_grad(P, None, 0, 0, P, P, 1, 0, plan(), None, 8, 8), "no matrices")
    refused(L, L.g53h_sorted_mm_grad(None, P, 0, 0, P, None, 1, 0, plan(), P, 8, 8), "no rows")
    refused(L, L.g53h_sorted_mm_grad(None, P + 2, 0, 0, P, P, 1, 0, plan(), P, 8, 8), "multiples of an element")
    refused(L, L.g53h_sorted_swiglu_grad(P, None, P, 1, 8, plan(), 1.0), "no rows")


def mx4(w=P, s=P, rows=8, cols=64):
    return C.byref(glm53h.G53hMx4(w, s, rows, cols))


@pytest.mark.parametrize("bad,word", [(dict(w=None), "unbound"), (dict(s=None), "unbound"), (dict(rows=-1), "levels"), (dict(cols=0), "levels"),
                                      (dict(cols=48), "levels"), (dict(cols=(1 << 24) + 32), "levels"), (dict(cols=-32), "levels"),
                                      (dict(w=P + 8), "multiple of 16")])
def test_microscaled_matrices(L, bad, word):
    refused(L, L.g53h_mx4_quant(mx4(**bad), P, 1), word)
    refused(L, L.g53h_mx4_dequant(P, 1, mx4(**bad)), word)
    for x, m in ((bad, {}), ({}, bad)):
        refused(L, L.g53h_mm_mx4(P, 1, mx4(**x), mx4(**m), 0.0), word)
        refused(L, L.g53h_sorted_mm_mx4(P, 1, mx4(**x), 1, plan(), mx4(**m), 0.0), word)


def test_microscaled_products(L):
    refused(L, L.g53h_mx4_quant(None, P, 1), "no matrix")
    refused(L, L.g53h_mx4_quant(mx4(), None, 1), "no rows")
    refused(L, L.g53h_mx4_quant(mx4(), P + 1, 1), "multiple of an element")
    refused(L, L.g53h_mx4_dequant(P + 2, 0, mx4()), "multiple of an element")
    for dt in (-1, 3):
        refused(L, L.g53h_mx4_quant(mx4(), P, dt), "element type")
        refused(L, L.g53h_mx4_dequant(P, dt, mx4()), "element type")
        refused(L, L.g53h_mm_mx4(P, dt, mx4(), mx4(), 0.0), "element type")
        refused(L, L.g53h_sorted_mm_mx4(P, dt, mx4(), 1, plan(), mx4(), 0.0), "element type")
    refused(L, L.g53h_mm_mx4(P, 1, mx4(), None, 0.0), "no matrix")
    refused(L, L.g53h_mm_mx4(P, 1, mx4(), mx4(rows=0), 0.0), "0 rows")
    refused(L, L.g53h_mm_mx4(P, 1, mx4(cols=32), mx4(), 0.0), "32 columns")
    refused(L, L.g53h_mm_mx4(P, 1, mx4(), mx4(rows=7), 1.0), "SwiGLU")
    for limit in (-1.0, float("nan"), float("inf")):
        refused(L, L.g53h_mm_mx4(P, 1, mx4(), mx4(), limit), "SwiGLU")
    refused(L, L.g53h_mm_mx4(None, 1, mx4(), mx4(), 0.0), "no results")
    refused(L, L.g53h_mm_mx4(P + 1, 1, mx4(), mx4(), 0.0), "multiple of an element")
    refused(L, L.g53h_sorted_mm_mx4(None, 1, mx4(), 1, plan(), mx4(), 0.0), "no results")
    for bad in (dict(T=-1), dict(topk=0), dict(NE=1025), dict(offsets=None), dict(pair=None)):
        refused(L, L.g53h_sorted_mm_mx4(P, 1, mx4(), 1, plan(**bad), mx4(), 0.0), "plan")
    refused(L, L.g53h_sorted_mm_mx4(P, 1, mx4(rows=3), 1, plan(T=4), mx4(), 0.0), "3 rows of x")
    refused(L, L.g53h_sorted_mm_mx4(P, 1, mx4(rows=7), 0, plan(T=4, topk=2), mx4(), 0.0), "7 rows of x")


def test_new_struct_sizes():
    assert C.sizeof(glm53h.G53hMx4) == 24


def test_expert_products_most_pairs(L):
    most = (1 << 31) - 1024
    refused(L, L.g53h_sorted_mm(P, None, P, 1, 0, plan(T=most + 1, topk=1), P, 8, 8, 0.0), "2^31 - 1024")
    refused(L, L.g53h_sorted_mm_grad(P, P, 0, 0, P, P, 1, 0, plan(T=most + 1, topk=1), P, 8, 8), "2^31 - 1024")
    refused(L, L.g53h_sorted_swiglu_grad(P, P, P, 1, 8, plan(T=most + 1, topk=1), 1.0), "2^31 - 1024")
