"""Timed cases of the experts' own products: matrices of one expert each over ragged sorted rows, forward and
backward, in 32 and 16 bits, and microscaled 4-bit matrices (E2M1 levels, one power of two for 32 columns),
quantised and multiplied.

A case is a dict of plain values:

  op      "mm"     the product of every token's rows with their experts' matrices
          "grad"   its gradients, to the rows and to the matrices
          "quant"  rows into microscaled 4 bits, and read back
          "mx4"    rows quantised, then multiplied with a quantised matrix, or with those of their experts
  dt      element type of activations (and of the matrices that are not quantised): "f32", "bf16", "f16"
  T, NE, K      tokens, experts (0: one matrix, no routing), experts per token; pad: trailing tokens without experts
  rows, cols    of a matrix; "quant": of what is quantised
  swiglu  whether a product's rows are gate and up, joined by the clamped SwiGLU; "grad": differentiated too
  keep    "mm" with swiglu: gate and up are returned as well, for the backward pass
  w_dt    "grad": type of the matrices' gradient

Where `own` is true, `run` calls the library; else it is elementary torch in 32 bits.
"""
import ctypes as C
import math
import os
import sys

import torch

own = False

LIMIT = 10.0
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
BIG = dict(NE=288, K=8, rows=4096, cols=4096)
MID = dict(NE=64, K=8, rows=4096, cols=4096)


def listed():
    return [
        # one generated token through the gate and up matrices of its eight experts
        dict(name="mm_1", op="mm", dt="bf16", T=1, pad=0, swiglu=True, keep=False, **BIG),
        # a ragged fine-tuning batch in odd sizes, padded at its end
        dict(name="mm_301", op="mm", dt="f16", T=301, pad=5, NE=37, K=3, rows=1001, cols=1023, swiglu=False, keep=False),
        # a training step's forward pass through gate and up, which the backward pass needs again
        dict(name="mm_4096", op="mm", dt="bf16", T=4096, pad=0, swiglu=True, keep=True, **MID),
        # down matrices in the layer's own 32 bits
        dict(name="mm_512_f32", op="mm", dt="f32", T=512, pad=0, NE=16, K=4, rows=2048, cols=1024, swiglu=False, keep=False),
        # a small batch in 32 bits, as a check of a training loop runs it
        dict(name="grad_37_f32", op="grad", dt="f32", T=37, pad=0, NE=8, K=2, rows=514, cols=301, swiglu=True, w_dt="f32"),
        # a fine-tuning batch through the down matrices of a smaller model
        dict(name="grad_700", op="grad", dt="f16", T=700, pad=9, NE=32, K=4, rows=2048, cols=1024, swiglu=False, w_dt="f16"),
        # a training step's backward pass through gate and up, the matrices' gradients in 32 bits
        dict(name="grad_2048", op="grad", dt="bf16", T=2048, pad=0, swiglu=True, w_dt="f32", **MID),
        # one generated token's activations
        dict(name="quant_1", op="quant", dt="bf16", rows=1, cols=4096),
        # sixteen experts' matrices after training
        dict(name="quant_experts", op="quant", dt="bf16", rows=16 * 4096, cols=4096),
        # one generated token through the gate and up matrices of its eight experts
        dict(name="mx4_1", op="mx4", dt="bf16", T=1, pad=0, swiglu=True, **BIG),
        # a few sequences through a large dense head
        dict(name="mx4_head_5", op="mx4", dt="f16", T=5, pad=0, NE=0, K=1, rows=65536, cols=4096, swiglu=False),
        # a prompt through gate and up
        dict(name="mx4_4096", op="mx4", dt="bf16", T=4096, pad=0, swiglu=True, **MID),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["mm", "mm", "grad", "grad", "quant", "mx4", "mx4"])
    dt = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quant":
        return dict(op=op, dt=dt, rows=_log_int(rng, 1, 16384), cols=32 * _log_int(rng, 1, 256))
    T, NE = rng.choice([1, _log_int(rng, 1, 2048), _log_int(rng, 64, 2048)]), _log_int(rng, 2, 64)
    c = dict(op=op, dt=dt, T=T, pad=rng.choice([0, T // 9]), NE=NE, K=rng.randint(1, min(8, NE)), swiglu=rng.random() < 0.5)
    size = lambda step: step * _log_int(rng, max(1, 64 // step), 2048 // step)  # noqa: E731
    c["rows"], c["cols"] = (rng.choice([size(64), size(2 if c["swiglu"] else 1)]) for _ in range(2))
    if op == "mm":
        c["keep"] = c["swiglu"] and rng.random() < 0.5
    elif op == "grad":
        c["w_dt"] = rng.choice([dt, "f32"])
    else:
        c["cols"] = size(32)
        if rng.random() < 0.4:
            c.update(NE=0, K=1, pad=0, rows=2 * _log_int(rng, 32, 8192))
    return c


# ------------------------------------------------------------------ inputs from a seed ----
def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 64 + stream)
    return g


def _normal(seed, stream, *shape, dt="f32", scale=1.0):
    g, out = _gen(seed, stream), torch.empty(shape, dtype=DT[dt], device="cuda")
    flat, step = out.view(-1), 1 << 28
    for i in range(0, flat.numel(), step):
        m = min(step, flat.numel() - i)
        flat[i:i + m] = torch.randn(m, generator=g, device="cuda").mul_(scale)
    return out


def _activations(seed, stream, rows, cols, dt):
    """Rows N(0, 1) whose channels differ in size, a few of them by much."""
    size = torch.exp(0.5 * torch.randn(cols, generator=_gen(seed, stream + 1), device="cuda"))
    size[::97] *= 8.0
    return (torch.randn((rows, cols), generator=_gen(seed, stream), device="cuda") * size).to(DT[dt])


def _routing(case, seed):
    """Experts [T][K] of every token, distinct, uneven in popularity, -1 for the padded tokens."""
    T, NE, K = case["T"], case["NE"], case["K"]
    bias = torch.rand(NE, generator=_gen(seed, 1), device="cuda")
    score = torch.rand((T, NE), generator=_gen(seed, 2), device="cuda") + bias
    idx = torch.argsort(score, dim=1, descending=True, stable=True)[:, :K].to(torch.int32).contiguous()
    idx[T - case["pad"]:] = -1
    return idx


def _sorted(idx, NE):
    """offsets [NE + 1], pair [n], row [n] of a routing: pairs in order of expert, then of pair."""
    flat = idx.reshape(-1).long()
    n = flat.numel()
    key, order = torch.sort(torch.where((flat >= 0) & (flat < NE), flat, NE), stable=True)
    offsets = torch.searchsorted(key, torch.arange(NE + 1, device=key.device))
    at = torch.arange(n, device=key.device)
    pair = torch.where(at < offsets[NE], order, -1)
    row = torch.empty_like(order)
    row[order] = at
    row = torch.where(row < offsets[NE], row, -1)
    return offsets.to(torch.int32), pair.to(torch.int32), row.to(torch.int32)


def _pow2(k):
    """2^k in 32 bits for whole k from -127 to 127."""
    return torch.where(k > -127, (k + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _levels(x):
    """Rows of fp32 to microscaled 4 bits: packed levels [rows][cols / 2] (the even column in the low nibble; bit 3 is
    the sign, bits 0 to 2 count 0, 0.5, 1, 1.5, 2, 3, 4, 6) and scales [rows][cols / 32], 127 + their power of two: that of
    the largest value, less 2."""
    v = x.view(x.shape[0], -1, 32)
    top = v.abs().amax(2, keepdim=True).view(torch.int32)
    s = ((top >> 23) - 2).clamp_(min=0)
    a = v.abs() * _pow2(127 - s)
    lv = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    lv = (lv + torch.signbit(v) * 8).to(torch.uint8).view(x.shape)
    return lv[:, 0::2] | (lv[:, 1::2] << 4), s.squeeze(2).to(torch.uint8)


def _mx4(seed, rows, cols):
    """A quantised matrix of weights N(0, 0.02)."""
    q = torch.empty((rows, cols // 2), dtype=torch.uint8, device="cuda")
    s = torch.empty((rows, cols // 32), dtype=torch.uint8, device="cuda")
    g, step = _gen(seed, 8), max(1, (1 << 27) // cols)
    for r in range(0, rows, step):
        m = min(step, rows - r)
        q[r:r + m], s[r:r + m] = _levels(torch.randn((m, cols), generator=g, device="cuda").mul_(0.02))
    return q, s


def _out_cols(case):
    return case["rows"] // 2 if case["swiglu"] else case["rows"]


# ----------------------------------------------------------------------------- prepare ----
def prepare(case, seed):
    op, dt, rows, cols = case["op"], case["dt"], case["rows"], case["cols"]
    st = dict(case=case, op=op)
    new = lambda *shape, t=DT[dt]: torch.zeros(shape, dtype=t, device="cuda")  # noqa: E731
    u8 = torch.uint8
    if op == "quant":
        st.update(x=_activations(seed, 4, rows, cols, dt), q=new(rows, cols // 2, t=u8), s=new(rows, cols // 32, t=u8),
                  back=new(rows, cols))
        torch.cuda.synchronize()
        return st
    T, NE, K = case["T"], case["NE"], case["K"]
    n = T * K
    if NE:
        st["plan"] = list(_sorted(_routing(case, seed), NE))
        st["most"] = int(st["plan"][0].diff().max())          # rows of the busiest expert
    if op == "mx4":
        st.update(x=_activations(seed, 4, T, cols, dt), m=_mx4(seed, max(NE, 1) * rows, cols), xq=new(T, cols // 2, t=u8),
                  xs=new(T, cols // 32, t=u8), y=new(n, _out_cols(case)))
    else:
        st.update(x=_normal(seed, 4, T, cols, dt=dt), w=_normal(seed, 8, NE, rows, cols, dt=dt, scale=0.02))
        if op == "mm":
            st.update(y=new(n, _out_cols(case)), gu=new(n, rows) if case["keep"] else None)
        else:
            st.update(dy=_normal(seed, 5, n, _out_cols(case), dt=dt), gu=_normal(seed, 6, n, rows, dt=dt) if case["swiglu"] else None,
                      dgu=new(n, rows) if case["swiglu"] else None, dx=new(n, cols), dw=new(NE, rows, cols, t=DT[case["w_dt"]]))
    torch.cuda.synchronize()          # the library works on a stream of its own
    return st


# ------------------------------------------------------------------------- plain forms ----
def _swiglu(y):
    g, u = y.chunk(2, -1)
    g = g.clamp(max=LIMIT)
    return g / (1.0 + torch.exp(-g)) * u.clamp(-LIMIT, LIMIT)


def _padded(st):
    """The experts that have rows first (as many as can have some), and each one's rows, padded to the most that one has:
    experts [b], rows [b][most], which of them are rows [b][most]."""
    NE, offsets, n = st["case"]["NE"], st["plan"][0].long(), st["plan"][1].numel()
    count = offsets.diff()
    busy = torch.argsort((count > 0).int(), descending=True, stable=True)[:min(n, NE)]
    at = torch.arange(st["most"], device=offsets.device)
    return busy, (offsets[busy][:, None] + at).clamp(max=n - 1), at < count[busy][:, None]


def _products(st, x, W):
    """Every sorted row's product with its expert's matrix, zeros behind the last: x in 32 bits, W(experts) theirs."""
    c, pair = st["case"], st["plan"][1]
    busy, p, keep = _padded(st)
    xe = x[pair[p].clamp(min=0).long() // c["K"]].transpose(1, 2).contiguous()
    y = torch.bmm(W(busy), xe).transpose(1, 2)
    out = torch.zeros((pair.numel(), c["rows"]), device=x.device)
    return out.index_add_(0, p.view(-1), torch.where(keep[..., None], y, 0).reshape(-1, c["rows"]))


def _plain_mm(st):
    c, t = st["case"], st["x"].dtype
    gu = _products(st, st["x"].float(), lambda e: st["w"][e].float())
    if not c["swiglu"]:
        return dict(y=gu.to(t))
    return dict(y=_swiglu(gu).to(t), gu=gu.to(t)) if c["keep"] else dict(y=_swiglu(gu).to(t))


def _plain_grad(st):
    c, t, w_t = st["case"], st["x"].dtype, st["dw"].dtype
    offsets, pair, _ = st["plan"]
    out, some = {}, (torch.arange(pair.numel(), device=pair.device) < offsets[-1])[:, None]
    dy = st["dy"].float()
    if c["swiglu"]:
        g, u = st["gu"].float().chunk(2, -1)
        gc, uc = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        sig = 1.0 / (1.0 + torch.exp(-gc))
        dg = torch.where(g <= LIMIT, dy * uc * sig * (1.0 + gc * (1.0 - sig)), 0)
        du = torch.where(u.abs() <= LIMIT, dy * gc * sig, 0)
        dgu = torch.where(some, torch.cat((dg, du), 1), 0).to(t)
        out["dgu"], dy = dgu, dgu.float()
    busy, p, keep = _padded(st)
    de = torch.where(keep[..., None], dy[p], 0)
    dxe = torch.bmm(de, st["w"][busy].float())
    dx = torch.zeros((pair.numel(), c["cols"]), device=dy.device)
    dx.index_add_(0, p.view(-1), torch.where(keep[..., None], dxe, 0).view(-1, c["cols"]))
    xe = st["x"].float()[pair[p].clamp(min=0).long() // c["K"]]
    dw = torch.zeros(st["dw"].shape, dtype=w_t, device=dy.device)
    dw[busy] = torch.bmm(de.transpose(1, 2).contiguous(), xe).to(w_t)
    return dict(out, dx=dx.to(t), dw=dw)


def _values(q, s):
    """What microscaled levels stand for, in 32 bits."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=q.device)
    table = torch.cat((table, -table))
    v = table[torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1).int()]
    return (v.view(q.shape[0], -1, 32) * _pow2(s.int()[..., None] - 127)).view(q.shape[0], -1)


def _plain_quant(st):
    return _values(*_levels(st["x"].float())).to(st["x"].dtype)


def _plain_mx4(st):
    c, (q, s) = st["case"], st["m"]
    x = _values(*_levels(st["x"].float()))
    if c["NE"]:
        mats = [v.view(c["NE"], c["rows"], -1) for v in (q, s)]
        y = _products(st, x, lambda e: _values(*(v[e].flatten(0, 1) for v in mats)).view(len(e), c["rows"], -1))
    else:
        y = x @ _values(q, s).T
    return (_swiglu(y) if c["swiglu"] else y).to(st["x"].dtype)


# -------------------------------------------------------------------- the library's calls ----
def _lib():
    if _lib.glm53h is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "glm-5.3-flash-in-c_amd"))
        import glm53h
        glm53h.init(0)
        _lib.glm53h = glm53h
    return _lib.glm53h


_lib.glm53h = None


def _ptr(t):
    return t.data_ptr() if t is not None and t.numel() else None


def _calls(st):
    """The library calls of a pass, (function, arguments), and what it returns. The descriptors and pointers of a
    program's own buffers are made once."""
    G = _lib()
    L, c, p = G.lib(), st["case"], lambda k: _ptr(st[k])
    dt, rows, cols = CODE[DT[c["dt"]]], c["rows"], c["cols"]
    limit = LIMIT if c.get("swiglu") else 0.0
    if st["op"] == "quant":
        m = G.G53hMx4(p("q"), p("s"), rows, cols)
        return [(L.g53h_mx4_quant, (C.byref(m), p("x"), dt)), (L.g53h_mx4_dequant, (p("back"), dt, C.byref(m)))], st["back"]
    if "plan" in st:
        plan = C.byref(G.G53hSort(c["T"], c["K"], c["NE"], *[t.data_ptr() for t in st["plan"]]))
    if st["op"] == "mx4":
        q, s = st["m"]
        x, m = G.G53hMx4(p("xq"), p("xs"), c["T"], cols), G.G53hMx4(q.data_ptr(), s.data_ptr(), rows, cols)
        calls = [(L.g53h_mx4_quant, (C.byref(x), p("x"), dt))]
        if c["NE"]:
            calls.append((L.g53h_sorted_mm_mx4, (p("y"), dt, C.byref(x), 1, plan, C.byref(m), limit)))
        else:
            calls.append((L.g53h_mm_mx4, (p("y"), dt, C.byref(x), C.byref(m), limit)))
        return calls, st["y"]
    if st["op"] == "mm":
        return [(L.g53h_sorted_mm, (p("y"), p("gu"), p("x"), dt, 1, plan, p("w"), rows, cols, limit))], dict(
            y=st["y"], gu=st["gu"]) if c["keep"] else dict(y=st["y"])
    out, calls, dy = dict(dx=st["dx"], dw=st["dw"]), [], "dy"
    if c["swiglu"]:
        calls.append((L.g53h_sorted_swiglu_grad, (p("dgu"), p("dy"), p("gu"), dt, rows // 2, plan, limit)))
        out, dy = dict(out, dgu=st["dgu"]), "dgu"
    calls.append((L.g53h_sorted_mm_grad, (p("dx"), p("dw"), CODE[st["dw"].dtype], 0, p(dy), p("x"), dt, 1, plan, p("w"), rows, cols)))
    return calls, out


def run(state):
    if not own:
        return {"mm": _plain_mm, "grad": _plain_grad, "quant": _plain_quant, "mx4": _plain_mx4}[state["op"]](state)
    if "calls" not in state:
        state["calls"] = _calls(state)
    calls, out = state["calls"]
    for f, args in calls:
        if f(*args):
            raise RuntimeError(_lib().lib().g53h_error().decode())
    return out


# -------------------------------------------------------------------------------- work ----
def work(case):
    op, b, rows, cols = case["op"], 4 if case["dt"] == "f32" else 2, case["rows"], case["cols"]
    if op == "quant":
        return {"bytes": 2 * rows * cols * (b + 17 / 32), "flops": 4 * rows * cols}
    T, NE, K = case["T"], case["NE"], case["K"]
    n, routed = T * K, (T - case["pad"]) * K
    busy = NE * (1.0 - (1.0 - K / NE) ** (T - case["pad"])) if NE else 1.0           # at even popularity
    lists = 4 * (n + NE + 1) if NE else 0
    if op == "mx4":
        one = rows * cols * 17 / 32
        return {"bytes": busy * one + lists + T * cols * (b + 17 / 16) + routed * _out_cols(case) * b, "flops": 2 * routed * rows * cols}
    if op == "mm":
        out = _out_cols(case) + (rows if case["keep"] else 0)
        return {"bytes": (busy * rows * cols + T * cols + routed * out) * b + lists, "flops": 2 * routed * rows * cols}
    wb = 4 if case["w_dt"] == "f32" else 2
    # with SwiGLU gate, up and their gradients pass once more
    act = (_out_cols(case) + 2 * rows) if case["swiglu"] else rows
    return {"bytes": (busy * rows * cols + T * cols + routed * (act + cols)) * b + NE * rows * cols * wb + lists,
            "flops": 4 * routed * rows * cols}


# ------------------------------------------------------------------------------- exact ----
def _two64(k):
    """2^k in 64 bits."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _quant64(x):
    """Values of microscaled 4 bits nearest to x, ties to the even level, from the format's definition."""
    v = x.double().view(x.shape[0], -1, 32)
    _, e = torch.frexp(v.abs().amax(2, keepdim=True))           # the largest lies in [2^(e - 1), 2^e)
    unit = _two64((e - 3).clamp(min=-127))
    a = v.abs() / unit
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    a = torch.clamp(torch.round(a / step) * step, max=6.0)
    return (torch.copysign(a, v) * unit).view(x.shape)


def _mx4_64(q, s):
    lv = torch.empty((q.shape[0], 2 * q.shape[1]), dtype=torch.int64, device=q.device)
    lv[:, 0::2], lv[:, 1::2] = q % 16, q // 16
    e, frac = (lv % 8) // 2, (lv % 2).double()                  # exponent and one bit of fraction
    v = torch.where(e == 0, frac / 2, (1.0 + frac / 2) * _two64(e - 1))
    v = torch.where(lv >= 8, -v, v).view(q.shape[0], -1, 32)
    return (v * _two64(s.long() - 127)[..., None]).view(q.shape[0], -1)


def _act64(y):
    half = y.shape[-1] // 2
    g, u = y[..., :half].clamp(max=LIMIT), y[..., half:].clamp(min=-LIMIT, max=LIMIT)
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    st = prepare(case, seed)
    op, rows = case["op"], case["rows"]
    if op == "quant":
        return torch.cat([_quant64(part) for part in st["x"].split(8192)])
    if not case["NE"]:
        x, (q, s) = _quant64(st["x"]), st["m"]
        y = torch.cat([x @ _mx4_64(q[r:r + 8192], s[r:r + 8192]).T for r in range(0, rows, 8192)], 1)
        return _act64(y) if case["swiglu"] else y
    idx, n = _routing(case, seed), case["T"] * case["K"]
    lists = [torch.nonzero(idx == e, as_tuple=True)[0] for e in range(case["NE"])]     # the tokens of every expert, in order
    new = lambda m: torch.zeros((n, m), dtype=torch.float64, device="cuda")  # noqa: E731
    at = 0
    if op in ("mm", "mx4"):
        gu = new(rows)
        x = st["x"].double() if op == "mm" else _quant64(st["x"])
        for e, t in enumerate(lists):
            if len(t):
                W = st["w"][e].double() if op == "mm" else _mx4_64(*(v[e * rows:(e + 1) * rows] for v in st["m"]))
                gu[at:at + len(t)] = x[t] @ W.T
                at += len(t)
        y = _act64(gu) if case["swiglu"] else gu
        if op == "mx4":
            return y
        return dict(y=y, gu=gu) if case["keep"] else dict(y=y)
    out = {}
    dy, m = st["dy"].double(), sum(len(t) for t in lists)
    if case["swiglu"]:
        gu = st["gu"].double().requires_grad_(True)
        dgu, = torch.autograd.grad((_act64(gu) * dy).sum(), gu)
        dgu[m:] = 0
        out["dgu"], dy = dgu, dgu.to(st["x"].dtype).double()        # the rounded gradient goes on
    x, dx, dw = st["x"].double(), new(case["cols"]), torch.zeros(st["w"].shape, dtype=torch.float64, device="cuda")
    for e, t in enumerate(lists):
        if len(t):
            d = dy[at:at + len(t)]
            dx[at:at + len(t)] = d @ st["w"][e].double()
            dw[e] = d.T @ x[t]
            at += len(t)
    return dict(out, dx=dx, dw=dw)
