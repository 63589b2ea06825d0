"""Timed cases of the operators around the expert products: tokens sorted by expert and back with
their gradients, products with 4-bit weights and group scales, and the norms before and after a
block with its gate and residual scale.

A case is a dict of plain values:

  op      "forward"   sort the routing, gather the rows of x by expert, combine given expert rows
          "backward"  the gradients of that combine and of that gather
          "w4"        one product of T tokens with a 4-bit matrix
          "experts"   one product of the sorted rows with their experts' 4-bit matrices
          "norm"      the norm after a block, its gate and residual, and the next block's norm
          "norm_grad" the gradient of that
  dt      element type of activations: "f32", "bf16", "f16"
  T, H, NE, K   tokens, hidden size, experts, experts per token; pad: trailing tokens without experts
  rows, cols, group, s_dt, zeros   4-bit matrix (experts: of each), its scales and zero points
  swiglu  whether a product's rows are gate and up, joined by the clamped SwiGLU
  gate    0 none, 1 per channel, 2 per token, 3 per token and channel

Where `own` is true, `run` calls the library; else it is elementary torch in 32 bits.
"""
import ctypes as C
import math
import os
import sys

import torch

own = False

LIMIT, EPS, SCALE = 10.0, 1e-6, 0.5
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
BIG = dict(H=4096, NE=288, K=8)


def listed():
    return [
        # one token being generated: its eight rows and their sum
        dict(name="forward_1", op="forward", dt="bf16", T=1, pad=0, **BIG),
        # a large prefill batch, padded at its end
        dict(name="forward_4096", op="forward", dt="bf16", T=4096, pad=37, **BIG),
        # a small ragged fine-tuning batch in 32 bits, odd sizes
        dict(name="backward_301", op="backward", dt="f32", T=301, pad=5, H=1023, NE=37, K=3),
        # a training step's micro-batch at the released sizes
        dict(name="backward_2048", op="backward", dt="bf16", T=2048, pad=0, **BIG),
        # one token through a dense projection in the engine's own int4 form (groups of 64, fp32 steps)
        dict(name="w4_1", op="w4", dt="bf16", T=1, rows=4096, cols=2048, group=64, s_dt="f32", zeros=False, swiglu=False),
        # a few sequences through an output head quantised with zero points
        dict(name="w4_head_5", op="w4", dt="f16", T=5, rows=65536, cols=4096, group=128, s_dt="f16", zeros=True,
             swiglu=False),
        # a ragged matrix in the drop-in's 32-bit activations, the finest groups
        dict(name="w4_24_f32", op="w4", dt="f32", T=24, rows=1001, cols=2080, group=32, s_dt="f16", zeros=True,
             swiglu=False),
        # one generated token through its eight experts' gate and up matrices
        dict(name="experts_1", op="experts", dt="bf16", T=1, NE=288, K=8, rows=4096, cols=4096, group=128, s_dt="bf16",
             zeros=False, swiglu=True),
        # a batch of sequences through a smaller model's down matrices
        dict(name="experts_64", op="experts", dt="bf16", T=64, NE=64, K=6, rows=2048, cols=1024, group=64, s_dt="f32",
             zeros=False, swiglu=False),
        # one generated token's residual stream
        dict(name="norm_1", op="norm", dt="bf16", T=1, H=4096, gate=1),
        # a prefill batch with a learned gate of every token and channel
        dict(name="norm_2048", op="norm", dt="bf16", T=2048, H=4096, gate=3),
        # the same trained, an odd number of tokens
        dict(name="norm_grad_1025", op="norm_grad", dt="bf16", T=1025, H=4096, gate=1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["forward", "backward", "w4", "w4", "experts", "experts", "norm", "norm_grad"])
    dt = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("forward", "backward"):
        T, H = _log_int(rng, 1, 4096 if op == "forward" else 2048), rng.choice([4096, _log_int(rng, 33, 4096)])
        c = dict(op=op, dt=dt, T=T, pad=rng.choice([0, T // 9]), H=H, NE=_log_int(rng, 2, 288), K=0)
        c["K"] = rng.randint(1, min(8, c["NE"]))
        if dt == "f32":
            c["T"], c["pad"] = (T + 1) // 2, c["pad"] // 2
        return c
    if op in ("norm", "norm_grad"):
        T = _log_int(rng, 1, 2048 if op == "norm" else 1024)
        return dict(op=op, dt=dt, T=(T + 1) // 2 if dt == "f32" else T, H=rng.choice([4096, _log_int(rng, 33, 4096)]),
                    gate=rng.randint(0, 3))
    c = dict(op=op, dt=dt, T=1, s_dt=rng.choice(["f32", "bf16", "f16"]), zeros=rng.random() < 0.5, swiglu=rng.random() < 0.4)
    if op == "w4":
        c.update(T=rng.choice([1, _log_int(rng, 1, 128)]), rows=2 * _log_int(rng, 32, 8192), cols=32 * _log_int(rng, 2, 128))
    else:
        c.update(T=rng.choice([1, _log_int(rng, 1, 256)]), NE=_log_int(rng, 8, 64), rows=2 * _log_int(rng, 64, 1024),
                 cols=32 * _log_int(rng, 4, 64), K=rng.choice([2, 4, 6, 8]))
    c["group"] = rng.choice([32, 64, 128, 128, c["cols"]])
    return c


# ------------------------------------------------------------------ inputs from a seed ----
def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 64 + stream)
    return g


def _normal(seed, stream, *shape, dt="f32"):
    return torch.randn(shape, generator=_gen(seed, stream), device="cuda").to(DT[dt])


def _routing(case, seed):
    """Experts [T][K] of every token, distinct, uneven in popularity, -1 for the padded tokens, and their weights."""
    T, NE, K = case["T"], case["NE"], case["K"]
    bias = torch.rand(NE, generator=_gen(seed, 1), device="cuda")
    score = torch.rand((T, NE), generator=_gen(seed, 2), device="cuda") + bias
    idx = torch.argsort(score, dim=1, descending=True, stable=True)[:, :K].to(torch.int32).contiguous()
    w = torch.rand((T, K), generator=_gen(seed, 3), device="cuda").add_(0.1)
    w = w.div_(w.sum(1, keepdim=True)).mul_(2.5)
    idx[T - case.get("pad", 0):] = -1
    return idx, w


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


def _w4(case, seed, n):
    """n matrices: packed levels [n * rows][cols / 2] (even column in the low nibble), scales [n * rows][groups]
    and packed zero points [n * rows][ceil(groups / 2)] or None, of weights N(0, 0.02)."""
    rows, cols, group = case["rows"], case["cols"], case["group"]
    groups = -(-cols // group)
    q = torch.empty((n * rows, cols // 2), dtype=torch.uint8, device="cuda")
    s = torch.empty((n * rows, groups), dtype=DT[case["s_dt"]], device="cuda")
    z = torch.empty((n * rows, (groups + 1) // 2), dtype=torch.uint8, device="cuda") if case["zeros"] else None
    g, step = _gen(seed, 8), max(1, (1 << 26) // cols)
    for r in range(0, n * rows, step):
        m = min(step, n * rows - r)
        w = torch.zeros((m, groups * group), device="cuda")
        w[:, :cols] = torch.randn((m, cols), generator=g, device="cuda").mul_(0.02)
        w = w.view(m, groups, group)
        if case["zeros"]:
            low = w.amin(2, keepdim=True).clamp_(max=0.0)
            sc = w.amax(2, keepdim=True).clamp_(min=0.0).sub_(low).div_(15.0)
            zp = low.neg_().div_(sc).round_().clamp_(0.0, 15.0)
            pad = torch.zeros((m, 2 * z.shape[1]), dtype=torch.uint8, device="cuda")
            pad[:, :groups] = zp.squeeze(2).to(torch.uint8)
            z[r:r + m] = pad[:, 0::2] | (pad[:, 1::2] << 4)
        else:
            sc, zp = w.abs().amax(2, keepdim=True).div_(7.0), 8.0
        lv = w.div_(sc).round_().add_(zp).clamp_(0.0, 15.0).to(torch.uint8).view(m, -1)[:, :cols]
        q[r:r + m] = lv[:, 0::2] | (lv[:, 1::2] << 4)
        s[r:r + m] = sc.squeeze(2).to(s.dtype)
    return q, s, z


def _out_cols(case):
    return case["rows"] // 2 if case["swiglu"] else case["rows"]


# ----------------------------------------------------------------------------- prepare ----
def prepare(case, seed):
    op, dt = case["op"], case["dt"]
    st = dict(case=case, op=op)
    new = lambda *shape, t=DT[dt]: torch.zeros(shape, dtype=t, device="cuda")  # noqa: E731
    if op in ("forward", "backward"):
        T, H, K, n = case["T"], case["H"], case["K"], case["T"] * case["K"]
        idx, w = _routing(case, seed)
        st.update(idx=idx, w=w, ys=_normal(seed, 5, n, H, dt=dt))
        if op == "forward":
            st.update(x=_normal(seed, 4, T, H, dt=dt), add=_normal(seed, 6, T, H, dt=dt), xs=new(n, H), out=new(T, H),
                      plan=[new(case["NE"] + 1, t=torch.int32), new(n, t=torch.int32), new(n, t=torch.int32)])
        else:
            st.update(dout=_normal(seed, 4, T, H, dt=dt), dxs=_normal(seed, 6, n, H, dt=dt), dx=new(T, H), dys=new(n, H),
                      dw=new(T, K, t=torch.float32), plan=list(_sorted(idx, case["NE"])))
    elif op == "w4":
        st.update(x=_normal(seed, 4, case["T"], case["cols"], dt=dt), m=_w4(case, seed, 1), y=new(case["T"], _out_cols(case)))
    elif op == "experts":
        idx, _ = _routing(case, seed)
        n = idx.numel()
        st.update(x=_normal(seed, 4, case["T"], case["cols"], dt=dt), m=_w4(case, seed, case["NE"]), y=new(n, _out_cols(case)),
                  plan=list(_sorted(idx, case["NE"])))
        st["most"] = int(st["plan"][0].diff().max())          # rows of the busiest expert
    else:
        T, H, gate = case["T"], case["H"], case["gate"]
        shape, gt = {0: ((0,), "f32"), 1: ((H,), "f32"), 2: ((T,), "f32"), 3: ((T, H), dt)}[gate]
        st.update(h=_normal(seed, 4, T, H, dt=dt), y=_normal(seed, 5, T, H, dt=dt).mul_(0.5),
                  gate=torch.sigmoid(_normal(seed, 6, *shape)).to(DT[gt]),
                  post=_normal(seed, 7, H).mul_(0.1).add_(1.0), next=_normal(seed, 8, H).mul_(0.1).add_(1.0))
        if op == "norm":
            st.update(h2=new(T, H), xn=new(T, H))
        else:
            st.update(dh2=_normal(seed, 9, T, H, dt=dt), dxn=_normal(seed, 10, T, H, dt=dt), dh=new(T, H), dy=new(T, H),
                      dgate=torch.zeros_like(st["gate"]), dpost=new(H, t=torch.float32), dnext=new(H, t=torch.float32))
    torch.cuda.synchronize()          # the library works on a stream of its own
    return st


# ------------------------------------------------------------------------- plain forms ----
def _plain_forward(st):
    c, x, ys, w = st["case"], st["x"], st["ys"], st["w"]
    offsets, pair, row = _sorted(st["idx"], c["NE"])
    some = (pair >= 0)[:, None]
    xs = torch.where(some, x[(pair.clamp(min=0) // c["K"]).long()], 0)
    rows = row.view(c["T"], c["K"])
    part = torch.where(rows[..., None] >= 0, ys[rows.clamp(min=0).long()].float() * w[..., None], 0)
    out = (part.sum(1) + st["add"].float()).to(x.dtype)
    return dict(offsets=offsets, pair=pair, row=row, xs=xs, out=out)


def _plain_backward(st):
    c, dout, ys, w = st["case"], st["dout"], st["ys"], st["w"]
    _, pair, row = st["plan"]
    some, p = (pair >= 0)[:, None], pair.clamp(min=0).long()
    dys = torch.where(some, dout[p // c["K"]].float() * w.view(-1)[p][:, None], 0).to(dout.dtype)
    rows = row.view(c["T"], c["K"])
    keep, r = rows >= 0, rows.clamp(min=0).long()
    dw = torch.where(keep, (ys[r].float() * dout[:, None].float()).sum(2), 0)
    dx = torch.where(keep[..., None], st["dxs"][r].float(), 0).sum(1).to(dout.dtype)
    return dict(dys=dys, dw=dw, dx=dx)


def _dense(m, group):
    """Matrices of packed levels in 32 bits: [rows][cols]."""
    q, s, z = m
    lv = torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1).float()
    cols, groups = lv.shape[1], s.shape[1]
    zp = 8.0 if z is None else torch.stack((z & 15, z >> 4), -1).view(z.shape[0], -1)[:, :groups].float()
    spread = lambda v: v.repeat_interleave(group, 1)[:, :cols]  # noqa: E731
    return (lv - (zp if z is None else spread(zp))) * spread(s.float())


def _swiglu(y):
    g, u = y.chunk(2, -1)
    g = g.clamp(max=LIMIT)
    return g / (1.0 + torch.exp(-g)) * u.clamp(-LIMIT, LIMIT)


def _plain_w4(st):
    c, x = st["case"], st["x"]
    y = x.float() @ _dense(st["m"], c["group"]).T
    return (_swiglu(y) if c["swiglu"] else y).to(x.dtype)


def _plain_experts(st):
    c, x, (offsets, pair, _) = st["case"], st["x"], st["plan"]
    offsets, n, rows, cols = offsets.long(), pair.numel(), c["rows"], c["cols"]
    count = offsets.diff()
    busy = torch.argsort((count > 0).int(), descending=True, stable=True)[:min(n, c["NE"])]     # experts with rows first
    q, s, z = (None if v is None else v.view(c["NE"], rows, -1)[busy].view(len(busy) * rows, -1) for v in st["m"])
    W = _dense((q, s, z), c["group"]).view(len(busy), rows, cols)
    at = torch.arange(st["most"], device=x.device)
    p = (offsets[busy][:, None] + at).clamp(max=n - 1)
    xe = x[pair[p].clamp(min=0).long() // c["K"]].float().transpose(1, 2).contiguous()
    y = torch.bmm(W, xe).transpose(1, 2)
    keep = at < count[busy][:, None]
    out = torch.zeros((n, rows), device=x.device)
    out.index_add_(0, p.view(-1), torch.where(keep[..., None], y, 0).reshape(-1, rows))
    return (_swiglu(out) if c["swiglu"] else out).to(x.dtype)


def _gates(st):
    """The gate as it applies to [T][H]."""
    kind, g = st["case"]["gate"], st["gate"].float()
    return 1.0 if kind == 0 else g[:, None] if kind == 2 else g


def _plain_norm(st):
    h, y = st["h"].float(), st["y"].float()
    u = y * torch.rsqrt(y.square().mean(1, keepdim=True) + EPS) * st["post"]
    h2 = h + SCALE * _gates(st) * u
    xn = h2 * torch.rsqrt(h2.square().mean(1, keepdim=True) + EPS) * st["next"]
    return dict(h2=h2.to(st["h"].dtype), xn=xn.to(st["h"].dtype))


def _plain_norm_grad(st):
    h, y, dh2, dxn = (st[k].float() for k in ("h", "y", "dh2", "dxn"))
    t, kind, gate = st["h"].dtype, st["case"]["gate"], _gates(st)
    ry = torch.rsqrt(y.square().mean(1, keepdim=True) + EPS)
    yh = y * ry
    u = yh * st["post"]
    h2 = h + SCALE * gate * u
    rh = torch.rsqrt(h2.square().mean(1, keepdim=True) + EPS)
    hh, v = h2 * rh, dxn * st["next"]
    dh = dh2 + rh * (v - hh * (v * hh).mean(1, keepdim=True))
    du, dg = SCALE * gate * dh, SCALE * u * dh
    v2 = du * st["post"]
    dy = ry * (v2 - yh * (v2 * yh).mean(1, keepdim=True))
    dgate = [st["gate"], dg.sum(0), dg.sum(1), dg][kind].to(st["gate"].dtype)
    return dict(dh=dh.to(t), dy=dy.to(t), dgate=dgate, dpost=(du * yh).sum(0), dnext=(dxn * hh).sum(0))


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
    dt = CODE[DT[c["dt"]]]
    if "plan" in st:
        plan = G.G53hSort(c["T"], c["K"], c["NE"], *[t.data_ptr() for t in st["plan"]])
    if st["op"] == "forward":
        return [(L.g53h_sort_tokens, (C.byref(plan), p("idx"))),
                (L.g53h_sorted_dispatch, (p("xs"), p("x"), dt, c["H"], C.byref(plan))),
                (L.g53h_sorted_combine, (p("out"), p("ys"), p("w"), p("add"), dt, c["H"], C.byref(plan)))], dict(
                    offsets=st["plan"][0], pair=st["plan"][1], row=st["plan"][2], xs=st["xs"], out=st["out"])
    if st["op"] == "backward":
        return [(L.g53h_sorted_combine_grad, (p("dys"), p("dw"), p("dout"), p("ys"), p("w"), dt, c["H"], C.byref(plan))),
                (L.g53h_sorted_dispatch_grad, (p("dx"), p("dxs"), dt, c["H"], C.byref(plan)))], {
                    k: st[k] for k in ("dys", "dw", "dx")}
    if st["op"] in ("w4", "experts"):
        q, s, z = st["m"]
        m = G.G53hW4(q.data_ptr(), s.data_ptr(), _ptr(z), c["rows"], c["cols"], c["group"], CODE[s.dtype])
        limit = LIMIT if c["swiglu"] else 0.0
        if st["op"] == "w4":
            return [(L.g53h_mm_w4, (p("y"), p("x"), dt, c["T"], C.byref(m), limit))], st["y"]
        return [(L.g53h_sorted_mm_w4, (p("y"), p("x"), dt, 1, C.byref(plan), C.byref(m), limit))], st["y"]
    b = G.G53hBlockNorm(c["T"], c["H"], dt, c["gate"], EPS, SCALE, p("post"), p("next"), p("gate"))
    if st["op"] == "norm":
        return [(L.g53h_block_norm, (p("h2"), p("xn"), p("h"), p("y"), C.byref(b)))], {k: st[k] for k in ("h2", "xn")}
    return [(L.g53h_block_norm_grad, (p("dh"), p("dy"), p("dgate"), p("dpost"), p("dnext"), p("dh2"), p("dxn"), p("h"),
                                      p("y"), C.byref(b)))], {k: st[k] for k in ("dh", "dy", "dgate", "dpost", "dnext")}


def run(state):
    if not own:
        return {"forward": _plain_forward, "backward": _plain_backward, "w4": _plain_w4, "experts": _plain_experts,
                "norm": _plain_norm, "norm_grad": _plain_norm_grad}[state["op"]](state)
    if "calls" not in state:
        state["calls"] = _calls(state)
    calls, out = state["calls"]
    for f, args in calls:
        if f(*args):
            raise RuntimeError(_lib().lib().g53h_error().decode())
    return out


# -------------------------------------------------------------------------------- work ----
def work(case):
    op, T, b = case["op"], case["T"], 4 if case["dt"] == "f32" else 2
    if op in ("forward", "backward"):
        H, n, routed = case["H"], T * case["K"], (T - case["pad"]) * case["K"]
        if op == "forward":
            return {"bytes": 12 * n + 4 * case["NE"] + 4 * routed + (2 * routed + 3 * T) * H * b, "flops": (2 * routed + T) * H}
        return {"bytes": 8 * n + 4 * n + 4 * routed + (3 * routed + 2 * T) * H * b, "flops": 4 * routed * H}
    if op in ("norm", "norm_grad"):
        H, kind, grad = case["H"], case["gate"], op == "norm_grad"
        gate = [0, 4 * H, 4 * T, b * T * H][kind]
        return {"bytes": (6 if grad else 4) * T * H * b + (2 if grad else 1) * (gate + 8 * H), "flops": (30 if grad else 10) * T * H}
    rows, cols = case["rows"], case["cols"]
    groups = -(-cols // case["group"])
    one = rows * (cols // 2 + groups * (4 if case["s_dt"] == "f32" else 2) + (groups + 1) // 2 * case["zeros"])
    if op == "w4":
        return {"bytes": one + T * (cols + _out_cols(case)) * b, "flops": 2 * T * rows * cols}
    n, NE = T * case["K"], case["NE"]
    busy = NE * (1.0 - (1.0 - case["K"] / NE) ** T) if case["K"] < NE else NE      # at even popularity
    return {"bytes": busy * one + 8 * n + 4 * NE + (T * cols + n * _out_cols(case)) * b, "flops": 2 * n * rows * cols}


# ------------------------------------------------------------------------------- exact ----
def _wide(m, group):
    """Matrices in 64 bits, column by column of the packed bytes."""
    q, s, z = m
    groups = s.shape[1]
    of = torch.arange(2 * q.shape[1], device=q.device) // group
    w = torch.empty((q.shape[0], 2 * q.shape[1]), dtype=torch.float64, device=q.device)
    w[:, 0::2], w[:, 1::2] = (q % 16).double(), (q // 16).double()
    if z is None:
        w -= 8
    else:
        zp = torch.empty((q.shape[0], 2 * z.shape[1]), dtype=torch.float64, device=q.device)
        zp[:, 0::2], zp[:, 1::2] = (z % 16).double(), (z // 16).double()
        w -= zp[:, :groups][:, of]
    return w.mul_(s.double()[:, of])


def _act64(y, swiglu):
    if not swiglu:
        return y
    half = y.shape[-1] // 2
    g, u = y[..., :half].clamp(max=LIMIT), y[..., half:].clamp(min=-LIMIT, max=LIMIT)
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    st = prepare(case, seed)
    op, T = case["op"], case["T"]
    if op == "w4":
        return _act64(st["x"].double() @ _wide(st["m"], case["group"]).T, case["swiglu"])
    if op in ("norm", "norm_grad"):
        return _exact_norm(st, op == "norm_grad")
    NE, K, idx = case["NE"], case["K"], st["idx"] if op != "experts" else _routing(case, seed)[0]
    lists = [torch.nonzero(idx == e, as_tuple=True) for e in range(NE)]           # (token, place) of every expert, in order
    if op == "experts":
        ys = torch.zeros((T * K, _out_cols(case)), dtype=torch.float64, device="cuda")
        at, rows = 0, case["rows"]
        for e, (t, _) in enumerate(lists):
            if len(t):
                mine = [None if v is None else v[e * rows:(e + 1) * rows] for v in st["m"]]
                ys[at:at + len(t)] = _act64(st["x"][t].double() @ _wide(mine, case["group"]).T, case["swiglu"])
                at += len(t)
        return ys
    t, j = (torch.cat([p[k] for p in lists]) for k in (0, 1))                     # of every sorted row
    m, w, ys = len(t), st["w"].double(), st["ys"].double()
    if op == "forward":
        xs, out = torch.zeros_like(ys), st["add"].double()
        xs[:m] = st["x"].double()[t]
        out.index_add_(0, t, ys[:m] * w[t, j, None])
        return dict(offsets=None, pair=None, row=None, xs=xs, out=out)
    dout, dys, dw = st["dout"].double(), torch.zeros_like(ys), torch.zeros_like(w)
    dys[:m] = dout[t] * w[t, j, None]
    dw[t, j] = torch.linalg.vecdot(dout[t], ys[:m])
    dx = torch.zeros_like(dout).index_add_(0, t, st["dxs"][:m].double())
    return dict(dys=dys, dw=dw, dx=dx)


def _exact_norm(st, grad):
    """The block's norms in 64 bits; the gradients by differentiating them."""
    kind = st["case"]["gate"]
    h, y, gate, post, nxt = (st[k].double().requires_grad_(grad) for k in ("h", "y", "gate", "post", "next"))
    norm = lambda v, gain: v / torch.sqrt((v * v).mean(dim=-1, keepdim=True) + EPS) * gain  # noqa: E731
    u = norm(y, post)
    h2 = h + SCALE * (u if kind == 0 else u * (gate.unsqueeze(1) if kind == 2 else gate))
    xn = norm(h2, nxt)
    if not grad:
        return dict(h2=h2, xn=xn)
    loss = (h2 * st["dh2"].double()).sum() + (xn * st["dxn"].double()).sum()
    wrt = [h, y, post, nxt] + ([gate] if kind else [])
    dh, dy, dpost, dnext, *rest = torch.autograd.grad(loss, wrt)
    return dict(dh=dh, dy=dy, dgate=rest[0] if rest else torch.zeros_like(gate), dpost=dpost, dnext=dnext)
