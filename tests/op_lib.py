"""Helpers of the tests of the operators beside the layer: element types on the host, device
buffers with a guard behind their end, and the operators in 64 bits."""
import numpy as np

import glm53h
from glm53h import DevBuf, check

F32, BF16, F16 = glm53h.G53H_F32, glm53h.G53H_BF16, glm53h.G53H_F16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}        # half a step, relative
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}     # and below the normal range
NP = {F32: np.float32, BF16: np.uint16, F16: np.float16}
GUARD = 64


def enc(a, dt):
    """Values to the bits of type dt, to nearest, ties to even."""
    a = np.asarray(a, np.float32)
    if dt != BF16:
        return a.astype(NP[dt])
    u = a.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7fc0), r)


def dec(b, dt):
    """Bits of type dt to 64-bit values."""
    if dt == BF16:
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


class Buf:
    """A device array of type `kind` (an element type or a numpy dtype) with a guard behind it, `shift` bytes off
    the allocation's alignment."""

    def __init__(self, a, kind=None, shift=0):
        self.dt = kind
        raw = enc(a, kind) if kind is not None else np.ascontiguousarray(a)
        self.shape, self.dtype, self.n, self.shift = raw.shape, raw.dtype, raw.nbytes, shift
        self.buf = DevBuf(shift + self.n + GUARD)
        self.buf.upload(np.concatenate([np.full(shift, 0xa5, np.uint8), raw.reshape(-1).view(np.uint8),
                                        np.full(GUARD, 0xa5, np.uint8)]))
        self.ptr = self.buf.ptr + shift

    @classmethod
    def out(cls, shape, kind, shift=0, fill=77.0):
        if kind in NP:
            return cls(np.full(shape, fill, np.float32), kind, shift)
        return cls(np.full(shape, int(fill), kind), None, shift)

    def get(self):
        """The bits; the guards are checked."""
        raw = self.buf.download(np.uint8)
        assert (raw[:self.shift] == 0xa5).all() and (raw[self.shift + self.n:] == 0xa5).all(), "written outside"
        return raw[self.shift:self.shift + self.n].view(self.dtype).reshape(self.shape)

    def val(self):
        b = self.get()
        return dec(b, self.dt) if self.dt is not None else b


def routing(rng, T, K, NE, drop=0.0):
    idx = rng.integers(0, NE, (T, K)).astype(np.int32)
    idx[rng.random((T, K)) < drop] = -1
    return idx


def sorted_plan(idx, NE):
    """offsets, pair, row by a stable sort on the host."""
    flat = idx.reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < NE), flat, NE)
    order = np.argsort(key, kind="stable")
    offsets = np.searchsorted(key[order], np.arange(NE + 1))
    pair = np.where(np.arange(flat.size) < offsets[NE], order, -1)
    row = np.empty(flat.size, np.int64)
    row[order] = np.arange(flat.size)
    row[key == NE] = -1
    return offsets.astype(np.int32), pair.astype(np.int32), row.astype(np.int32)


class Plan:
    """A plan on the device, filled by the library from idx (or from the host, given = True)."""

    def __init__(self, idx, NE, given=False):
        T, K = idx.shape
        self.idx = Buf(idx)
        arrays = sorted_plan(idx, NE) if given else [np.full(n, -7, np.int32) for n in (NE + 1, T * K, T * K)]
        self.bufs = [Buf(a) for a in arrays]
        self.c = glm53h.G53hSort(T, K, NE, *[b.ptr for b in self.bufs])
        if not given:
            check(glm53h.lib().g53h_sort_tokens(self.c, self.idx.ptr), "g53h_sort_tokens")

    def arrays(self):
        return [b.get() for b in self.bufs]


def close(got, want, tol, what=""):
    """|got - want| <= tol elementwise, the same NaN and infinities."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True), what
    off = np.abs(got - want)[fine] - np.broadcast_to(tol, want.shape)[fine]
    assert not off.size or (off <= 0).all(), (what, "by", off.max(), "over", int((~(off <= 0)).sum()), "of", off.size)


# ---------------------------------------------------------------------- 4-bit matrices ----
class W4:
    """n stacked matrices of 4-bit levels, on the host (wide: 64-bit values [n][rows][cols]) and on the device."""

    def __init__(self, rng, n, rows, cols, group, s_dt, zeros, exact=False):
        gs = -(-cols // group)
        lv = rng.integers(0, 16, (n, rows, cols))
        s = 2.0 ** rng.integers(-2, 2, (n, rows, gs)) if exact else rng.uniform(0.002, 0.02, (n, rows, gs))
        s = dec(enc(s, s_dt), s_dt)
        z = rng.integers(0, 16, (n, rows, gs)) if zeros else np.full((n, rows, gs), 8)
        self.s = np.repeat(s, group, 2)[:, :, :cols]
        self.lv, self.z = lv, np.repeat(z, group, 2)[:, :, :cols]
        self.wide = (lv - self.z) * self.s
        self.group = min(group, cols)
        zp = np.zeros((n, rows, gs + gs % 2), np.uint8)
        zp[..., :gs] = z
        self.w_d = Buf((lv[..., 0::2] | (lv[..., 1::2] << 4)).astype(np.uint8))
        self.s_d = Buf(s, s_dt)
        self.z_d = Buf(zp[..., 0::2] | (zp[..., 1::2] << 4)) if zeros else None
        self.c = glm53h.G53hW4(self.w_d.ptr, self.s_d.ptr, self.z_d.ptr if zeros else None, rows, cols, group, s_dt)

    def product(self, x, e=0):
        """x [T][cols] times matrix e, and what its fp32 sums may be off: every level enters as 16 + level and the
        surplus comes off per group, so partial sums of a group reach (16 + 15) sum |x| twice; a group has `group`
        products and as many in the surplus, added in an unknown order, then groups and partial sums of the waves
        are added (at most groups + 16 more). Every addition is off by at most 2^-24 of its partial sum."""
        y = x @ self.wide[e].T
        depth = 2 * self.group + -(-x.shape[1] // self.group) + 24
        return y, depth * 2.0 ** -24 * 62.0 * (np.abs(x) @ self.s[e].T)


def swiglu(y, limit):
    g, u = np.split(y, 2, -1)
    g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
    return g / (1.0 + np.exp(-g)) * u


# --------------------------------------------------------------------------- the norms ----
def block(h, y, post, nxt, gate, kind, scale, eps):
    """h2 and xn in 64 bits; post None: no norm of y, nxt None: no xn."""
    u = y if post is None else y / np.sqrt((y * y).mean(1, keepdims=True) + eps) * post
    g = 1.0 if kind == 0 else gate[:, None] if kind == 2 else gate
    h2 = h + scale * g * u
    return h2, None if nxt is None else h2 / np.sqrt((h2 * h2).mean(1, keepdims=True) + eps) * nxt
