"""The operators of include/b200.h restated in 64 bits, and how far a kernel may be from them.

Bounds follow the roundings: a value stored in a type is off by at most half a step of it (`EPS[prec] / 2` relative); 16-bit
weights and score gradients are rounded once more before they are multiplied, which moves a sum of products by at most
EPS / 2 times the sum of their sizes; sums in single precision, exp2 and tanh are given 2^-15 of that sum: scores of up to
100 times a few 2^-23 each.  Half weights below the normal range are off by 2^-25 of the largest.
"""
import numpy as np

from ocannl_b200 import backend as bk
from ocannl_b200.low_level import Tnode
from ocannl_b200.workloads import load, store

EPS = {"single": 2.0 ** -23, "half": 2.0 ** -10, "bfloat16": 2.0 ** -7}
ARITH = 2.0 ** -15


def rounded(prec, a):
    """The values that `a` has once stored in `prec`, in 64 bits."""
    return load(prec, store(prec, np.asarray(a, np.float32))).astype(np.float64)


class Nodes:
    """A context over named arrays; outputs start as NaN (or -1)."""

    def __init__(self, device, arrays, packing="aligned", odd_first=False):
        """arrays: {name: (prec, dims, values or None)}."""
        self.device = device
        tns, i = [], 0
        if odd_first:
            tns.append(Tnode(1, "odd", "half", (3,)))
        for name, (prec, dims, _) in arrays.items():
            tns.append(Tnode(len(tns) + 1, name, prec, tuple(dims)))
        if packing == "aligned":
            self.context = bk.Context(device).allocate(tns)
        else:
            # one node behind the other, aligned to its element alone
            where, sizes = bk.plan_pool_segments([(t.size_in_bytes, {"single": 4, "int32": 4}.get(t.prec, 2)) for t in tns])
            pool = device.alloc_pool(max(sizes[0], 1))
            self.context = bk.Context(device, {t.ident: (pool, off, t) for t, (_, off) in zip(tns, where)})
        self.precs = {n: p for n, (p, _, _) in arrays.items()}
        for name, (prec, dims, values) in arrays.items():
            if 0 in dims:
                continue
            if values is None:
                values = np.full(dims, -1, np.int32) if prec == "int32" else np.full(dims, np.nan, np.float32)
            self.context.from_host(name, np.asarray(values, np.int32) if prec == "int32" else store(prec, np.asarray(values, np.float32)))

    def read(self, name):
        if 0 in self.context.arrays[name][2].dims:
            return np.zeros(self.context.arrays[name][2].dims)
        return load(self.precs[name], self.context.to_host(name)).astype(np.float64)

    def free(self):
        self.device.await_()
        for p in {p for p, _, _ in self.context.arrays.values()}:
            self.device.free_pool(p)


# ------------------------------------------------------------------ layer norm
def layer_norm(x, gamma, beta, residual=None, eps=1e-5):
    h = x if residual is None else x + residual
    mean = h.mean(-1)
    rstd = 1.0 / np.sqrt(((h - mean[..., None]) ** 2).mean(-1) + eps)
    u = (h - mean[..., None]) * rstd[..., None]
    return u * gamma + beta, h, mean, rstd, u


def layer_norm_grad(x, mean, rstd, gamma, dy, d_total=None):
    u = (x - mean[..., None]) * rstd[..., None]
    g = dy * gamma
    dx = rstd[..., None] * (g - g.mean(-1, keepdims=True) - u * (g * u).mean(-1, keepdims=True))
    flat = lambda a: a.reshape(-1, a.shape[-1])  # noqa: E731
    return (dx if d_total is None else dx + d_total), (flat(dy * u)).sum(0), flat(dy).sum(0), u, g


# ------------------------------------------------------------------ rotary
def rotary(x, frequencies, positions, layout="half", inverse=False, magnitude=1.0):
    m = len(frequencies)
    angle = positions[:, :, None, None].astype(np.float64) * np.asarray(frequencies, np.float64)
    angle = -angle if inverse else angle
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    y = x.copy()
    i, j = (np.arange(m), np.arange(m) + m) if layout == "half" else (2 * np.arange(m), 2 * np.arange(m) + 1)
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    return y


# ------------------------------------------------------------------ attention
def visible(b, s, n, mask="causal", prefix=None, qdoc=None, kdoc=None, lengths=None):
    """[b, s, n] of truth values, and the positions [b, s] of the queries."""
    length = np.full(b, n) if lengths is None else np.clip(np.asarray(lengths, np.int64), 0, n)
    pos = (length - s)[:, None] + np.arange(s)
    j = np.arange(n)
    seen = np.broadcast_to((j < length[:, None])[:, None, :], (b, s, n)).copy()
    if mask == "causal":
        seen &= j <= pos[:, :, None]
    if mask == "prefix":
        seen &= (j <= pos[:, :, None]) | (j < np.asarray(prefix)[:, None, None])
    if qdoc is not None:
        seen &= (qdoc[:, :, None] == kdoc[:, None, :]) & (qdoc[:, :, None] >= 0)
    return seen, pos


def _masked(a, seen):
    return np.where(seen, a, 0.0)


def attention(q, k, v, seen, pos, scale, cap=0.0, slopes=None):
    """out, lse, and the bound's sums: sum_j p_j |v_j|, sum_j |v_j| over the visible keys."""
    b, s, h, d = q.shape
    n, hk = k.shape[1:3]
    out, lse = np.zeros_like(q), np.full((b, h, s), -np.inf)
    size, flat = np.zeros_like(q), np.zeros_like(q)
    with np.errstate(invalid="ignore", over="ignore"):
        for i in range(b):
            for g in range(h):
                kk, vv = k[i, :, g // (h // hk)], v[i, :, g // (h // hk)]
                z, _ = _scores(q[i, :, g], kk, pos[i], scale, cap, 0.0 if slopes is None else slopes[g])
                for r in range(s):
                    w = seen[i, r]
                    if not w.any():
                        continue
                    zr = z[r, w]
                    top = zr.max()
                    e = np.exp(zr - top)
                    p = e / e.sum()
                    out[i, r, g] = p @ vv[w]
                    size[i, r, g] = p @ np.abs(vv[w])
                    flat[i, r, g] = np.abs(vv[w]).sum(0)
                    lse[i, g, r] = top + np.log(e.sum())
    return out, lse, size, flat


def _scores(q, k, pos, scale, cap, slope):
    x = q @ k.T * scale
    t = np.tanh(x / cap) if cap else np.zeros_like(x)
    c = cap * t if cap else x
    return c - slope * np.abs(pos[:, None] - np.arange(k.shape[0])), 1.0 - t * t


def attention_grad(q, k, v, out, lse, d_out, seen, pos, scale, cap=0.0, slopes=None, prec="single"):
    """The gradients and bounds on how far each may be, as (value, bound) pairs."""
    b, s, h, d = q.shape
    n, hk = k.shape[1:3]
    e = EPS[prec] / 2 if prec != "single" else 0.0
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    bq, bk_, bv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    with np.errstate(invalid="ignore", over="ignore"):
        for i in range(b):
            for g in range(h):
                rows, keys = seen[i].any(1), seen[i].any(0)
                gk = g // (h // hk)
                kk, vv = np.where(keys[:, None], k[i, :, gk], 0.0), np.where(keys[:, None], v[i, :, gk], 0.0)
                qq, do, oo = (np.where(rows[:, None], a[i, :, g], 0.0) for a in (q, d_out, out))
                z, t2 = _scores(qq, kk, pos[i], scale, cap, 0.0 if slopes is None else slopes[g])
                p = _masked(np.exp(z - np.where(np.isneginf(lse[i, g]), 0.0, lse[i, g])[:, None]), seen[i])
                dp, delta = do @ vv.T, (do * oo).sum(1)
                ds = p * (dp - delta[:, None]) * t2
                size = np.abs(do) @ np.abs(vv).T + (np.abs(do) * np.abs(oo)).sum(1)[:, None]
                # rounded once; computed from p (ARITH) and from two sums of products in single precision
                ds_off = np.abs(ds) * (e + ARITH) + p * (ARITH * np.abs(dp - delta[:, None]) * (1.0 - t2) + 2.0 ** -20 * size)
                p_off = p * (e + ARITH)
                if prec == "half":
                    # below the normal range: weights, and gradients scaled to at least 2^-6 of the largest |d_out| |v|
                    p_off = p_off + 2.0 ** -25 * seen[i]
                    ds_off = ds_off + 2.0 ** -25 * 2.0 ** -5 * np.linalg.norm(d_out[i][rows], axis=-1).max(initial=0.0) * seen[i]
                dq[i, :, g] += scale * ds @ kk
                bq[i, :, g] += scale * ds_off @ np.abs(kk)
                dk[i, :, gk] += scale * ds.T @ qq
                bk_[i, :, gk] += scale * ds_off.T @ np.abs(qq)
                dv[i, :, gk] += p.T @ do
                bv[i, :, gk] += p_off.T @ np.abs(do)
    half = EPS[prec] / 2
    return [(a, c + half * np.abs(a) + (2.0 ** -25 if prec == "half" else 1e-30)) for a, c in ((dq, bq), (dk, bk_), (dv, bv))]


def within(got, want, bound, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), "%s: undefined values in other places" % what
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), "%s: infinities differ" % what
    bound = np.broadcast_to(bound, want.shape)
    err = np.abs(got - want)[fine]
    worst = (err / np.maximum(bound[fine], 1e-300)).max(initial=0.0)
    assert worst <= 1.0, "%s: off by %.3g times what the roundings allow" % (what, worst)
