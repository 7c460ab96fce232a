"""The operators over a paged cache and the choice of tokens restated in 64 bits, and how far a kernel may be from them.

Bounds follow the roundings: a value stored in a type is off by at most half a step of it (`EPS[prec] / 2` relative; codes of 8 bits: 2^-4, or half of the
least step 2^-9 of their scale); cosines and sines in single precision are off by 2^-22 (sincospi: two units in the last place, the angle's step 2^-33 of a
turn), and the turn's products and their sum by 2^-24 each: 2^-21 of |a| + |b| together.  Attention: as in operators_reference, with weights of 11
bits beside codes.
"""
import numpy as np

from ocannl_b200 import backend as bk
from ocannl_b200.low_level import Tnode
from ocannl_b200.workloads import load, store
from tests.operators_reference import ARITH, EPS, rounded, within  # noqa: F401


def _table():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


E4M3 = _table()


def decode(codes):
    return E4M3[np.asarray(codes, np.uint8)]


def encode(x):
    """The nearest code, ties to even; what is undefined stays so."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        _, e = np.frexp(x)
        step = np.ldexp(1.0, np.maximum(e - 4, -9))
        y = np.minimum(np.abs(np.round(x / step) * step), 448.0)
    codes = np.searchsorted(E4M3[:127], np.where(np.isnan(y), 0.0, y))
    return np.where(np.isnan(x), 127, codes | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def exponent(amax):
    """The least e >= -40 with amax <= 448 * 2^e."""
    e = -40
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


class Nodes:
    """A context over named arrays (byte: codes); outputs start as NaN (int32: -7, byte: 0x55)."""

    def __init__(self, device, arrays, packing="aligned"):
        self.device = device
        tns = [Tnode(i + 1, name, prec, tuple(dims)) for i, (name, (prec, dims, _)) in enumerate(arrays.items())]
        if packing == "aligned":
            self.context = bk.Context(device).allocate(tns)
        else:
            # one node behind the other, aligned to its element alone, an odd one first
            sizes = {"single": 4, "int32": 4, "byte": 1}
            where, total = bk.plan_pool_segments([(2, 2)] + [(t.size_in_bytes, sizes.get(t.prec, 2)) for t in tns])
            pool = device.alloc_pool(max(total[0], 1))
            self.context = bk.Context(device, {t.ident: (pool, off, t) for t, (_, off) in zip(tns, where[1:])})
        self.precs = {n: p for n, (p, _, _) in arrays.items()}
        for name, (prec, dims, values) in arrays.items():
            if 0 not in dims:
                self.write(name, np.full(dims, {"int32": -7, "byte": 0x55}.get(prec, np.nan)) if values is None else values)

    def write(self, name, values):
        prec = self.precs[name]
        if prec in ("int32", "byte"):
            a = np.asarray(values, np.int32 if prec == "int32" else np.uint8)
        else:
            a = store(prec, np.asarray(values, np.float32))
        self.context.from_host(name, np.ascontiguousarray(a))

    def raw(self, name):
        return self.context.to_host(name)

    def read(self, name):
        if 0 in self.context.arrays[name][2].dims:
            return np.zeros(self.context.arrays[name][2].dims)
        a = self.raw(name)
        return a if self.precs[name] in ("int32", "byte") else load(self.precs[name], a).astype(np.float64)

    def free(self):
        self.device.await_()
        for p in {p for p, _, _ in self.context.arrays.values()}:
            self.device.free_pool(p)


def rows_of(lengths, starts, tokens, batch):
    """(rows, position of the first) of each sequence."""
    res = []
    for b in range(batch):
        if starts is None:
            lo, hi = b * (tokens // batch), (b + 1) * (tokens // batch)
        else:
            lo = min(max(int(starts[b]), 0), tokens)
            hi = min(max(int(starts[b + 1]), lo), tokens)
        res.append((range(lo, hi), max(int(lengths[b]), 0) - (hi - lo)))
    return res


def place(table, pages, page, b, j):
    """(page, slot) of token j of sequence b, or None."""
    if j < 0 or j // page >= table.shape[1]:
        return None
    p = int(table[b, j // page])
    return (p, j % page) if 0 <= p < pages else None


def turned(x, frequencies, position, layout="half", magnitude=1.0):
    """x [heads, d] turned by a position, and |a| + |b| of every element's pair."""
    m = len(frequencies)
    angle = np.float64(position) * np.asarray(frequencies, np.float64)
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    y, size = x.copy(), np.zeros_like(x)
    i, j = (np.arange(m), np.arange(m) + m) if layout == "half" else (2 * np.arange(m), 2 * np.arange(m) + 1)
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    size[..., i] = size[..., j] = (np.abs(a) + np.abs(b)) * abs(magnitude)
    return y, size


def append(x, prec, table, lengths, starts, page, frequencies=(), layout="half", magnitude=1.0, positions=None):
    """x: {"k", "v", optional "q"; "k_cache", "v_cache" as values or codes, "k_scale", "v_scale"}.  {node: (values, bounds)} of q_out and of caches of
    the nodes' type; of codes {node: codes} and {scale: values}, and the bounds of the values that the codes stand for."""
    coded = "k_scale" in x
    n, hk, d = x["k"].shape
    pages, batch = x["k_cache"].shape[0], table.shape[0]
    half = EPS[prec] / 2
    res = {g: x[g].copy() for g in ("k_cache", "v_cache")}
    off = {g: np.zeros(x[g].shape) for g in ("k_cache", "v_cache")}
    if "q" in x:
        res["q_out"], off["q_out"] = np.full(x["q"].shape, np.nan), np.zeros(x["q"].shape)
    if coded:
        res.update({g: np.array(x[g], np.float64) for g in ("k_scale", "v_scale")})
    received = {}
    for b, (rows, pos0) in enumerate(rows_of(lengths, starts, n, batch)):
        for i, r in enumerate(rows):
            pos = pos0 + i
            by = pos if positions is None else int(positions[r])
            if "q" in x:
                y, size = turned(x["q"][r], frequencies, by, layout, magnitude)
                res["q_out"][r], off["q_out"][r] = y, half * np.abs(y) + 2.0 ** -21 * size
            at = place(table, pages, page, b, pos)
            if at is None:
                continue
            for g in "kv":
                y, size = turned(x[g][r], frequencies, by, layout, magnitude) if g == "k" else (x[g][r], np.zeros((hk, d)))
                if coded:
                    received.setdefault((at[0], g), []).append((at[1], y, size))
                else:
                    res[g + "_cache"][at[0], :, at[1]] = y
                    off[g + "_cache"][at[0], :, at[1]] = half * np.abs(y) + 2.0 ** -21 * size
    for (p, g), new in received.items():
        first = min(s for s, _, _ in new)
        for h in range(hk):
            fine = [np.abs(np.where(np.abs(y[h]) <= 448.0 * 2.0 ** 40, y[h], 0.0)).max(initial=0.0) for _, y, _ in new]
            before, scale = float(x[g + "_scale"][p, h]), 2.0 ** exponent(max(fine))
            if first:
                scale = max(scale, before)
                if scale > before:
                    old = decode(x[g + "_cache"][p, h, :first]) * before
                    res[g + "_cache"][p, h, :first] = encode(old / scale)
                    off[g + "_cache"][p, h, :first] = np.where(np.isnan(old), 0.0, scale * 2.0 ** -10)
            res[g + "_scale"][p, h] = scale
            for s, y, size in new:
                v = np.where(np.abs(y[h]) <= 448.0 * 2.0 ** 40, y[h], np.nan)
                res[g + "_cache"][p, h, s] = encode(v / scale)
                off[g + "_cache"][p, h, s] = np.where(np.isnan(v), 0.0, np.maximum(2.0 ** -4 * np.abs(v), scale * 2.0 ** -10) + 2.0 ** -21 * size[h])
    return res, off


def attention(q, k_cache, v_cache, table, lengths, starts, page, prec, k_scale=None, v_scale=None, window=0, sinks=0, cap=0.0, slopes=None, scale=None):
    """(out, lse, bounds of both); rows of no sequence: NaN."""
    n, h, d = q.shape
    pages, hk = k_cache.shape[:2]
    coded = k_scale is not None
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    out, lse, off, lse_off = np.full(q.shape, np.nan), np.full((n, h), np.nan), np.zeros(q.shape), np.zeros((n, h))
    half = EPS[prec] / 2
    of_weights = 0.0 if prec == "single" else 2.0 ** -11 if coded else half
    for b, (rows, pos0) in enumerate(rows_of(lengths, starts, n, table.shape[0])):
        if not len(rows):
            continue
        rows, pos = np.array(rows), pos0 + np.arange(len(rows))[:, None]
        j = np.arange(max(0, min(int(pos[-1, 0]) + 1, table.shape[1] * page)))
        p = table[b, j // page]
        there = (p >= 0) & (p < pages)
        seen = (j <= pos) & there
        if window:
            seen &= (j > pos - window) | (j < sinks)
        used = seen.any(0)
        p, slot = np.where(used, p, 0), j % page
        for g in range(hk):
            k, v = k_cache[p, g, slot], v_cache[p, g, slot]
            if coded:
                k, v = decode(k) * k_scale[p, g][:, None], decode(v)
            k, v = np.where(used[:, None], k, 0.0), np.where(used[:, None], v, 0.0)
            # (rows below the largest weight of a half: sizes of all values that a row sees)
            fine = np.where(np.isfinite(v), v, 0.0)
            odd = np.flatnonzero(~np.isfinite(v).all(1))       # (added below, for the rows that see them)
            flat = seen @ np.abs(fine)
            if coded:
                flat = flat * np.where(seen, v_scale[p, g], 0.0).max(1, initial=0.0)[:, None]
                by = np.where(used, v_scale[p, g], 0.0)[:, None]
                v, fine = v * by, fine * by
            for hh in range(g * (h // hk), (g + 1) * (h // hk)):
                with np.errstate(all="ignore"):
                    z = q[rows, hh] @ k.T * scale
                    z = cap * np.tanh(z / cap) if cap else z
                    z = z - (0.0 if slopes is None else slopes[hh]) * (pos - j)
                    z = np.where(seen, z, -np.inf)
                    top = z.max(1, initial=-np.inf, keepdims=True)
                    e = np.where(seen, np.exp(z - np.where(np.isneginf(top), 0.0, top)), 0.0)
                    total = e.sum(1, keepdims=True)
                    w = e / np.where(total == 0.0, 1.0, total)
                    out[rows, hh], lse[rows, hh] = w @ fine, (top + np.log(total))[:, 0]
                    for i in odd:
                        at = np.flatnonzero(seen[:, i])
                        out[rows[at], hh] += w[at, i][:, None] * np.where(np.isfinite(v[i]), 0.0, v[i])
                size = w @ np.abs(fine)
                off[rows, hh] = half * np.abs(out[rows, hh]) + (of_weights + ARITH) * size + (2.0 ** -25 * (flat + 1) if prec == "half" or (coded and prec != "single") else 1e-30)
                lse_off[rows, hh] = np.where(np.isfinite(lse[rows, hh]), ARITH * (1 + np.abs(np.where(np.isfinite(lse[rows, hh]), lse[rows, hh], 0.0))), 0.0)
    return out, lse, off, lse_off


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob) of one row in 64 bits; the settings and the random number are single, as the operator has them."""
    temperature, top_p, min_p, u = (float(np.float32(a)) for a in (temperature, top_p, min_p, u))
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf
    if not temperature > 0:
        return int(np.argmax(x)), 0.0
    with np.errstate(all="ignore"):
        w = np.where(x == top, 1.0, 0.0 if top == np.inf else np.exp((x - top) / np.float64(temperature)))
    order = np.argsort(-x, kind="stable")
    k = x.size if top_k <= 0 else min(int(top_k), x.size)
    sums = np.cumsum(w[order[:k]])
    n = k
    if top_p < 1:
        n = min(n, 1 + int(np.searchsorted(sums, max(float(top_p), 0.0) * sums[-1])))
    if min_p > 0:
        n = min(n, int((w >= min(float(min_p), 1.0)).sum()))
    kept = np.sort(order[:n])
    kept = kept[w[kept] > 0]
    sums = np.cumsum(w[kept])
    target = (float(u) if u > 0 else 0.0) * sums[-1]
    i = min(int(np.searchsorted(sums, target, side="right")), kept.size - 1)
    return int(kept[i]), float(np.log(w[kept[i]] / sums[-1]))
