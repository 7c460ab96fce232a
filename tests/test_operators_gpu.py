"""Layer norm, rotary positions and attention as linked operators, against their definitions in 64 bits."""
import ctypes

import numpy as np
import pytest

from ocannl_b200 import backend as bk
from ocannl_b200.low_level import Tnode
from tests import operators_reference as R

pytestmark = pytest.mark.gpu
PRECS = ("single", "bfloat16", "half")
S24 = 2.0 ** -24


# ------------------------------------------------------------------ layer norm
NORMS = [(1, 1), (3, 7), (1, 512), (37, 96), (200, 512), (5, 777), (33, 1000), (9, 2048), (4, 5000), (3, 8192), (2, 8200), (3, 12345), (0, 64)]


def norm_case(rows, n, prec, seed, residual):
    rng = np.random.default_rng(seed)
    x = R.rounded(prec, rng.standard_normal((rows, n)) * np.exp(rng.standard_normal((rows, 1))) + 3.0 * rng.standard_normal((rows, 1)))
    r = R.rounded(prec, rng.standard_normal((rows, n))) if residual else None
    return x, r, R.rounded("single", 1.0 + 0.2 * rng.standard_normal(n)), R.rounded("single", 0.2 * rng.standard_normal(n)), rng


def mean_off(h, n):
    # a sum of n values in single precision, tree-like, at most 64 in a row: 2^-24 each of the partial sums
    return 80 * S24 * np.abs(h).mean(-1)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("rows,n", NORMS)
def test_layer_norm(device, rows, n, prec):
    for residual, packing in ((False, "aligned"), (True, "aligned"), (True, "tight")):
        x, r, gamma, beta, _ = norm_case(rows, n, prec, 1, residual)
        a = dict(x=(prec, (rows, n), x), gamma=("single", (n,), gamma), beta=("single", (n,), beta), y=(prec, (rows, n), None),
                 mean=("single", (rows,), None), rstd=("single", (rows,), None))
        if residual:
            a.update(r=(prec, (rows, n), r), h=(prec, (rows, n), None))
        nodes = R.Nodes(device, a, packing, odd_first=packing == "tight")
        op = nodes.context.layer_norm("x", "y", gamma="gamma", beta="beta", mean="mean", rstd="rstd",
                                      **(dict(residual="r", total="h") if residual else {}))
        op.run()
        y, h, mean, rstd, u = R.layer_norm(x, gamma, beta, r)
        moff = mean_off(h, n)
        # the mean's error moves every u alike; the variance's is relative: 80 steps, and the mean's error squared
        roff = rstd * (100 * S24 + (moff * rstd) ** 2)
        uoff = moff * rstd + np.abs(u).max(-1, initial=0.0) * 104 * S24 + np.abs(u).max(-1, initial=0.0) * (moff * rstd) ** 2
        half = R.EPS[prec] / 2
        if rows:
            R.within(nodes.read("mean"), mean, moff + 1e-30, "mean")
            R.within(nodes.read("rstd"), rstd, roff, "rstd")
            R.within(nodes.read("y"), y, (uoff[:, None] * np.abs(gamma) + 4 * S24 * (np.abs(u * gamma) + np.abs(beta))) * (1 + half) + half * np.abs(y) + 2.0 ** -25, "y")
            if residual:
                R.within(nodes.read("h"), h, (half + S24) * np.abs(h) + 2.0 ** -25, "h")
        op.free()
        nodes.free()


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("rows,n", NORMS + [(5000, 128), (3000, 40), (700, 9000)])
def test_layer_norm_grad(device, rows, n, prec):
    for stream, packing in ((False, "aligned"), (True, "tight")):
        x, _, gamma, _, rng = norm_case(rows, n, prec, 2, False)
        dy, dh = R.rounded(prec, rng.standard_normal((rows, n))), R.rounded(prec, rng.standard_normal((rows, n))) if stream else None
        _, _, mean, rstd, _ = R.layer_norm(x, gamma, 0.0 * gamma)
        mean, rstd = R.rounded("single", mean), R.rounded("single", rstd)
        a = dict(x=(prec, (rows, n), x), dy=(prec, (rows, n), dy), gamma=("single", (n,), gamma), mean=("single", (rows,), mean),
                 rstd=("single", (rows,), rstd), dx=(prec, (rows, n), None), dg=("single", (n,), None), db=("single", (n,), None))
        if stream:
            a["dh"] = (prec, (rows, n), dh)
        nodes = R.Nodes(device, a, packing, odd_first=packing == "tight")
        op = nodes.context.layer_norm_grad("x", "dy", "dx", "mean", "rstd", gamma="gamma", dgamma="dg", dbeta="db", d_total="dh" if stream else None)
        op.run()
        first = nodes.read("dg"), nodes.read("db")
        op.run()      # the same bits again
        assert np.array_equal(first[0], nodes.read("dg")) and np.array_equal(first[1], nodes.read("db"))
        dx, dg, db, u, g = R.layer_norm_grad(x, mean, rstd, gamma, dy, dh)
        half = R.EPS[prec] / 2
        uoff = 3 * S24 * (np.abs(u) + np.abs(mean * rstd)[:, None])
        if rows:
            sums = 90 * S24 * (np.abs(g).mean(-1) + np.abs(u).max(-1) * np.abs(g * u).mean(-1)) + uoff.max(-1) * (np.abs(g * u).mean(-1) + np.abs(u).max(-1) * np.abs(g).mean(-1))
            bound = rstd[:, None] * (sums[:, None] + 8 * S24 * np.abs(g))
            R.within(nodes.read("dx"), dx, bound * (1 + half) + (half + S24) * np.abs(dx) + 2.0 ** -25, "dx")
        # sums over the rows: runs of rows / (number of runs), at most 200 additions in a row at these sizes
        R.within(nodes.read("dg"), dg, 220 * S24 * np.abs(dy * u).sum(0) + (np.abs(dy) * uoff).sum(0) + 1e-30, "dgamma")
        R.within(nodes.read("db"), db, 220 * S24 * np.abs(dy).sum(0) + 1e-30, "dbeta")
        op.free()
        nodes.free()


def test_layer_norm_gradients_by_differences(device):
    """The gradients that the operator gives against central differences of the forward operator, in single precision."""
    rows, n = 6, 40
    x, _, gamma, beta, rng = norm_case(rows, n, "single", 3, False)
    c = rng.standard_normal((rows, n))
    a = dict(x=("single", (rows, n), x), dy=("single", (rows, n), c), gamma=("single", (n,), gamma), beta=("single", (n,), beta),
             y=("single", (rows, n), None), dx=("single", (rows, n), None), mean=("single", (rows,), None), rstd=("single", (rows,), None),
             dg=("single", (n,), None), db=("single", (n,), None))
    nodes = R.Nodes(device, a)
    fwd = nodes.context.layer_norm("x", "y", gamma="gamma", beta="beta", mean="mean", rstd="rstd")
    bwd = nodes.context.layer_norm_grad("x", "dy", "dx", "mean", "rstd", gamma="gamma", dgamma="dg", dbeta="db")
    fwd.run()
    bwd.run()
    got = {w: nodes.read(g) for w, g in (("x", "dx"), ("gamma", "dg"), ("beta", "db"))}
    dy = R.rounded("single", c)
    for name, base in (("x", x), ("gamma", gamma), ("beta", beta)):
        direction = rng.standard_normal(base.shape)
        step, vals = 2.0 ** -7, []
        for sign in (1, -1):
            nodes.context.from_host(name, (base + sign * step * direction).astype(np.float32))
            fwd.run()
            vals.append((nodes.read("y") * dy).sum())
        nodes.context.from_host(name, base.astype(np.float32))
        diff, want = (vals[0] - vals[1]) / (2 * step), (got[name] * direction).sum()
        # values of size sum|y dy| in single precision, divided by the step; the difference's own error is step^2 of third derivatives
        size = np.abs(nodes.read("y") * dy).sum()
        assert abs(diff - want) <= 64 * S24 * size / step + 64 * step ** 2 * np.abs(got[name] * direction).sum(), (name, diff, want)
    for x_ in (fwd, bwd):
        x_.free()
    nodes.free()


# ------------------------------------------------------------------ rotary
@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("b,s,h,hk,d,pairs", [(1, 1, 1, 0, 2, 1), (2, 5, 3, 1, 64, 32), (3, 33, 4, 2, 96, 16), (1, 130, 2, 2, 80, 20), (2, 9, 5, 1, 33, 7),
                                               (1, 3, 1, 1, 128, 0), (2, 0, 2, 1, 64, 32), (1, 700, 8, 8, 128, 64)])
def test_rotary(device, b, s, h, hk, d, pairs, prec):
    rng = np.random.default_rng(5)
    q, k = R.rounded(prec, rng.standard_normal((b, s, h, d))), R.rounded(prec, rng.standard_normal((b, s, max(hk, 1), d)))
    pos = rng.integers(-5, 2 ** 31 - 1, (b, s)).astype(np.int32)
    f, mag = bk.rotary_frequencies(2 * pairs, scaling="yarn", factor=4.0)
    for layout in ("half", "interleaved"):
        for inverse in (False, True):
            for packing, in_place in (("aligned", False), ("tight", False), ("aligned", True)):
                a = dict(q=(prec, q.shape, q), k=(prec, k.shape, k), pos=("int32", (b, s), pos), yq=(prec, q.shape, None), yk=(prec, k.shape, None))
                nodes = R.Nodes(device, a, packing, odd_first=packing == "tight")
                to = ("q", "k") if in_place else ("yq", "yk")
                given = not in_place
                op = nodes.context.rotary([("q", to[0])] + ([("k", to[1])] if hk else []), f, mag, positions="pos" if given else None,
                                          first_position=1000003, layout=layout, inverse=inverse)
                op.run()
                p = pos.astype(np.int64) if given else np.broadcast_to(1000003 + np.arange(s), (b, s))
                for x, name in ((q, to[0]), (k, to[1]))[:2 if hk else 1]:
                    # (angles of 2^31 radians are off by 2^-22 in 64 bits themselves: extended precision for the test's own)
                    want = rotary_long(x, f, p, layout, inverse, mag)
                    size = np.abs(x).max(-1, keepdims=True, initial=0.0) * 2 * max(mag, 1.0)
                    R.within(nodes.read(name), want, R.EPS[prec] / 2 * np.abs(want) + 12 * S24 * size + 2.0 ** -25, name)
                op.free()
                nodes.free()


def rotary_long(x, f, p, layout, inverse, mag):
    turns = np.asarray(f, np.longdouble) / (2 * np.longdouble("3.14159265358979323846264338327950288"))
    whole = p[:, :, None, None].astype(np.longdouble) * turns
    angle = ((whole - np.floor(whole)) * (2 * np.longdouble("3.14159265358979323846264338327950288"))).astype(np.float64)
    m = len(f)
    c, s = np.cos(angle) * mag, np.sin(angle) * (-mag if inverse else mag)
    i, j = (np.arange(m), np.arange(m) + m) if layout == "half" else (2 * np.arange(m), 2 * np.arange(m) + 1)
    y = x.copy()
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    return y


# ------------------------------------------------------------------ attention
def docs_of(rng, b, n):
    ids = np.cumsum(rng.random((b, n)) < 4.0 / max(n, 4), 1).astype(np.int32)
    ids[:, n - n // 9:] = -1
    if n > 4:
        ids[0, 1] = -7          # a hole
    return ids


# batch, queries, keys, heads, kv_heads, d, mask, documents, lengths, cap, slopes
ATTENTION = [
    (1, 1, 1, 1, 1, 1, "causal", False, None, 0.0, False),
    (2, 3, 0, 2, 1, 16, "causal", False, None, 0.0, False),
    (1, 0, 5, 2, 1, 16, "causal", False, None, 0.0, False),
    (2, 1, 300, 8, 2, 64, "causal", False, (300, 17), 0.0, False),
    (3, 1, 129, 4, 4, 128, "causal", False, (0, 1, 129), 30.0, True),
    (2, 5, 1000, 8, 1, 72, "causal", False, (999, 3), 0.0, True),
    (1, 128, 128, 1, 1, 64, "none", False, None, 0.0, False),
    (2, 77, 77, 4, 2, 40, "causal", False, None, 0.0, False),
    (1, 130, 257, 2, 1, 64, "none", False, None, 20.0, False),
    (1, 260, 260, 3, 1, 128, "causal", True, None, 0.0, False),
    (2, 300, 300, 2, 2, 96, "prefix", True, None, 50.0, True),
    (2, 33, 190, 2, 1, 33, "prefix", False, (500, -3), 0.0, True),
    (1, 400, 150, 2, 2, 24, "causal", False, None, 0.0, False),      # more queries than keys: the first see nothing
    (1, 513, 513, 4, 4, 8, "causal", True, None, 0.0, False),
    (2, 200, 200, 2, 1, 80, "none", True, (200, 64), 10.0, False),
]


def attention_case(case, prec, seed=7):
    b, s, n, h, hk, d, mask, docs, lengths, cap, slopes = case
    rng = np.random.default_rng(seed)
    spread = 2.0 if cap else 1.0
    x = dict(q=R.rounded(prec, rng.standard_normal((b, s, h, d)) * spread), k=R.rounded(prec, rng.standard_normal((b, n, hk, d)) * spread),
             v=R.rounded(prec, rng.standard_normal((b, n, hk, d))), d_out=R.rounded(prec, rng.standard_normal((b, s, h, d)) * 0.3))
    t = dict(mask=mask, cap=cap)
    more = {}
    if mask == "prefix":
        more["prefix"] = rng.integers(-2, n // 2 + 1, b).astype(np.int32)
    if docs:
        more["kdoc"] = docs_of(rng, b, n)
        more["qdoc"] = more["kdoc"][:, n - s:] if s <= n else np.zeros((b, s), np.int32)
    if lengths is not None:
        more["lengths"] = np.array(lengths, np.int32)
    sl = R.rounded("single", 2.0 ** -np.arange(1, h + 1)) if slopes else None
    seen, pos = R.visible(b, s, n, mask, more.get("prefix"), more.get("qdoc"), more.get("kdoc"), more.get("lengths"))
    return x, t, more, sl, seen, pos, 1.0 / np.sqrt(d)


def link_attention(device, case, prec, x, t, more, sl, packing, grad=False):
    b, s, n, h, hk, d = case[:6]
    a = {name: (prec, v.shape, v) for name, v in x.items()}
    a.update(out=(prec, (b, s, h, d), x.get("out")), lse=("single", (b, h, s), x.get("lse")))
    if "lse" in x:
        a["lse"] = ("single", (b, h, s), x["lse"])
    if grad:
        a.update(dq=(prec, x["q"].shape, None), dk=(prec, x["k"].shape, None), dv=(prec, x["v"].shape, None))
    a.update({m: ("int32", v.shape, v) for m, v in more.items()})
    if sl is not None:
        a["slopes"] = ("single", (h,), sl)
    nodes = R.Nodes(device, a, packing, odd_first=packing == "tight")
    kw = dict(mask=t["mask"], cap=t["cap"], prefix="prefix" if "prefix" in more else None, lengths="lengths" if "lengths" in more else None,
              documents=("qdoc", "kdoc") if "qdoc" in more else None, slopes="slopes" if sl is not None else None)
    if grad:
        return nodes, nodes.context.attention_grad("q", "k", "v", "out", "lse", "d_out", "dq", "dk", "dv", **kw)
    return nodes, nodes.context.attention("q", "k", "v", "out", lse="lse", **kw)


def out_bound(prec, out, size, flat):
    half = R.EPS[prec] / 2
    return half * np.abs(out) + ((half if prec != "single" else 0.0) + R.ARITH) * size + (2.0 ** -25 * (flat + 1) if prec == "half" else 1e-30)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("case", ATTENTION)
def test_attention(device, case, prec):
    x, t, more, sl, seen, pos, scale = attention_case(case, prec)
    out, lse, size, flat = R.attention(x["q"], x["k"], x["v"], seen, pos, scale, t["cap"], sl)
    for packing in ("aligned", "tight"):
        nodes, op = link_attention(device, case, prec, {n: x[n] for n in "qkv"}, t, more, sl, packing)
        op.run()
        device.await_()
        R.within(nodes.read("out"), out, out_bound(prec, out, size, flat), "out")
        R.within(nodes.read("lse"), lse, R.ARITH * (1 + np.abs(np.where(np.isinf(lse), 0, lse))), "lse")
        op.free()
        nodes.free()


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("case", ATTENTION)
def test_attention_grad(device, case, prec):
    x, t, more, sl, seen, pos, scale = attention_case(case, prec)
    out, lse, _, _ = R.attention(x["q"], x["k"], x["v"], seen, pos, scale, t["cap"], sl)
    x["out"], x["lse"] = R.rounded(prec, out), R.rounded("single", lse)
    want = R.attention_grad(x["q"], x["k"], x["v"], x["out"], x["lse"], x["d_out"], seen, pos, scale, t["cap"], sl, prec)
    for packing in ("aligned", "tight"):
        nodes, op = link_attention(device, case, prec, x, t, more, sl, packing, grad=True)
        op.run()
        device.await_()
        first = [nodes.read(n) for n in ("dq", "dk", "dv")]
        for n, got, (v, bound) in zip(("dq", "dk", "dv"), first, want):
            R.within(got, v, bound, n)
        op.run()
        device.await_()
        assert all(np.array_equal(nodes.read(n), f) for n, f in zip(("dq", "dk", "dv"), first)), "the same inputs give the same bits"
        op.free()
        nodes.free()


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("case", [ATTENTION[3], ATTENTION[5], ATTENTION[9], ATTENTION[10], ATTENTION[14]])
def test_attention_ignores_what_is_not_seen(device, case, prec):
    """Infinities and NaN at keys and queries that are not seen, at hidden keys between visible ones too."""
    x, t, more, sl, seen, pos, scale = attention_case(case, prec)
    rows, keys = seen.any(2), seen.any(1)
    for name, on in (("k", keys), ("v", keys), ("q", rows), ("d_out", rows)):
        x[name] = np.where(on[:, :, None, None], x[name], np.nan)
        x[name][~on] = np.where(np.arange(x[name].shape[-1]) % 2, np.nan, np.inf)
    # one value that only later queries see
    b, s, n = case[:3]
    if case[6] == "causal" and s > 40:
        j = n - 20
        x["v"][:, j] = np.where(keys[:, j, None, None], np.inf, x["v"][:, j])
    with np.errstate(all="ignore"):
        clean = {m: np.where(np.isfinite(x[m]), x[m], 0.0) for m in ("q", "k")}
        out, lse, size, flat = R.attention(clean["q"], clean["k"], x["v"], seen, pos, scale, t["cap"], sl)
    nodes, op = link_attention(device, case, prec, {m: x[m] for m in "qkv"}, t, more, sl, "aligned")
    op.run()
    device.await_()
    with np.errstate(all="ignore"):
        R.within(nodes.read("out"), out, np.where(np.isfinite(out), out_bound(prec, np.where(np.isfinite(out), out, 0), size, flat), 0.0), "out")
    R.within(nodes.read("lse"), lse, R.ARITH * (1 + np.abs(np.where(np.isinf(lse), 0, lse))), "lse")
    op.free()
    nodes.free()
    x["v"] = np.where(np.isinf(x["v"]) & keys[:, :, None, None], 1.0, x["v"])
    out, lse, _, _ = R.attention(clean["q"], clean["k"], x["v"], seen, pos, scale, t["cap"], sl)
    x["out"], x["lse"] = R.rounded(prec, out), R.rounded("single", lse)
    x["out"][~rows] = np.nan
    want = R.attention_grad(clean["q"], clean["k"], np.where(keys[:, :, None, None], x["v"], 0.0), np.where(rows[:, :, None, None], x["out"], 0.0), x["lse"],
                            np.where(rows[:, :, None, None], x["d_out"], 0.0), seen, pos, scale, t["cap"], sl, prec)
    nodes, op = link_attention(device, case, prec, x, t, more, sl, "aligned", grad=True)
    op.run()
    device.await_()
    for m, (v, bound) in zip(("dq", "dk", "dv"), want):
        R.within(nodes.read(m), v, bound, m)
    op.free()
    nodes.free()


@pytest.mark.parametrize("prec", ("bfloat16", "half"))
@pytest.mark.parametrize("case", [(1, 60, 1100, 2, 1, 33, "causal", False, None, 0.0, False), (2, 20, 2048, 4, 2, 128, "causal", False, (2048, 40), 30.0, True)])
def test_attention_over_split_keys_ignores_what_is_not_seen(device, case, prec):
    test_attention_ignores_what_is_not_seen(device, case, prec)


def test_attention_gradients_by_differences(device):
    """The gradients that the operator gives against central differences of the forward operator, in single precision."""
    case = (2, 70, 70, 4, 2, 24, "prefix", True, None, 8.0, True)
    x, t, more, sl, seen, pos, scale = attention_case(case, "single")
    nodes, fwd = link_attention(device, case, "single", {n: x[n] for n in "qkv"}, t, more, sl, "aligned")
    fwd.run()
    x["out"], x["lse"] = nodes.read("out"), nodes.read("lse")
    grads, bwd = link_attention(device, case, "single", x, t, more, sl, "aligned", grad=True)
    bwd.run()
    rng = np.random.default_rng(3)
    for name in "qkv":
        got = grads.read("d" + name)
        direction, step, vals = rng.standard_normal(x[name].shape), 2.0 ** -6, []
        for sign in (1, -1):
            nodes.context.from_host(name, (x[name] + sign * step * direction).astype(np.float32))
            fwd.run()
            vals.append((nodes.read("out") * x["d_out"]).sum())
        nodes.context.from_host(name, x[name].astype(np.float32))
        diff, want = (vals[0] - vals[1]) / (2 * step), (got * direction).sum()
        # values in single precision (2^-15 of their sizes at most), divided by the step; the third derivative's share is step^2
        # of a sum of products like the first's
        size = np.abs(x["out"] * x["d_out"]).sum()
        assert abs(diff - want) <= R.ARITH * np.sqrt(x["out"].size) * size / x["out"].size / step + 64 * step ** 2 * np.abs(got * direction).sum(), (name, diff, want)
    for o in (fwd, bwd):
        o.free()
    nodes.free()
    grads.free()


def test_weights_of_16_bits_in_the_norm(device):
    x, _, gamma, beta, _ = norm_case(9, 96, "bfloat16", 4, False)
    gamma, beta = R.rounded("bfloat16", gamma), R.rounded("bfloat16", beta)
    nodes = R.Nodes(device, dict(x=("bfloat16", (9, 96), x), gamma=("bfloat16", (96,), gamma), beta=("bfloat16", (96,), beta), y=("bfloat16", (9, 96), None)))
    op = nodes.context.layer_norm("x", "y", gamma="gamma", beta="beta")
    op.run()
    y = R.layer_norm(x, gamma, beta)[0]
    R.within(nodes.read("y"), y, R.EPS["bfloat16"] / 2 * np.abs(y) + 2.0 ** -14, "y")
    op.free()
    bare = nodes.context.layer_norm("x", "y")
    bare.run()
    y = R.layer_norm(x, 1.0, 0.0)[0]
    R.within(nodes.read("y"), y, R.EPS["bfloat16"] / 2 * np.abs(y) + 2.0 ** -14, "y")
    bare.free()
    nodes.free()


def test_operators_of_one_kernel_and_different_sizes(device):
    """A later link of a smaller problem takes nothing from an earlier one of a larger, and the other way round."""
    sizes = ((3, 8192), (3, 5000), (2, 8192))
    made = []
    for rows, n in sizes:
        x, _, gamma, beta, _ = norm_case(rows, n, "single", n, False)
        nodes = R.Nodes(device, dict(x=("single", (rows, n), x), g=("single", (n,), gamma), b=("single", (n,), beta), y=("single", (rows, n), None)))
        made.append((nodes, nodes.context.layer_norm("x", "y", gamma="g", beta="b"), R.layer_norm(x, gamma, beta)[0]))
    cases = [(1, 70, 70, 2, 2, 64, "causal", True, None, 0.0, False), (1, 20, 20000, 2, 2, 64, "causal", True, None, 0.0, False), ATTENTION[13],
             (1, 130, 20000, 1, 1, 64, "causal", True, None, 0.0, False)]
    attn = []
    for case in cases:
        x, t, more, sl, seen, pos, scale = attention_case(case, "bfloat16")
        out, _, size, flat = R.attention(x["q"], x["k"], x["v"], seen, pos, scale)
        attn.append(link_attention(device, case, "bfloat16", {m: x[m] for m in "qkv"}, t, more, sl, "aligned") + (out, out_bound("bfloat16", out, size, flat)))
    for nodes, op, y in made + made[::-1]:
        op.run()
        R.within(nodes.read("y"), y, 2.0 ** -16 * (1 + np.abs(y)), "y")
    for nodes, op, out, bound in attn + attn[::-1]:
        op.run()
        device.await_()
        R.within(nodes.read("out"), out, bound, "out")
    for x in made + attn:
        x[1].free()
        x[0].free()


def test_memory_around_the_outputs_is_left_alone(device):
    """Outputs between other nodes, aligned to their elements alone: what lies before and behind them keeps its values."""
    for prec in PRECS:
        case = (1, 70, 70, 2, 1, 40, "causal", True, None, 0.0, False)
        x, t, more, sl, seen, pos, scale = attention_case(case, prec)
        b, s, n, h, hk, d = case[:6]
        out, lse, _, _ = R.attention(x["q"], x["k"], x["v"], seen, pos, scale)
        mark = np.arange(5, dtype=np.float64) + 1
        a = {m: (prec, v.shape, v) for m, v in x.items()}
        a.update({m: ("int32", v.shape, v) for m, v in more.items()})
        a.update(fwd_out=(prec, out.shape, None), lse=("single", lse.shape, R.rounded("single", lse)), out=(prec, out.shape, R.rounded(prec, out)))
        for i, m in enumerate(("dq", "dk", "dv", "y")):
            a["guard%d" % i] = (prec, (5,), mark)
            a[m] = (prec, x["k" if m in ("dk", "dv") else "q"].shape, None)
        a["guard9"] = (prec, (5,), mark)
        nodes = R.Nodes(device, a, "tight", odd_first=True)
        ctx, docs = nodes.context, ("qdoc", "kdoc")
        ops = [ctx.attention("q", "k", "v", "fwd_out", documents=docs), ctx.attention_grad("q", "k", "v", "out", "lse", "d_out", "dq", "dk", "dv", documents=docs),
               ctx.rotary([("q", "y")], bk.rotary_frequencies(20)[0])]
        for o in ops:
            o.run()
        device.await_()
        for g in ("guard0", "guard1", "guard2", "guard3", "guard9"):
            assert np.array_equal(nodes.read(g), mark), g
        assert np.array_equal(nodes.read("q"), x["q"]) and np.array_equal(nodes.read("k"), x["k"])
        for o in ops:
            o.free()
        nodes.free()


def test_captured_replayed_and_with_a_growing_cache(device):
    """One operator captured into a CUDA graph: replays read the lengths and keys of their time; a second operator of the same
    sizes runs between them."""
    import torch
    case = (3, 1, 400, 8, 2, 64, "causal", False, (5, 100, 250), 0.0, False)
    x, t, more, sl, _, _, scale = attention_case(case, "bfloat16")
    nodes, op = link_attention(device, case, "bfloat16", {n: x[n] for n in "qkv"}, t, more, sl, "aligned")
    others, other = link_attention(device, case, "bfloat16", {n: x[n] * 0.5 for n in "qkv"}, t, more, sl, "aligned")
    device.await_()
    stream = torch.cuda.ExternalStream(device.stream_handle())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        op.run()
    for lengths in ((5, 100, 250), (6, 101, 251), (400, 0, 399)):
        nodes.context.from_host("lengths", np.array(lengths, np.int32))
        with torch.cuda.stream(stream):
            graph.replay()
        other.run()
        with torch.cuda.stream(stream):
            graph.replay()
        device.await_()
        seen, pos = R.visible(3, 1, 400, "causal", lengths=lengths)
        out, lse, size, flat = R.attention(x["q"], x["k"], x["v"], seen, pos, scale)
        R.within(nodes.read("out"), out, out_bound("bfloat16", out, size, flat), "out")
    del graph
    for o in (op, other):
        o.free()
    nodes.free()
    others.free()


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("s,n", [(3, 60), (40, 300), (300, 40)])
def test_one_node_as_queries_keys_and_values(device, s, n, prec):
    """Inputs may be one node, each of the rows that its own shape says; heads of 20 elements take copies with padded rows."""
    most = max(s, n)
    rng = np.random.default_rng(17)
    both = R.rounded(prec, rng.standard_normal((1, most, 2, 20)))
    x = dict(q=both[:, :s], k=both[:, :n], v=both[:, :n], d_out=both[:, :s])
    seen, pos = R.visible(1, s, n, "none")
    scale = 1.0 / np.sqrt(20)
    out, lse, size, flat = R.attention(x["q"], x["k"], x["v"], seen, pos, scale)
    o, l = R.rounded(prec, out), R.rounded("single", lse)
    want = R.attention_grad(x["q"], x["k"], x["v"], o, l, x["d_out"], seen, pos, scale, 0.0, None, prec)
    nodes = R.Nodes(device, dict(both=(prec, both.shape, both), out=(prec, out.shape, None), lse=("single", lse.shape, None), o=(prec, out.shape, o),
                                 l=("single", lse.shape, l), dq=(prec, x["q"].shape, None), dk=(prec, x["k"].shape, None), dv=(prec, x["k"].shape, None)))
    pool, off, _ = nodes.context.arrays["both"]
    for i, (name, rows) in enumerate((("queries", s), ("keys", n))):
        nodes.context.arrays[name] = (pool, off, Tnode(90 + i, name, prec, (1, rows, 2, 20)))
    ops = [nodes.context.attention("queries", "keys", "keys", "out", lse="lse", mask="none"),
           nodes.context.attention_grad("queries", "keys", "keys", "o", "l", "queries", "dq", "dk", "dv", mask="none")]
    for op in ops:
        op.run()
    device.await_()
    R.within(nodes.read("out"), out, out_bound(prec, out, size, flat), "out")
    for name, (v, bound) in zip(("dq", "dk", "dv"), want):
        R.within(nodes.read(name), v, bound, name)
    for op in ops:
        op.free()
    nodes.free()


def test_runs_wait_for_uploads(device):
    """With uploads on a second stream a run sees what was uploaded before it."""
    rows, n = 4096, 1024
    rng = np.random.default_rng(8)
    x = rng.standard_normal((rows, n)).astype(np.float32)
    nodes = R.Nodes(device, dict(x=("single", (rows, n), np.zeros((rows, n))), y=("single", (rows, n), None)))
    op = nodes.context.layer_norm("x", "y")
    device.set_async_uploads(True)
    try:
        pool, off, _ = nodes.context.arrays["x"]
        buf = bk.PinnedBuffer((rows, n), np.float32)
        buf.array[...] = x
        device.from_host(pool, off, buf.array)
        op.run()
        got = nodes.read("y")
    finally:
        device.set_async_uploads(False)
    y = R.layer_norm(x.astype(np.float64), 1.0, 0.0)[0]
    R.within(got, y, 2.0 ** -17 * (1 + np.abs(y)), "y")
    buf.free()
    op.free()
    nodes.free()


@pytest.mark.parametrize("queries", [1, 20])
def test_offsets_behind_two_to_the_31(device, queries):
    """A cache of 2.1 million positions: 2^31 elements and more of keys and of values.  All keys are zero, so all weights are equal."""
    n, hk, d = 2_100_000, 8, 128
    assert n * hk * d > 2 ** 31
    pools = [device.alloc_pool(n * hk * d * 2) for _ in range(2)]
    for p in pools:
        device.memset_zero(p, 0, n * hk * d * 2)
    tail = 64
    last = R.rounded("bfloat16", np.random.default_rng(1).standard_normal((tail, hk, d)) * n / 100)
    from ocannl_b200.workloads import store
    device.from_host(pools[1], (n - tail) * hk * d * 2, store("bfloat16", last.astype(np.float32)))
    from ocannl_b200.low_level import Tnode
    nodes = R.Nodes(device, dict(q=("bfloat16", (1, queries, hk, d), np.ones((1, queries, hk, d))), out=("bfloat16", (1, queries, hk, d), None)))
    arrays = dict(nodes.context.arrays, k=(pools[0], 0, Tnode(90, "k", "bfloat16", (1, n, hk, d))), v=(pools[1], 0, Tnode(91, "v", "bfloat16", (1, n, hk, d))))
    op = bk.Context(device, arrays).attention("q", "k", "v", "out", mask="none")
    op.run()
    want = last.sum(0) / n
    # equal weights of one; sums of n of them and of 64 products in single precision, added in parts
    R.within(nodes.read("out"), np.broadcast_to(want, (1, queries, hk, d)), R.EPS["bfloat16"] / 2 * np.abs(want) + 2.0 ** -12 * np.abs(last).sum(0) / n, "out")
    op.free()
    for p in pools:
        device.free_pool(p)
    nodes.free()


def test_what_link_refuses(device):
    nodes = R.Nodes(device, dict(x=("single", (64, 64), np.ones((64, 64))), q=("bfloat16", (2, 8, 4, 16), None), k=("bfloat16", (2, 8, 2, 16), None), o=("bfloat16", (2, 8, 4, 16), None)))
    pool, off, _ = nodes.context.arrays["x"]

    def linked(entry, spec):
        return bk.Operator(device, entry, spec)

    def norm(**kw):
        base = dict(rows=4, n=16, dtype=0, weight_dtype=0, eps=1e-5, x=bk.Operand(pool, off), y=bk.Operand(pool, off + 1024))
        return bk.LayerNormSpec(**dict(base, **kw))

    def attn(**kw):
        at = {n: bk.Operand(*nodes.context.arrays[n][:2]) for n in "qk"}
        base = dict(batch=2, queries=8, keys=8, heads=4, kv_heads=2, d=16, dtype=1, mask=1, scale=0.25, cap=0.0, q=at["q"], k=at["k"], v=at["k"],
                    out=bk.Operand(*nodes.context.arrays["o"][:2]))
        return bk.AttentionSpec(**dict(base, **kw))

    def rot(**kw):
        f = (ctypes.c_double * 8)(*([1.0] * 8))
        base = dict(batch=2, seq=8, heads=(4, 0), d=16, pairs=8, dtype=1, magnitude=1.0, frequencies=f, x=two("q"), y=two("o"))
        return bk.RotarySpec(**dict(base, **kw))

    def two(name):
        return (bk.Operand * 2)(bk.Operand(*nodes.context.arrays[name][:2]), bk.Operand(-1, 0))

    for entry, spec, code, words in [
            ("b200_layer_norm_link", norm(y=bk.Operand(pool, off + 16)), -1, "overlaps"),
            ("b200_layer_norm_link", norm(y=bk.Operand(pool, off)), -1, "overlaps"),
            ("b200_layer_norm_link", norm(y=bk.Operand(pool, off + 1026)), -1, "multiple of its element"),
            ("b200_layer_norm_link", norm(rows=1 << 20), -1, "exceeds pool"),
            ("b200_layer_norm_link", norm(rows=1 << 60, n=1 << 29), -1, "too many"),
            ("b200_layer_norm_link", norm(x=bk.Operand(987654, 0)), -1, "unknown pool"),
            ("b200_layer_norm_link", norm(x=bk.Operand(-1, 0)), -1, "'x' is required"),
            ("b200_layer_norm_link", norm(dtype=7), -1, "element type"),
            ("b200_layer_norm_link", norm(weight_dtype=1), -1, "gamma and beta"),
            ("b200_layer_norm_link", norm(n=0), -1, "n between"),
            ("b200_layer_norm_link", norm(eps=-1.0), -1, "eps"),
            ("b200_layer_norm_link", norm(total=bk.Operand(pool, off + 2048)), -1, "residual"),
            ("b200_layer_norm_grad_link", norm(), -1, "required"),
            ("b200_rotary_link", rot(pairs=9), -1, "2 * pairs"),
            ("b200_rotary_link", rot(heads=(0, 0)), -1, "heads"),
            ("b200_rotary_link", rot(magnitude=float("nan")), -1, "magnitude"),
            ("b200_rotary_link", rot(frequencies=(ctypes.c_double * 8)(*([float("inf")] * 8))), -1, "frequency"),
            ("b200_rotary_link", rot(heads=(4, 2)), -1, "'x[1]' is required"),
            ("b200_attention_link", attn(d=129), -4, "128"),
            ("b200_attention_link", attn(heads=3), -1, "multiple of kv_heads"),
            ("b200_attention_link", attn(scale=0.0), -1, "scale"),
            ("b200_attention_link", attn(scale=float("inf")), -1, "scale"),
            ("b200_attention_link", attn(cap=-1.0), -1, "cap"),
            ("b200_attention_link", attn(mask=3), -1, "mask"),
            ("b200_attention_link", attn(mask=2), -1, "prefix"),
            ("b200_attention_link", attn(query_documents=bk.Operand(pool, off)), -1, "documents"),
            ("b200_attention_link", attn(out=bk.Operand(*nodes.context.arrays["q"][:2])), -1, "overlaps"),
            ("b200_attention_link", attn(keys=-1), -1, "between 0"),
            ("b200_attention_grad_link", attn(), -1, "'lse' is required")]:
        with pytest.raises(bk.B200Error) as e:
            linked(entry, spec)
        assert e.value.code == code and words in str(e.value), (entry, words, str(e.value))
    nodes.free()


# ------------------------------------------------------------------ together
def matmul_routine(name, terms, rows):
    """out[r, o] = sum over (w, x, transposed) of sum_i w[o, i] (or w[i, o]) x[r, i], single precision."""
    from ocannl_b200.low_level import Routine, Seq, Set, loops
    from ocannl_b200.workloads import reduce_scope
    r = Routine(name)
    tns, body = {}, []

    def tn(n, dims):
        if n not in tns:
            tns[n] = r.tn(n, "single", dims)
        return tns[n]
    for out, o_dim, w, x, i_dim, transposed in terms:
        wt, xt, ot = tn(w, (i_dim, o_dim) if transposed else (o_dim, i_dim)), tn(x, (rows, i_dim)), tn(out, (rows, o_dim))
        a, o, i = r.syms(3)
        body.append(loops([(a, rows), (o, o_dim)], Set(ot, (a, o), reduce_scope(
            r, out + "_mm", "single", [(i, i_dim)], lambda: (wt[i, o] if transposed else wt[o, i], xt[a, i]), orig=(a, o)))))
    r.body = Seq(body)
    return r


def test_a_decoder_layer_forward_and_backward(device):
    """Norm, projections (a routine), rotary positions, attention, projection, residual and norm; then all gradients back to the
    input, with the operators and routines of the framework in turn on one stream.  Against the layer in 64 bits and the
    central difference of its loss."""
    from ocannl_b200.low_level import Tnode
    b, s, h, hk, e = 2, 45, 4, 2, 16
    dm, rows = 48, 2 * 45
    rng = np.random.default_rng(12)
    w = {n: R.rounded("single", rng.standard_normal(shape) / np.sqrt(shape[1])) for n, shape in
         (("wq", (h * e, dm)), ("wk", (hk * e, dm)), ("wv", (hk * e, dm)), ("wo", (dm, h * e)))}
    g1, b1, g2, b2 = (R.rounded("single", o + 0.2 * rng.standard_normal(dm)) for o in (1, 0, 1, 0))
    x, dy = (R.rounded("single", rng.standard_normal((rows, dm))) for _ in range(2))
    docs = docs_of(rng, b, s)
    freq = bk.rotary_frequencies(e)[0]
    seen, pos = R.visible(b, s, s, "causal", qdoc=docs, kdoc=docs)
    seat = np.broadcast_to(np.arange(s), (b, s))

    def model(x):
        n1, _, m1, r1, _ = R.layer_norm(x, g1, b1)
        q, k, v = ((n1 @ w[n].T).reshape(b, s, -1, e) for n in ("wq", "wk", "wv"))
        out, _, _, _ = R.attention(R.rotary(q, freq, seat), R.rotary(k, freq, seat), v, seen, pos, 0.25, 20.0)
        return R.layer_norm(x, g2, b2, residual=out.reshape(rows, h * e) @ w["wo"].T)[0]

    single = lambda n, dims, v=None: (n, dims, v)  # noqa: E731
    plan = [single("x", (rows, dm), x), single("dy", (rows, dm), dy)] + [single(n, v.shape, v) for n, v in w.items()]
    plan += [single(n, (dm,), v) for n, v in (("g1", g1), ("b1", b1), ("g2", g2), ("b2", b2))]
    plan += [single(n, (rows, dm)) for n in ("n1", "o", "t", "y", "dt", "dn_q", "dn_k", "dn_v", "dn", "dx")]
    plan += [single(n, (rows,)) for n in ("m1", "r1", "m2", "r2")] + [single(n, (dm,)) for n in ("dg1", "db1", "dg2", "db2")]
    plan += [single(n, (b, h, s)) for n in ("lse",)]
    wide, narrow = ("q", "av", "d_av", "dq"), ("k", "v", "dk", "dv")
    tns = [Tnode(i + 1, n, "single", d) for i, (n, d, _) in enumerate(plan)]
    # the projections' rows and the heads that the operators see are the same memory
    ctx = bk.Context(device).allocate(tns + [Tnode(100, "docs", "int32", (b, s))] + [Tnode(200 + i, n, "single", (b, s, h if n in wide else hk, e)) for i, n in enumerate(wide + narrow)])
    flat = dict(ctx.arrays)
    for n in wide + narrow:
        p, off, t = flat[n]
        flat[n] = (p, off, Tnode(t.id, n, "single", (rows, (h if n in wide else hk) * e)))
    for n, _, v in plan:
        if v is not None:
            ctx.from_host(n, v.astype(np.float32))
    ctx.from_host("docs", docs)
    by_rows = bk.Context(device, flat)
    from ocannl_b200.low_level import Routine, Set, loops
    codes = [bk.Code(matmul_routine("proj", [("q", h * e, "wq", "n1", dm, False), ("k", hk * e, "wk", "n1", dm, False), ("v", hk * e, "wv", "n1", dm, False)], rows), "tf32=0"),
             bk.Code(matmul_routine("out_proj", [("o", dm, "wo", "av", h * e, False)], rows), "tf32=0"),
             bk.Code(matmul_routine("out_grad", [("d_av", h * e, "wo", "dt", dm, True)], rows), "tf32=0"),
             bk.Code(matmul_routine("proj_grad", [("dn_q", dm, "wq", "dq", h * e, True), ("dn_k", dm, "wk", "dk", hk * e, True), ("dn_v", dm, "wv", "dv", hk * e, True)], rows), "tf32=0")]
    add = Routine("add")
    parts = [add.tn(n, "single", (rows, dm), read_only=True) for n in ("dn_q", "dn_k", "dn_v")]
    dn = add.tn("dn", "single", (rows, dm))
    i, j = add.syms(2)
    add.body = loops([(i, rows), (j, dm)], Set(dn, (i, j), parts[0][i, j] + parts[1][i, j] + parts[2][i, j]))
    codes.append(bk.Code(add))
    proj, out_proj, out_grad, proj_grad, adding = (by_rows.link(c) for c in codes)
    terms = dict(documents="docs", cap=20.0, scale=0.25)
    av_as_heads, turned = ctx, [("q", "q"), ("k", "k")]
    steps = [ctx.layer_norm("x", "n1", gamma="g1", beta="b1", mean="m1", rstd="r1"), proj, ctx.rotary(turned, freq),
             av_as_heads.attention("q", "k", "v", "av", lse="lse", **terms), out_proj,
             ctx.layer_norm("x", "y", gamma="g2", beta="b2", residual="o", total="t", mean="m2", rstd="r2"),
             ctx.layer_norm_grad("t", "dy", "dt", "m2", "r2", gamma="g2", dgamma="dg2", dbeta="db2"), out_grad,
             ctx.attention_grad("q", "k", "v", "av", "lse", "d_av", "dq", "dk", "dv", **terms),
             ctx.rotary([("dq", "dq"), ("dk", "dk")], freq, inverse=True), proj_grad, adding,
             ctx.layer_norm_grad("x", "dn", "dx", "m1", "r1", gamma="g1", dgamma="dg1", dbeta="db1", d_total="dt")]
    first = None
    for _ in range(2):
        for st in steps:
            st.run()
        device.await_()
        got = {n: ctx.to_host(n).astype(np.float64) for n in ("y", "dx", "dg1", "db2")}
        first = first or got
        assert all(np.array_equal(first[n], got[n]) for n in got), "the same inputs give the same bits"
    want = model(x)
    assert np.abs(got["y"] - want).max() <= 2.0 ** -14 * (1 + np.abs(want).max())
    for _ in range(3):
        direction, step = rng.standard_normal(x.shape), 1e-5
        diff = ((model(x + step * direction) - model(x - step * direction)) * dy).sum() / (2 * step)
        assert abs((got["dx"] * direction).sum() - diff) <= 2.0 ** -13 * np.abs(got["dx"] * direction).sum(), (diff, (got["dx"] * direction).sum())
    for st in steps:
        st.free()
    for c in codes:
        c.free()
    for p in {p for p, _, _ in ctx.arrays.values()}:
        device.free_pool(p)


# many tiles in a row, where a wait that is missing or too early would show
LONG = [
    (2, 1030, 1030, 2, 1, 64, "causal", False, None, 0.0, False),
    (3, 1030, 1030, 4, 2, 128, "causal", True, None, 30.0, False),
    (40, 513, 513, 2, 2, 128, "none", False, None, 0.0, True),
    (24, 640, 640, 4, 4, 128, "prefix", False, None, 20.0, True),
    (30, 300, 900, 4, 1, 32, "causal", False, None, 0.0, False),
    (3, 700, 700, 12, 2, 72, "prefix", True, None, 0.0, True),       # few key heads: their query heads are shared out and joined
    # up to 128 queries over many keys
    (3, 100, 2100, 6, 2, 64, "causal", True, (2100, 1400, 60), 0.0, False),
    (3, 128, 2304, 3, 1, 96, "prefix", True, None, 20.0, True),
    (3, 17, 4099, 5, 5, 40, "none", False, (4099, 0, 3), 0.0, True),
]


@pytest.mark.parametrize("prec", ("bfloat16", "half"))
@pytest.mark.parametrize("case", LONG)
def test_attention_over_many_tiles(device, case, prec):
    x, t, more, sl, seen, pos, scale = attention_case(case, prec)
    some = [0, case[0] // 2, case[0] - 1]          # sequences that are compared; all have to repeat their bits
    part = {n: v[some] for n, v in x.items()}
    out, lse, size, flat = R.attention(part["q"], part["k"], part["v"], seen[some], pos[some], scale, t["cap"], sl)
    nodes, op = link_attention(device, case, prec, {n: x[n] for n in "qkv"}, t, more, sl, "aligned")
    first = None
    for _ in range(6):
        op.run()
        got = nodes.read("out"), nodes.read("lse")
        first = first or got
        assert all(np.array_equal(f, g) for f, g in zip(first, got)), "the same inputs give the same bits"
    R.within(first[0][some], out, out_bound(prec, out, size, flat), "out")
    R.within(first[1][some], lse, R.ARITH * (1 + np.abs(np.where(np.isinf(lse), 0, lse))), "lse")
    x["out"], x["lse"] = first
    op.free()
    nodes.free()
    part = {n: v[some] for n, v in x.items()}
    want = R.attention_grad(part["q"], part["k"], part["v"], part["out"], part["lse"], part["d_out"], seen[some], pos[some], scale, t["cap"], sl, prec)
    nodes, op = link_attention(device, case, prec, x, t, more, sl, "aligned", grad=True)
    first = None
    for _ in range(6):
        op.run()
        got = [nodes.read(n) for n in ("dq", "dk", "dv")]
        first = first or got
        assert all(np.array_equal(f, g) for f, g in zip(first, got)), "the same inputs give the same bits"
    for n, got, (v, bound) in zip(("dq", "dk", "dv"), first, want):
        R.within(got[some], v, bound, n)
    op.free()
    nodes.free()
