"""Layer norm, rotary positions and attention as linked operators, against their definitions in 64 bits."""
import numpy as np
import pytest

from ocannl_b200 import backend as bk
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


def test_rotary_frequencies():
    f, m = bk.rotary_frequencies(64)
    assert m == 1.0 and f[0] == 1.0 and abs(f[31] - 10000.0 ** (-62 / 64)) < 1e-18
    g, _ = bk.rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert g[0] == 1.0 and abs(g[31] / f[31] * 8.0 - 1.0) < 1e-12
    y, m = bk.rotary_frequencies(64, scaling="yarn", factor=8.0)
    assert y[0] == f[0] and abs(y[31] / f[31] * 8.0 - 1.0) < 1e-12 and m > 1.0 and np.all(np.diff(y) < 0)
    with pytest.raises(bk.UserError):
        bk.rotary_frequencies(63)
    with pytest.raises(bk.UserError):
        bk.rotary_frequencies(64, scaling="unknown")


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
