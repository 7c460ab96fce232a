"""The operators at values, sizes and arguments where a kernel could go wrong, against their definitions in 64 bits."""
import numpy as np
import pytest

from ocannl_b200 import backend as bk
from ocannl_b200.low_level import Tnode
from ocannl_b200.workloads import load, store
from tests import operators_reference as R
from tests.test_operators_gpu import PRECS, attention_case, link_attention, out_bound
from tests import test_operators_gpu as T

pytestmark = pytest.mark.gpu


def check_forward(device, case, prec, x, t, more, sl, seen, pos, scale, sequences=None):
    """out and lse of one run against the definition, undefined and infinite values in the same places; `sequences`: those compared."""
    some = list(range(case[0])) if sequences is None else sequences
    with np.errstate(all="ignore"):
        out, lse, size, flat = R.attention(x["q"][some], x["k"][some], x["v"][some], seen[some], pos[some], scale, t["cap"], sl)
    nodes, op = link_attention(device, case, prec, {m: x[m] for m in "qkv"}, t, more, sl, "aligned")
    op.run()
    device.await_()
    got, got_lse = nodes.read("out")[some], nodes.read("lse")[some]
    op.free()
    nodes.free()
    with np.errstate(all="ignore"):
        bound = np.where(np.isfinite(out), out_bound(prec, np.where(np.isfinite(out), out, 0), np.where(np.isfinite(size), size, 0), np.where(np.isfinite(flat), flat, 0)), 0.0)
        R.within(got, out, bound, "out")
        R.within(got_lse, lse, R.ARITH * (1 + np.abs(np.where(np.isfinite(lse), lse, 0))), "lse")


# batch, queries, keys, heads, kv_heads, d, mask, documents, lengths, cap, slopes: a case for every forward kernel
SEEN = [
    (2, 1, 17, 4, 4, 64, "causal", False, None, 0.0, False),          # one row; a warp of four has the last key alone
    (2, 1, 17, 8, 2, 128, "causal", False, None, 20.0, True),         # four rows share the keys
    (2, 1, 700, 2, 2, 72, "none", False, (700, 513), 0.0, False),     # the keys in ranges, joined by the block that comes last
    (1, 5, 1500, 8, 1, 64, "causal", False, None, 0.0, False),         # joined by a launch of its own
    (1, 40, 1500, 2, 1, 40, "prefix", False, None, 30.0, True),       # more than 16 rows
    (2, 150, 150, 2, 2, 64, "causal", False, None, 0.0, False),       # tiles of 128 queries
    (2, 150, 150, 2, 1, 128, "causal", True, None, 20.0, True),
    (38, 260, 260, 4, 4, 72, "causal", False, None, 0.0, False),      # two tiles a block
]


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("what", ("query", "key", "keys of a sequence", "infinite key"))
@pytest.mark.parametrize("case", SEEN)
def test_undefined_values_that_are_seen_show(device, case, what, prec):
    """NaN in a query, in one visible key or in all of them, and an infinity in a key: undefined where the definition is."""
    x, t, more, sl, seen, pos, scale = attention_case(case, prec, seed=19)
    b, s, n = case[:3]
    rows, keys = seen.any(2), seen.any(1)
    at = [(i, np.flatnonzero(keys[i])[-1]) for i in {0, b - 1} if keys[i].any()]
    for i, j in at:
        if what == "query":
            x["q"][i, np.flatnonzero(rows[i])[0], 0, 0] = np.nan
        elif what == "key":
            x["k"][i, j, 0, 0] = np.nan
        elif what == "infinite key":
            x["k"][i, j, 0, 0] = np.inf
        else:
            x["k"][i, :, 0, 0] = np.nan
    check_forward(device, case, prec, x, t, more, sl, seen, pos, scale, sorted({0, b - 1}))


def relink(nodes, op, t, more, sl, grad, **kw):
    """The operator of `link_attention`'s nodes with other arguments."""
    op.free()
    kw = dict(dict(mask=t["mask"], cap=t["cap"], prefix="prefix" if "prefix" in more else None, lengths="lengths" if "lengths" in more else None,
                   slopes="slopes" if sl is not None else None), **kw)
    if grad:
        return nodes.context.attention_grad("q", "k", "v", "out", "lse", "d_out", "dq", "dk", "dv", **kw)
    return nodes.context.attention("q", "k", "v", "out", lse="lse", **kw)


# one node of documents: batch, queries, keys, heads, kv_heads, d, mask, documents, lengths, cap, slopes
ONE_NODE = [
    (3, 200, 200, 2, 1, 64, "causal", True, (200, 64, 131), 0.0, False),
    (3, 260, 260, 2, 2, 128, "none", True, (0, 260, 77), 0.0, False),
    (2, 140, 300, 4, 2, 40, "prefix", True, (170, 290), 20.0, True),
    (2, 300, 140, 2, 2, 72, "causal", True, None, 0.0, False),         # more queries than keys: the first have no position
    (4, 3, 90, 4, 2, 64, "causal", True, (1, 90, 50, 20), 0.0, False),
    (2, 1, 900, 4, 4, 128, "causal", True, (700, 300), 0.0, True),
    (2, 40, 1100, 2, 1, 64, "causal", True, (1000, 500), 0.0, False),
]


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("case", ONE_NODE)
def test_documents_in_one_node_go_by_position(device, case, prec):
    x, t, more, sl, _, _, scale = attention_case(case, prec, seed=23)
    b, s, n = case[:3]
    del more["qdoc"]
    lengths = np.full(b, n) if "lengths" not in more else more["lengths"]
    at = (lengths - s)[:, None] + np.arange(s)
    qdoc = np.where(at < 0, -1, np.take_along_axis(more["kdoc"], np.maximum(at, 0), 1))
    seen, pos = R.visible(b, s, n, case[6], more.get("prefix"), qdoc, more["kdoc"], more.get("lengths"))
    out, lse, size, flat = R.attention(x["q"], x["k"], x["v"], seen, pos, scale, t["cap"], sl)
    assert seen.any() and not np.isneginf(lse).all()
    nodes, op = link_attention(device, case, prec, {m: x[m] for m in "qkv"}, t, more, sl, "aligned")
    op = relink(nodes, op, t, more, sl, False, documents="kdoc")
    op.run()
    device.await_()
    R.within(nodes.read("out"), out, out_bound(prec, out, size, flat), "out")
    R.within(nodes.read("lse"), lse, R.ARITH * (1 + np.abs(np.where(np.isinf(lse), 0, lse))), "lse")
    op.free()
    nodes.free()
    x["out"], x["lse"] = R.rounded(prec, out), R.rounded("single", lse)
    want = R.attention_grad(x["q"], x["k"], x["v"], x["out"], x["lse"], x["d_out"], seen, pos, scale, t["cap"], sl, prec)
    nodes, op = link_attention(device, case, prec, x, t, more, sl, "aligned", grad=True)
    op = relink(nodes, op, t, more, sl, True, documents="kdoc")
    op.run()
    device.await_()
    for m, (v, bound) in zip(("dq", "dk", "dv"), want):
        R.within(nodes.read(m), v, bound, m)
    op.free()
    nodes.free()


@pytest.mark.parametrize("prec", ("bfloat16", "half"))
@pytest.mark.parametrize("queries,d,heads", [(1, 8, 1), (130, 8, 1), (130, 72, 1), (260, 128, 149)])
def test_sums_over_a_million_keys(device, queries, d, heads, prec):
    """Equal weights of one: the output is the values' mean, rounded once, however many keys there are."""
    n = 1_000_003 if heads == 1 else 100_003
    rng = np.random.default_rng(37)
    v = R.rounded(prec, 1.0 + rng.random((1, n, 1, d)))
    zero, q = np.zeros((1, n, 1, d)), np.zeros((1, queries, heads, d))
    nodes = R.Nodes(device, dict(q=(prec, q.shape, q), k=(prec, zero.shape, zero), v=(prec, v.shape, v), out=(prec, q.shape, None), lse=("single", (1, heads, queries), None)))
    op = nodes.context.attention("q", "k", "v", "out", lse="lse", mask="none")
    for _ in range(2):
        op.run()
    device.await_()
    want = np.broadcast_to(v.mean(1, keepdims=True), q.shape)
    R.within(nodes.read("out"), want, (R.EPS[prec] / 2 + 2.0 ** -12) * want, "out")
    R.within(nodes.read("lse"), np.full((1, heads, queries), np.log(n)), R.ARITH * 15, "lse")
    op.free()
    nodes.free()


@pytest.mark.parametrize("prec", ("bfloat16", "half"))
@pytest.mark.parametrize("case", [(1, 150, 40000, 1, 1, 16, "causal", False, None, 0.0, True), (1, 130, 34000, 1, 1, 72, "prefix", True, None, 20.0, False)])
def test_sums_over_many_keys_of_different_weights(device, case, prec):
    """Maxima that move between the times when accumulators are added to the sums; places that are not seen."""
    x, t, more, sl, seen, pos, scale = attention_case(case, prec, seed=41)
    x["k"] = R.rounded(prec, x["k"] * np.linspace(0.2, 3.0, case[2])[None, :, None, None])
    check_forward(device, case, prec, x, t, more, sl, seen, pos, scale)


@pytest.mark.parametrize("prec", ("bfloat16", "half"))
@pytest.mark.parametrize("queries", (1, 130))
def test_many_small_weights_beside_a_large_one(device, queries, prec):
    """A million keys of weight 2^-20 of the largest, which has the value 0: small weights keep the bits of their type."""
    n, d = 1_000_003, 8
    rng = np.random.default_rng(29)
    k, v = np.zeros((1, n, 1, d)), R.rounded(prec, 1.0 + rng.random((1, n, 1, d)))
    q = np.zeros((1, queries, 1, d))
    q[..., 0], k[0, 5, 0, 0], v[0, 5] = 1.0, 13.875, 0.0
    nodes = R.Nodes(device, dict(q=(prec, q.shape, q), k=(prec, k.shape, k), v=(prec, v.shape, v), out=(prec, q.shape, None), lse=("single", (1, 1, queries), None)))
    op = nodes.context.attention("q", "k", "v", "out", lse="lse", mask="none", scale=1.0)
    op.run()
    device.await_()
    small = np.exp(-13.875)
    total = 1.0 + (n - 1) * small
    want = v.sum(1, keepdims=True) * small / total
    # weights and the output are rounded once each; the sums in single precision
    R.within(nodes.read("out"), np.broadcast_to(want, q.shape), (R.EPS[prec] + R.ARITH) * want, "out")
    R.within(nodes.read("lse"), np.full((1, 1, queries), 13.875 + np.log(total)), R.ARITH * 15, "lse")
    op.free()
    nodes.free()


@pytest.mark.parametrize("prec", ("bfloat16", "half"))
def test_gradients_of_values_of_many_keys(device, prec):
    """Weights of one in a million, alike for all keys: dv is the sum of d_out's rows over a million."""
    n, s, d = 1_000_003, 130, 8
    rng = np.random.default_rng(31)
    do = R.rounded(prec, 1000.0 * (1.0 + rng.random((1, s, 1, d))))
    v = R.rounded(prec, rng.standard_normal((1, n, 1, d)))
    out = R.rounded(prec, np.broadcast_to(v.mean(1, keepdims=True), do.shape))
    zero, q = np.zeros((1, n, 1, d)), np.zeros((1, s, 1, d))
    nodes = R.Nodes(device, dict(q=(prec, q.shape, q), k=(prec, zero.shape, zero), v=(prec, v.shape, v), out=(prec, q.shape, out), d_out=(prec, q.shape, do),
                                 lse=("single", (1, 1, s), np.full((1, 1, s), np.log(n))), dq=(prec, q.shape, None), dk=(prec, zero.shape, None), dv=(prec, zero.shape, None)))
    op = nodes.context.attention_grad("q", "k", "v", "out", "lse", "d_out", "dq", "dk", "dv", mask="none")
    op.run()
    device.await_()
    want = np.broadcast_to(do.sum(1, keepdims=True) / n, zero.shape)
    R.within(nodes.read("dv"), want, (R.EPS[prec] + R.ARITH) * want, "dv")
    assert not nodes.read("dq").any() and not nodes.read("dk").any()
    op.free()
    nodes.free()


R.EPS["half, scaled"] = R.EPS["half"]       # a half's steps, without what the scales of gradients add: see below


def scaled_grad(x, seen, pos, scale, cap, sl):
    """The gradients of half heads and how far each may be: score gradients lie within 2^13 and 2^14 of the bound of their own row
    (a query's |d_out| (max |v| + |out|); a key's max |d_out| |v| + max |d_out| |out|, over its sequence and the heads that share it), so
    that half a step below the normal numbers, 2^-25, is 2^-38 of it; weights are stored times 2^14: 2^-39."""
    b, s, h, d = x["q"].shape
    n, hk = x["k"].shape[1:3]
    want = R.attention_grad(x["q"], x["k"], x["v"], x["out"], x["lse"], x["d_out"], seen, pos, scale, cap, sl, "half, scaled")
    of = {m: np.linalg.norm(x[m], axis=-1) for m in ("d_out", "out", "v")}
    more = [np.zeros_like(a) for a, _ in want]
    for i in range(b):
        for g in range(h):
            k = g // (h // hk)
            rows, keys = seen[i].any(1), seen[i].any(0)
            heads = slice(k * (h // hk), (k + 1) * (h // hk))
            top = of["d_out"][i][rows][:, heads].max(initial=0.0)
            both = (of["d_out"][i] * of["out"][i])[rows][:, heads].max(initial=0.0)
            mine = of["d_out"][i, :, g] * (of["v"][i, keys, k].max(initial=0.0) + of["out"][i, :, g])
            theirs = top * of["v"][i, :, k] + both
            more[0][i, :, g] += scale * 2.0 ** -38 * mine[:, None] * (seen[i] @ np.abs(x["k"][i, :, k]))
            more[1][i, :, k] += scale * 2.0 ** -38 * theirs[:, None] * (seen[i].T @ np.abs(x["q"][i, :, g]))
            more[2][i, :, k] += 2.0 ** -39 * (seen[i].T @ np.abs(x["d_out"][i, :, g]))
    return [(v, bound + m + 2.0 ** -25) for (v, bound), m in zip(want, more)]


# batch, queries, keys, heads, kv_heads, d, mask, documents, lengths, cap, slopes
SCALED = [
    (2, 512, 512, 2, 2, 64, "none", False, None, 0.0, False),
    (2, 700, 700, 2, 1, 128, "causal", False, None, 20.0, False),
    (2, 300, 900, 3, 1, 40, "prefix", True, (900, 700), 0.0, True),
]


@pytest.mark.parametrize("of_v", (1.0, 2.0 ** -6, 100.0))
@pytest.mark.parametrize("case", SCALED)
def test_half_gradients_of_different_sizes(device, case, of_v):
    """Rows, heads and sequences of d_out that differ by 10^4, small and large values: each keeps the bits that its own size allows."""
    x, t, more, sl, seen, pos, scale = attention_case(case, "half", seed=43)
    x["v"] = R.rounded("half", x["v"] * of_v)
    rows = np.flatnonzero(seen[0].any(1))
    x["d_out"] = x["d_out"] * 0.1
    x["d_out"][0, rows[len(rows) // 2], 0] *= 1e4      # one row of a head
    x["d_out"][1] *= 1e3                               # a sequence
    x["d_out"] = R.rounded("half", x["d_out"])
    out, lse, _, _ = R.attention(x["q"], x["k"], x["v"], seen, pos, scale, t["cap"], sl)
    x["out"], x["lse"] = R.rounded("half", out), R.rounded("single", lse)
    nodes, op = link_attention(device, case, "half", x, t, more, sl, "aligned", grad=True)
    op.run()
    device.await_()
    for m, (v, bound) in zip(("dq", "dk", "dv"), scaled_grad(x, seen, pos, scale, t["cap"], sl)):
        assert np.abs(v).max() < 65504.0, m
        R.within(nodes.read(m), v, bound, m)
    op.free()
    nodes.free()


def test_keys_beyond_what_classes_of_tiles_have_room_for(device):
    """Ten million keys: without documents nothing is kept of their tiles; with them the call is refused."""
    n, s, d = 10_600_000, 130, 8
    rng = np.random.default_rng(47)
    q, do = np.zeros((1, s, 1, d)), R.rounded("bfloat16", 1e6 * (1.0 + rng.random((1, s, 1, d))))
    nodes = R.Nodes(device, dict(q=("bfloat16", q.shape, q), out=("bfloat16", q.shape, None), lse=("single", (1, 1, s), None), d_out=("bfloat16", q.shape, do),
                                 dq=("bfloat16", q.shape, None), docs=("int32", (1, n), np.zeros((1, n))),
                                 **{m: ("bfloat16", (1, n, 1, d), None if m in ("dk", "dv") else np.full((1, n, 1, d), of)) for m, of in (("k", 0.0), ("v", 1.5), ("dk", 0.0), ("dv", 0.0))}))
    ctx, args = nodes.context, ("q", "k", "v", "out")
    back = args + ("lse", "d_out", "dq", "dk", "dv")
    for refused in (lambda: ctx.attention(*args, documents="docs"), lambda: ctx.attention_grad(*back, documents="docs")):
        with pytest.raises(bk.B200Error) as e:
            refused()
        assert e.value.code == -4 and "too many keys" in str(e.value)
    ops = [ctx.attention(*args, lse="lse", mask="none"), ctx.attention_grad(*back, mask="none")]
    for op in ops:
        op.run()
    device.await_()
    assert np.array_equal(nodes.read("out"), np.full(q.shape, 1.5))
    R.within(nodes.read("lse"), np.full((1, 1, s), np.log(n)), R.ARITH * 17, "lse")
    want = np.broadcast_to(do.sum(1, keepdims=True) / n, (1, n, 1, d))
    R.within(nodes.read("dv"), want, (R.EPS["bfloat16"] + 16 * R.ARITH) * want, "dv")      # (p from an lse of up to 16, in single precision)
    for op in ops:
        op.free()
    nodes.free()


# two tiles of queries a block, tiles of which one sees keys that the other does not, documents in all of them
TWO_TILES = [
    (20, 1030, 1030, 4, 2, 128, "causal", True, None, 30.0, False),
    (20, 1030, 1030, 4, 2, 128, "causal", True, None, 0.0, False),
    (19, 700, 900, 4, 1, 96, "prefix", True, None, 0.0, True),
    (38, 513, 513, 2, 2, 72, "none", True, tuple(513 - 13 * i for i in range(38)), 20.0, True),
]


@pytest.mark.parametrize("prec", ("bfloat16", "half"))
@pytest.mark.parametrize("case", TWO_TILES)
def test_two_tiles_of_queries_with_documents(device, case, prec):
    T.test_attention_over_many_tiles(device, case, prec)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("rows,n", [(2, 16400), (3, 20001), (1, 70000)])
def test_wide_rows_of_the_norm(device, rows, n, prec):
    T.test_layer_norm(device, rows, n, prec)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("rows,n", [(70, 28672), (70, 28680), (65, 30001), (3, 70000)])
def test_wide_rows_of_the_norms_gradients(device, rows, n, prec):
    T.test_layer_norm_grad(device, rows, n, prec)


@pytest.mark.parametrize("prec", ("bfloat16", "half"))
def test_tiles_and_gradients_behind_two_to_the_31(device, prec):
    """130 queries over 2.1 million positions, 2^31 elements and more of k, v, dk and dv.  All keys are zero, so all weights are equal; all
    values but the last are zero."""
    n, hk, d, s, tail = 2_100_000, 8, 128, 130, 64
    assert n * hk * d > 2 ** 31
    rng = np.random.default_rng(53)
    pools = {m: device.alloc_pool(n * hk * d * 2) for m in ("k", "v", "dk", "dv")}
    for p in pools.values():
        device.memset_zero(p, 0, n * hk * d * 2)
    last = R.rounded(prec, rng.standard_normal((tail, hk, d)) * n / 1000)
    device.from_host(pools["v"], (n - tail) * hk * d * 2, store(prec, last.astype(np.float32)))
    do = R.rounded(prec, 1000.0 * rng.standard_normal((1, s, hk, d)))
    mean = last.sum(0) / n
    out = R.rounded(prec, np.broadcast_to(mean, (1, s, hk, d)))
    nodes = R.Nodes(device, dict(q=(prec, do.shape, np.ones(do.shape)), out=(prec, do.shape, None), lse=("single", (1, hk, s), None), given=(prec, do.shape, out),
                                 d_out=(prec, do.shape, do), dq=(prec, do.shape, None)))
    arrays = dict(nodes.context.arrays, **{m: (p, 0, Tnode(90 + i, m, prec, (1, n, hk, d))) for i, (m, p) in enumerate(pools.items())})
    ctx = bk.Context(device, arrays)
    ops = [ctx.attention("q", "k", "v", "out", lse="lse", mask="none"), ctx.attention_grad("q", "k", "v", "given", "lse", "d_out", "dq", "dk", "dv", mask="none")]
    for op in ops:
        op.run()
    device.await_()
    half = R.EPS[prec] / 2
    # equal weights of one; sums of n of them and of 64 products in single precision, added in parts
    R.within(nodes.read("out"), np.broadcast_to(mean, do.shape), half * np.abs(mean) + 2.0 ** -12 * np.abs(last).sum(0) / n + 2.0 ** -25, "out")
    R.within(nodes.read("lse"), np.full((1, hk, s), np.log(n)), R.ARITH * 16, "lse")
    assert not nodes.read("dq").any()
    delta = (do * out).sum(-1)[0]                                        # [s, hk]
    for first, v in ((0, np.zeros((2, hk, d))), (n // 2, np.zeros((2, hk, d))), (n - tail - 2, np.concatenate([np.zeros((2, hk, d)), last]))):
        rows = v.shape[0]
        dp = np.einsum("rhd,jhd->rjh", do[0], v)
        ds, size = (dp - delta[:, None]) / n, (np.abs(np.einsum("rhd,jhd->rjh", np.abs(do[0]), np.abs(v))) + np.abs(do * out).sum(-1)[0][:, None]) / n
        want = {"dv": np.broadcast_to(do[0].sum(0) / n, v.shape), "dk": np.broadcast_to(ds.sum(0)[..., None] / np.sqrt(d), v.shape)}
        # weights and score gradients are rounded once; p comes from an lse of 15 in single precision
        off = {"dv": (half + 16 * R.ARITH) * np.abs(do[0]).sum(0) / n,
               "dk": (((half + 16 * R.ARITH) * np.abs(ds) + 2.0 ** -20 * size).sum(0) / np.sqrt(d))[..., None]}
        for m in ("dv", "dk"):
            host = np.empty((rows, hk, d), np.float16 if prec == "half" else np.uint16)
            device.to_host(pools[m], first * hk * d * 2, host)
            device.await_()
            R.within(load(prec, host), want[m], off[m] + half * np.abs(want[m]) + 2.0 ** -25, m)
    for op in ops:
        op.free()
    for p in pools.values():
        device.free_pool(p)
    nodes.free()


@pytest.mark.parametrize("rows,n", [(9472, 64), (9472, 40), (700, 28680)])
def test_column_sums_of_the_norms_gradients(device, rows, n):
    """Rows that are all alike, of a value whose last bits a running sum in single precision drops once it has reached 32."""
    c = float(np.float32(1 + 2.0 ** -19 - 2.0 ** -23))
    same = lambda v: ("single", (rows, n), np.full((rows, n), v, np.float32))  # noqa: E731
    nodes = R.Nodes(device, dict(x=same(1.0), dy=same(c), dx=("single", (rows, n), None), mean=("single", (rows,), np.zeros(rows)), rstd=("single", (rows,), np.ones(rows)),
                                 dg=("single", (n,), None), db=("single", (n,), None)))
    op = nodes.context.layer_norm_grad("x", "dy", "dx", "mean", "rstd", dgamma="dg", dbeta="db")
    op.run()
    # a thread's own rows (one to four of them here, or a slice in double), a block's sum and the result are rounded
    for name in ("dg", "db"):
        R.within(nodes.read(name), np.full(n, rows * c), 6 * 2.0 ** -24 * rows * c, name)
    op.free()
    nodes.free()


def test_single_precision_weights_of_large_scores(device):
    """Every query sees one key, with scores of up to 60 and an lse that is the score: weights of one."""
    n, d = 200, 16
    rng = np.random.default_rng(59)
    q, k = np.zeros((1, n, 1, d)), np.zeros((1, n, 1, d))
    q[0, :, 0, 0], k[..., 0] = np.arange(n) + 1, 1.0
    scale = np.float32(0.3)
    lse = (q[0, :, 0, 0].astype(np.float32) * scale).astype(np.float32)
    v, do = (R.rounded("single", rng.standard_normal((1, n, 1, d))) for _ in range(2))
    single = lambda a: ("single", a.shape, a)  # noqa: E731
    nodes = R.Nodes(device, dict(q=single(q), k=single(k), v=single(v), out=single(v), d_out=single(do), lse=single(lse.reshape(1, 1, n)), docs=("int32", (1, n), np.arange(n)[None]),
                                 dq=("single", q.shape, None), dk=("single", q.shape, None), dv=("single", q.shape, None)))
    op = nodes.context.attention_grad("q", "k", "v", "out", "lse", "d_out", "dq", "dk", "dv", documents="docs", scale=float(scale))
    op.run()
    # two tf32 parts keep 2^-21 of each operand
    R.within(nodes.read("dv"), do, 2.0 ** -20 * np.abs(do) + 1e-30, "dv")
    op.free()
    nodes.free()


@pytest.mark.parametrize("scale,cap,words", [(3e38, 0.0, "scale is too large"), (0.125, 1e-45, "cap is too far"), (0.125, 1e38, "cap is too far"), (1e-30, 3e9, "cap is too far"),
                                             (0.125, 3e38, "cap is too far")])
def test_scales_and_caps_that_scores_cannot_have(device, scale, cap, words):
    one = ("bfloat16", (1, 2, 1, 16), np.ones((1, 2, 1, 16)))
    nodes = R.Nodes(device, dict(q=one, k=one, v=one, out=("bfloat16", (1, 2, 1, 16), None)))
    with pytest.raises(bk.B200Error) as e:
        nodes.context.attention("q", "k", "v", "out", scale=scale, cap=cap)
    assert e.value.code == -1 and words in str(e.value)
    nodes.free()


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("scale,cap", [(1e-30, 1e-30), (1e30, 0.0), (0.125, 1e30)])
def test_scales_and_caps_far_from_one(device, scale, cap, prec):
    """Scores of 1e-30 weigh all keys alike; those of 1e30 the largest alone; a cap far above the scores changes none."""
    rng = np.random.default_rng(61)
    n, d = 40, 16
    q, k, v = (R.rounded(prec, rng.standard_normal((1, n, 1, d))) for _ in range(3))
    nodes = R.Nodes(device, dict(q=(prec, q.shape, q), k=(prec, k.shape, k), v=(prec, v.shape, v), out=(prec, q.shape, None)))
    op = nodes.context.attention("q", "k", "v", "out", mask="none", scale=scale, cap=cap)
    op.run()
    device.await_()
    seen, pos = R.visible(1, n, n, "none")
    out, _, size, flat = R.attention(q, k, v, seen, pos, float(np.float32(scale)), float(np.float32(cap)))
    R.within(nodes.read("out"), out, out_bound(prec, out, size, flat), "out")
    op.free()
    nodes.free()


@pytest.mark.parametrize("case", [(2, 400, 400, 2, 1, 64, "causal", True, None, 0.0, False), (2, 300, 500, 2, 2, 128, "causal", True, (450, 333), 0.0, True)])
def test_half_gradients_beside_large_values_that_are_not_seen(device, case):
    """Values of 60000 at padding and behind the lengths take nothing from the gradients of values of 2^-8."""
    x, t, more, sl, seen, pos, scale = attention_case(case, "half", seed=67)
    keys = seen.any(1)
    x["v"] = R.rounded("half", np.where(keys[:, :, None, None], x["v"] * 2.0 ** -8, 60000.0))
    x["k"] = R.rounded("half", np.where(keys[:, :, None, None], x["k"], 200.0))
    out, lse, _, _ = R.attention(x["q"], x["k"], x["v"], seen, pos, scale, t["cap"], sl)
    x["out"], x["lse"] = R.rounded("half", out), R.rounded("single", lse)
    nodes, op = link_attention(device, case, "half", x, t, more, sl, "aligned", grad=True)
    op.run()
    device.await_()
    for m, (v, bound) in zip(("dq", "dk", "dv"), scaled_grad(x, seen, pos, scale, t["cap"], sl)):
        R.within(nodes.read(m), v, bound, m)
    op.free()
    nodes.free()
