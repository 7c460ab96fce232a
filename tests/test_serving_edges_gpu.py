"""The operators over a paged cache and the choice of tokens together, captured, and where they can go wrong: undefined values that are seen and that are not,
shared and far pages, nothing to do, calls that are refused."""
import numpy as np
import pytest

from ocannl_b200 import backend as bk
from ocannl_b200.low_level import Tnode
from tests import serving_reference as R
from tests.test_serving_gpu import ATTEND, PROMPTS, TILES, append_case, append_nodes, attend_case, attend_nodes, check_attend, link_append, link_attend, want_attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("prec", ["bfloat16", "single"])
def test_a_prompt_and_the_tokens_behind_it(device, prec, coded):
    """Prompts of several lengths are appended and attended to, then step by step a token a sequence, captured into one graph with its choice; pages are
    handed out as they are needed.  A second set of the same operators runs in between."""
    import torch
    rng = np.random.default_rng(31)
    b, page, hk, h, d, prompts, steps = 3, 16, 2, 4, 64, [21, 1, 40], 12
    most, pages, f = 4, 14, 10000.0 ** (-np.arange(32) / 32)
    first = sum(prompts)
    cache = {g: np.full((pages, hk, page, d), 0x7f, np.uint8) if coded else np.full((pages, hk, page, d), np.nan) for g in ("k_cache", "v_cache")}
    scales = {g: np.full((pages, hk), np.nan) for g in ("k_scale", "v_scale")} if coded else {}
    arrays = {g: ("byte" if coded else prec, a.shape, a) for g, a in cache.items()}
    arrays.update({g: ("single", a.shape, a) for g, a in scales.items()})
    arrays.update(pages=("int32", (b, most), None), lengths=("int32", (b,), None), starts=("int32", (b + 1,), np.concatenate([[0], np.cumsum(prompts)])))
    for n, rows in (("p", first), ("t", b)):
        arrays.update({n + "q": (prec, (rows, h, d), None), n + "k": (prec, (rows, hk, d), None), n + "v": (prec, (rows, hk, d), None), n + "out": (prec, (rows, h, d), None)})
    arrays.update(u=("single", (b,), None), tokens=("int32", (b,), None), logprob=("single", (b,), None))
    sets = []
    for _ in range(2):
        nodes = R.Nodes(device, arrays)
        ctx = nodes.context
        pool, off, _ = ctx.arrays["tout"]
        ctx.arrays["logits"] = (pool, off, Tnode(99, "logits", prec, (b, h * d)))      # (what a model's head would make of it)
        where = dict(pages="pages", lengths="lengths", **({g: g for g in scales}))
        ops = {}
        for n, starts in (("p", "starts"), ("t", None)):
            ops[n] = [ctx.cache_append(n + "k", n + "v", "k_cache", "v_cache", q=n + "q", q_out=n + "q", frequencies=f, starts=starts, **where),
                      ctx.cache_attention(n + "q", "k_cache", "v_cache", n + "out", starts=starts, window=30, sinks=2, **where)]
        ops["t"].append(ctx.sample("logits", "u", "tokens", temperature=0.5, top_k=20, top_p=0.9, logprob="logprob"))
        sets.append((nodes, ops))
    (nodes, ops), (others, other_ops) = sets
    table, lengths = np.full((b, most), -1), np.array(prompts)
    free = list(rng.permutation(pages))

    def hand_out():
        for i in range(b):
            for k in range(-(-int(lengths[i]) // page)):
                if table[i, k] < 0:
                    table[i, k] = free.pop()
        for n in (nodes, others):
            n.write("pages", table)
            n.write("lengths", lengths)

    held = dict(cache, **scales)

    def check(n, x, starts):
        nonlocal held
        want, off = R.append({**x, **held}, prec, table, lengths, starts, page, f)
        for g in cache:
            if coded:
                assert np.array_equal(nodes.read(g[0] + "_scale")[table[table >= 0]], want[g[0] + "_scale"][table[table >= 0]])
                by = np.where(np.isnan(want[g[0] + "_scale"]), 1.0, want[g[0] + "_scale"])[:, :, None, None]
                R.within(R.decode(nodes.raw(g)) * by, R.decode(want[g]) * by, 2 * off[g], g)
            else:
                R.within(nodes.read(g), want[g], off[g], g)
        q = nodes.read(n + "q")
        R.within(q, want["q_out"], off["q_out"], "q")
        # attention of what the device has
        held = {g: nodes.raw(g) if coded else nodes.read(g) for g in cache}
        held.update({g: nodes.read(g) for g in scales})
        out, _, bound, _ = R.attention(q, held["k_cache"], held["v_cache"], table, lengths, starts, page, prec, held.get("k_scale"), held.get("v_scale"), window=30, sinks=2)
        R.within(nodes.read(n + "out"), out, bound, "out")

    def inputs(n, rows):
        x = {g: R.rounded(prec, rng.standard_normal((rows, h if g == "q" else hk, d)) * 2.0) for g in "qkv"}
        for s, scale in ((nodes, 1.0), (others, 0.5)):
            for g, a in x.items():
                s.write(n + g, a * scale)
        return x

    hand_out()
    x = inputs("p", first)
    for o, p in zip(ops["p"], other_ops["p"]):
        o.run()
        p.run()
    device.await_()
    check("p", x, np.concatenate([[0], np.cumsum(prompts)]))
    stream = torch.cuda.ExternalStream(device.stream_handle())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for o in ops["t"]:
            o.run()
    for i in range(steps):
        lengths = lengths + 1
        hand_out()
        x = inputs("t", b)
        u = R.rounded("single", rng.random(b))
        nodes.write("u", u)
        for o in other_ops["t"][:2]:
            o.run()
        with torch.cuda.stream(stream):
            graph.replay()
        other_ops["t"][1].run()
        device.await_()
        check("t", x, None)
        logits = nodes.read("tout").reshape(b, -1)
        for r in range(b):
            assert nodes.read("tokens")[r] == R.sample(logits[r], u[r], 0.5, 20, 0.9)[0]
    del graph
    for s, o in sets:
        for op in o["p"] + o["t"]:
            op.free()
        s.free()


EVERY = [ATTEND[1], ATTEND[3], ATTEND[5], ATTEND[8], ATTEND[9], PROMPTS[1], PROMPTS[4], PROMPTS[9], TILES[1], TILES[4]]


@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("prec", ["bfloat16", "half", "single"])
@pytest.mark.parametrize("what", ["query", "key", "value", "infinite value"])
@pytest.mark.parametrize("case", EVERY)
def test_undefined_values_that_are_seen(device, case, what, prec, coded):
    """... reach the rows that see them, and no others: what the last token brings is behind all rows but the last."""
    x, table, lengths, starts, page, t = attend_case(case, prec, coded, seed=41)
    b = int(np.argmax(lengths))
    rows = R.rows_of(lengths, starts, x["q"].shape[0], table.shape[0])[b][0]
    p, s = R.place(table, x["k_cache"].shape[0], page, b, int(lengths[b]) - 1)
    if what == "query":
        x["q"][rows[-1], 0, 0] = np.nan
    elif coded:
        x["k_cache" if what == "key" else "v_cache"][p, 0, s, 0] = 0x7f
    else:
        x["k_cache" if what == "key" else "v_cache"][p, 0, s, 0] = np.inf if what == "infinite value" else np.nan
    with np.errstate(all="ignore"):
        want = want_attend(x, table, lengths, starts, page, prec, t)
    assert not np.isfinite(want[0][rows[-1]]).all() and np.isfinite(want[0][rows[:-1]]).all()
    nodes = attend_nodes(device, x, prec, table, lengths, starts)
    op = link_attend(nodes, x, starts, t)
    op.run()
    device.await_()
    # (other elements of an undefined row, and bounds of rows that are none)
    out, lse, off, lse_off = want
    R.within(nodes.read("out"), out, np.where(np.isfinite(off), off, 0.0), "out")
    R.within(nodes.read("lse"), lse, np.where(np.isfinite(lse_off), lse_off, 0.0), "lse")
    op.free()
    nodes.free()


@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("case", [ATTEND[1], ATTEND[4], PROMPTS[1], TILES[1]])
def test_pages_of_several_sequences(device, case, coded):
    """Two sequences with one beginning."""
    case = (2,) + case[1:] if isinstance(case[1], int) else (2, case[1][:2]) + case[2:]
    case = case[:2] + (case[2][:2],) + case[3:]
    x, table, lengths, starts, page, t = attend_case(case, "bfloat16", coded, stale=1.0)
    shared = min(int(lengths.min()) // page, table.shape[1])
    table[1, :shared] = table[0, :shared]
    want = want_attend(x, table, lengths, starts, page, "bfloat16", t)
    nodes = attend_nodes(device, x, "bfloat16", table, lengths, starts)
    op = link_attend(nodes, x, starts, t)
    op.run()
    device.await_()
    check_attend(nodes, want)
    op.free()
    nodes.free()


@pytest.mark.parametrize("coded,new", [(True, 1), (True, 200), (False, 1), (False, 200)])
def test_pages_behind_4_gb(device, coded, new):
    """The first page of a cache of 4.5 GB, one in the middle and the last ones: appended to and attended to."""
    rng = np.random.default_rng(51)
    hk, page, d, h = 4, 64, 128, 8
    each = hk * page * d * (1 if coded else 2)
    pages = int(4.5 * 2 ** 30) // each
    length = max(new, 200) + 20
    table = np.array([[0, pages - 1, pages // 2, pages - 2][:-(-length // page)]])
    small = np.arange(table.shape[1])[None]                # the same pages of a small cache, for the restatement
    nodes = R.Nodes(device, dict(k_cache=("byte", (0, hk, page, d), None), pages=("int32", table.shape, table), lengths=("int32", (1,), [length]),
                                 q=("bfloat16", (new, h, d), None), k=("bfloat16", (new, hk, d), None), v=("bfloat16", (new, hk, d), None), out=("bfloat16", (new, h, d), None),
                                 k_scale=("single", (pages, hk), np.full((pages, hk), 2.0 ** -6)), v_scale=("single", (pages, hk), np.full((pages, hk), 2.0 ** -6))))
    x = {g: R.rounded("bfloat16", rng.standard_normal((new, h if g == "q" else hk, d))) for g in "qkv"}
    for g, a in x.items():
        nodes.write(g, a)
    old, pools = {}, []
    for g in ("k_cache", "v_cache"):
        pool = device.alloc_pool(pages * each)
        pools.append(pool)
        nodes.context.arrays[g] = (pool, 0, Tnode(90 + len(pools), g, "byte" if coded else "bfloat16", (pages, hk, page, d)))
        values = rng.standard_normal((table.shape[1], hk, page, d))
        old[g] = R.encode(values * 64.0) if coded else R.rounded("bfloat16", values)
        for i, p in enumerate(table[0]):
            a = old[g][i] if coded else R.store("bfloat16", old[g][i].astype(np.float32))
            device.from_host(pool, int(p) * each, np.ascontiguousarray(a))
            device.await_()
    scales = dict(k_scale="k_scale", v_scale="v_scale") if coded else {}
    f = 10000.0 ** (-np.arange(64) / 64)
    ops = [nodes.context.cache_append("k", "v", "k_cache", "v_cache", "pages", "lengths", frequencies=f, **scales),
           nodes.context.cache_attention("q", "k_cache", "v_cache", "out", "pages", "lengths", **scales)]
    for op in ops:
        op.run()
    device.await_()
    n = table.shape[1]
    sc = {g: np.full((n, hk), 2.0 ** -6) for g in scales}
    want, off = R.append({"k": x["k"], "v": x["v"], **old, **sc}, "bfloat16", small, [length], None, page, f)
    got = {}
    for g, pool in zip(("k_cache", "v_cache"), pools):
        a = np.empty((n, hk, page, d), np.uint8 if coded else np.uint16)
        for i, p in enumerate(table[0]):
            one = np.empty((hk, page, d), a.dtype)
            device.to_host(pool, int(p) * each, one)
            device.await_()
            a[i] = one
        if coded:
            by = want[g[0] + "_scale"][:, :, None, None]
            got[g] = a
            R.within(R.decode(a) * by, R.decode(want[g]) * by, 2 * off[g], g)
        else:
            got[g] = R.load("bfloat16", a).astype(np.float64)
            R.within(got[g], want[g], off[g], g)
    out, _, bound, _ = R.attention(x["q"], got["k_cache"], got["v_cache"], small, [length], None, page, "bfloat16", want.get("k_scale"), want.get("v_scale"))
    R.within(nodes.read("out"), out, bound, "out")
    for op in ops:
        op.free()
    for pool in pools:
        device.free_pool(pool)
    del nodes.context.arrays["k_cache"], nodes.context.arrays["v_cache"]
    nodes.free()


@pytest.mark.parametrize("coded", [False, True])
def test_starts_beyond_the_rows(device, coded):
    """Numbers of rows are taken between none and all of them."""
    case = (3, [2, 3, 4], [20, 30, 7], 16, 2, 4, 64, 0, 0, 0.0, False)
    x, table, lengths, starts, page, t = attend_case(case, "bfloat16", coded, extra=0)
    for starts in (np.array([-5, 2, 5, 1000]), np.array([3, 3, 9, 9])):
        want = want_attend(x, table, lengths, starts, page, "bfloat16", t)
        nodes = attend_nodes(device, x, "bfloat16", table, lengths, starts)
        op = link_attend(nodes, x, starts, t)
        op.run()
        device.await_()
        check_attend(nodes, want)
        op.free()
        nodes.free()
    case = (3, [2, 3, 4], [20, 30, 7], 16, 2, 4, 64, 32, "half")
    x, table, lengths, _, page, f, layout = append_case(case, "bfloat16", coded, extra=0)
    for starts in (np.array([-5, 2, 5, 1000]), np.array([3, 3, 9, 9])):
        want, off = R.append(x, "bfloat16", table, lengths, starts, page, f, layout)
        nodes = append_nodes(device, x, "bfloat16", table, lengths, starts)
        op = link_append(nodes, x, starts, f, layout)
        op.run()
        device.await_()
        R.within(nodes.read("q_out"), want["q_out"], off["q_out"], "q_out")
        for g in "kv":
            by = want[g + "_scale"][:, :, None, None] if coded else 1.0
            R.within(R.decode(nodes.raw(g + "_cache")) * by if coded else nodes.read(g + "_cache"), R.decode(want[g + "_cache"]) * by if coded else want[g + "_cache"],
                     2 * off[g + "_cache"], g)
        op.free()
        nodes.free()


def test_nothing_to_do(device):
    """No rows, no sequences, no pages, no tokens of a sequence."""
    one = np.ones
    for tokens, b, pages, most in ((0, 2, 3, 2), (0, 0, 3, 2), (4, 2, 0, 2), (4, 2, 3, 0)):
        for prec in ("bfloat16", "single"):
            nodes = R.Nodes(device, dict(q=(prec, (tokens, 2, 64), one((tokens, 2, 64))), k=(prec, (tokens, 2, 64), one((tokens, 2, 64))), out=(prec, (tokens, 2, 64), None),
                                         lse=("single", (tokens, 2), None), c=(prec, (pages, 2, 16, 64), one((pages, 2, 16, 64))), d=(prec, (pages, 2, 16, 64), one((pages, 2, 16, 64))),
                                         pages=("int32", (b, most), np.zeros((b, most))), lengths=("int32", (b,), np.full(b, 2))))
            ops = [nodes.context.cache_append("k", "k", "c", "d", "pages", "lengths"), nodes.context.cache_attention("q", "c", "d", "out", "pages", "lengths", lse="lse")]
            for op in ops:
                op.run()
            device.await_()
            if tokens and not (pages and most):
                assert np.array_equal(nodes.read("out"), np.zeros((tokens, 2, 64))) and np.all(nodes.read("lse") == -np.inf)
            for op in ops:
                op.free()
            nodes.free()
    nodes = R.Nodes(device, dict(x=("half", (0, 5), None), u=("single", (0,), None), t=("int32", (0,), None)))
    op = nodes.context.sample("x", "u", "t")
    op.run()
    device.await_()
    op.free()
    nodes.free()


def test_refusals(device):
    bf = "bfloat16"
    nodes = R.Nodes(device, dict(q=(bf, (6, 4, 64), None), out=(bf, (6, 4, 64), None), k=(bf, (6, 2, 64), None), v=(bf, (6, 2, 64), None), c=(bf, (5, 2, 8, 64), None), d=(bf, (5, 2, 8, 64), None),
                                 pages=("int32", (3, 4), None), lengths=("int32", (3,), None), pages4=("int32", (4, 4), None), lengths4=("int32", (4,), None), odd=(bf, (6, 3, 64), None),
                                 wide=(bf, (6, 2, 136), None), cw=(bf, (5, 2, 8, 136), None), x=(bf, (5, 9), None), u=("single", (5,), None), t=("int32", (5,), None),
                                 f32=("single", (6, 2, 64), None), scale=("single", (5, 2), None)))
    c = nodes.context
    attn = lambda **more: c.cache_attention("q", "c", "d", "out", "pages", "lengths", **more)  # noqa: E731
    for call, code, words in (
            (lambda: c.cache_append("k", "v", "c", "d", "pages4", "lengths4"), -1, "multiple of batch"),
            (lambda: c.cache_append("k", "v", "c", "c", "pages", "lengths"), -1, "overlaps"),
            (lambda: c.cache_append("k", "v", "c", "d", "pages", "lengths", frequencies=np.ones(33)), -1, "2 * pairs"),
            (lambda: c.cache_append("k", "v", "c", "d", "pages", "lengths", frequencies=[np.nan]), -1, "not finite"),
            (lambda: c.cache_append("k", "v", "c", "d", "pages", "lengths", frequencies=[1.0], magnitude=np.inf), -1, "magnitude"),
            (lambda: c.cache_attention("odd", "c", "d", "odd", "pages", "lengths"), -1, "multiple of kv_heads"),
            (lambda: c.cache_attention("q", "c", "d", "q", "pages", "lengths"), -1, "overlaps"),
            (lambda: c.cache_attention("wide", "cw", "cw", "wide", "pages", "lengths"), -4, "more than 128"),
            (lambda: attn(window=-1), -1, "window and sinks"), (lambda: attn(sinks=-1), -1, "window and sinks"), (lambda: attn(scale=-1.0), -1, "scale must"),
            (lambda: attn(scale=3e38), -1, "scale is too large"), (lambda: attn(cap=-1.0), -1, "cap must"), (lambda: attn(scale=0.1, cap=1e38), -1, "cap is too far"),
            (lambda: c.sample("x", "u", "t", temperature=float("nan")), -1, "undefined"), (lambda: c.sample("x", "u", "t", logprob="u"), -1, "overlaps")):
        with pytest.raises(bk.B200Error) as e:
            call()
        assert e.value.code == code and words in str(e.value), words
    nodes.free()


def test_numbers_to_keep_that_pass_32_bits(device):
    """As many as there are, or none: all."""
    rng = np.random.default_rng(47)
    x, u = R.rounded("single", rng.normal(size=(4, 300))), R.rounded("single", np.full(4, 0.97))
    nodes = R.Nodes(device, {"x": ("single", x.shape, x), "u": ("single", u.shape, u), "t": ("int32", u.shape, None)})
    for top_k in (2 ** 32 + 2, 2 ** 31, -2 ** 32 + 2, -2 ** 31 - 1):
        op = nodes.context.sample("x", "u", "t", top_k=top_k)
        op.run()
        device.await_()
        assert nodes.read("t").tolist() == [R.sample(x[r], u[r])[0] for r in range(4)]
        op.free()
    nodes.free()
