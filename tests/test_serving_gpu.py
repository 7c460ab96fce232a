"""Appending to a paged cache, attention over it and the choice of tokens on the device, against restatements in 64 bits (serving_reference)."""
import numpy as np
import pytest

from ocannl_b200 import backend as bk
from tests import serving_reference as R

pytestmark = pytest.mark.gpu
PRECS = ("bfloat16", "half", "single")


def pool(rng, batch, page, max_pages, spare=2):
    """A table of pages handed out in no order; how many there are."""
    pages = batch * max_pages + spare
    return rng.permutation(pages)[:batch * max_pages].reshape(batch, max_pages).astype(np.int32), pages


# (batch, new tokens of each sequence or one number for all, lengths, page, kv_heads, heads, d, pairs, layout)
APPEND = [
    (3, 1, [1, 17, 32], 16, 2, 4, 64, 32, "half"),
    (2, [5, 0], [5, 9], 8, 1, 1, 16, 4, "interleaved"),
    (4, [3, 40, 1, 0], [3, 75, 64, 10], 32, 3, 6, 80, 40, "half"),
    (1, 130, [200], 64, 2, 2, 128, 64, "interleaved"),
    (2, [70, 33], [70, 99], 7, 5, 5, 24, 6, "half"),
    (3, [9, 2, 30], [4, 2, 100], 16, 2, 0, 33, 5, "half"),
    (2, 2, [2, 40], 1, 9, 9, 32, 16, "half"),
    (2, 300, [300, 431], 128, 1, 2, 128, 0, "half"),
    (1, 37, [37], 40, 1, 1, 40, 20, "interleaved"),
]


def append_case(case, prec, coded, seed=3, extra=3):
    batch, new, lengths, page, hk, h, d, m, layout = case
    rng = np.random.default_rng(seed)
    counts = [new] * batch if isinstance(new, int) else new
    starts = None if isinstance(new, int) else np.concatenate([[0], np.cumsum(counts)])
    n = sum(counts) + (extra if starts is not None else 0)
    max_pages = -(-max(lengths) // page) + 1
    table, pages = pool(rng, batch, page, max_pages)
    x = {"k": rng.standard_normal((n, hk, d)) * np.exp(rng.standard_normal((n, 1, 1))), "v": rng.standard_normal((n, hk, d)) * 3.0}
    if h:
        x["q"] = rng.standard_normal((n, h, d))
    x = {g: R.rounded(prec, a) for g, a in x.items()}
    for g in "kv":
        if coded:
            x[g + "_cache"] = rng.integers(0, 256, (pages, hk, page, d)).astype(np.uint8)
            x[g + "_scale"] = 2.0 ** rng.integers(-9, -4, (pages, hk))
        else:
            x[g + "_cache"] = R.rounded(prec, rng.standard_normal((pages, hk, page, d)))
    f = 10000.0 ** (-np.arange(m) / max(m, 1))
    return x, table, np.array(lengths), starts, page, f, layout


def append_nodes(device, x, prec, table, lengths, starts, packing="aligned", **more):
    coded = "k_scale" in x
    arrays = {g: ("byte" if coded and g.endswith("cache") else "single" if g.endswith("scale") else prec, a.shape, a) for g, a in x.items()}
    arrays.update(pages=("int32", table.shape, table), lengths=("int32", lengths.shape, lengths))
    if starts is not None:
        arrays["starts"] = ("int32", starts.shape, starts)
    if "q" in x:
        arrays["q_out"] = (prec, x["q"].shape, None)
    arrays.update(more)
    return R.Nodes(device, arrays, packing)


def link_append(nodes, x, starts, f, layout, magnitude=1.0, positions=None):
    scales = dict(k_scale="k_scale", v_scale="v_scale") if "k_scale" in x else {}
    q = dict(q="q", q_out="q_out") if "q" in x else {}
    return nodes.context.cache_append("k", "v", "k_cache", "v_cache", "pages", "lengths", starts=None if starts is None else "starts", frequencies=f, layout=layout,
                                      magnitude=magnitude, positions=positions, **scales, **q)


def check_append(nodes, want, off, coded):
    for g, v in want.items():
        if g.endswith("cache") and coded:
            scale = want[g[0] + "_scale"][:, :, None, None]
            raw = nodes.raw(g)
            untouched = off[g] == 0
            assert np.array_equal(raw[untouched & ~np.isnan(R.decode(v))], v[untouched & ~np.isnan(R.decode(v))]), g
            # (twice the bound: the wanted codes are rounded too)
            R.within(R.decode(raw) * scale, R.decode(v) * scale, 2 * off[g], g)
        elif g.endswith("scale"):
            assert np.array_equal(nodes.read(g), v), g
        else:
            R.within(nodes.read(g), v, off[g], g)


@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("case", APPEND)
def test_append(device, case, prec, coded):
    x, table, lengths, starts, page, f, layout = append_case(case, prec, coded)
    want, off = R.append(x, prec, table, lengths, starts, page, f, layout, magnitude=1.5)
    for packing in ("aligned", "tight"):
        nodes = append_nodes(device, x, prec, table, lengths, starts, packing)
        op = link_append(nodes, x, starts, f, layout, magnitude=1.5)
        op.run()
        device.await_()
        check_append(nodes, want, off, coded)
        # again: nothing grows any more, the same tokens to the same slots
        first = {g: nodes.raw(g) for g in want}
        op.run()
        device.await_()
        for g in want:
            assert nodes.raw(g).tobytes() == first[g].tobytes(), g
        op.free()
        nodes.free()


@pytest.mark.parametrize("coded", [False, True])
def test_append_where_no_page_is(device, coded):
    """Numbers that are no pages, positions before the first and behind the last page, lengths below zero: nothing is written there."""
    case = (5, [4, 6, 3, 2, 5], [2, 40, 21, -3, 5], 8, 2, 2, 32, 16, "half")
    x, table, lengths, starts, page, f, layout = append_case(case, "bfloat16", coded)
    table = table[:, :4].copy()          # 32 tokens at most
    table[2, 2] = -1
    table[4, 0] = 1 << 30
    want, off = R.append(x, "bfloat16", table, lengths, starts, page, f, layout)
    nodes = append_nodes(device, x, "bfloat16", table, lengths, starts)
    op = link_append(nodes, x, starts, f, layout)
    op.run()
    device.await_()
    check_append(nodes, want, off, coded)
    op.free()
    nodes.free()


@pytest.mark.parametrize("prec", PRECS)
def test_scales_that_grow(device, prec):
    """Token by token, each up to 2^12 times the one before or 2^-12: codes are rounded again where the scale grows, and stay where it does not."""
    rng = np.random.default_rng(5)
    page, hk, d, steps = 16, 2, 16, 20
    sizes = 2.0 ** rng.integers(-6, 7, steps) if prec == "half" else 2.0 ** rng.integers(-12, 13, steps)
    table = np.array([[1, 0]], np.int32)
    held = {g: np.full((2, hk, page, d), 0x55, np.uint8) for g in ("k_cache", "v_cache")}
    scales = {g: np.full((2, hk), np.nan) for g in ("k_scale", "v_scale")}
    nodes = R.Nodes(device, dict(k=(prec, (1, hk, d), None), v=(prec, (1, hk, d), None), pages=("int32", (1, 2), table), lengths=("int32", (1,), None),
                                 **{g: ("byte", a.shape, a) for g, a in held.items()}, **{g: ("single", a.shape, a) for g, a in scales.items()}))
    op = nodes.context.cache_append("k", "v", "k_cache", "v_cache", "pages", "lengths", k_scale="k_scale", v_scale="v_scale")
    for i, s in enumerate(sizes):
        new = {g: R.rounded(prec, rng.standard_normal((1, hk, d)) * s) for g in "kv"}
        for g in "kv":
            nodes.write(g, new[g])
        nodes.write("lengths", [i + 1])
        op.run()
        device.await_()
        want, _ = R.append({**new, **held, **scales}, prec, table, [i + 1], None, page)
        for g in ("k", "v"):
            # (no turn: the values and so the codes are exact)
            assert np.array_equal(nodes.read(g + "_scale")[table[0, :i // page + 1]], want[g + "_scale"][table[0, :i // page + 1]])
            assert np.array_equal(nodes.raw(g + "_cache"), want[g + "_cache"]), (g, i)
        held, scales = {g: want[g] for g in held}, {g: want[g] for g in scales}
    op.free()
    nodes.free()


def test_values_that_have_no_code(device):
    """Undefined and infinite values become undefined codes and count in no scale; those beyond 448 * 2^40 too; zeros have the least scale."""
    d, page = 16, 4
    k = np.zeros((4, 1, d))
    k[0, 0, :4] = [np.nan, np.inf, -np.inf, 3.0]
    k[1, 0, :2] = [448.0 * 2.0 ** 41, 448.0]
    k[2, 0, 0] = 2.0 ** -60
    v = np.zeros((4, 1, d))
    x = dict(k=R.rounded("bfloat16", k), v=v, k_cache=np.full((1, 1, page, d), 3, np.uint8), v_cache=np.full((1, 1, page, d), 3, np.uint8),
             k_scale=np.ones((1, 1)), v_scale=np.ones((1, 1)))
    table, lengths = np.zeros((1, 1), np.int32), np.array([4])
    nodes = append_nodes(device, x, "bfloat16", table, lengths, None)
    op = link_append(nodes, x, None, (), "half")
    op.run()
    device.await_()
    want, _ = R.append(x, "bfloat16", table, lengths, None, page)
    got = nodes.raw("k_cache")
    assert np.array_equal(np.isnan(R.decode(got)), np.isnan(R.decode(want["k_cache"])))
    fine = ~np.isnan(R.decode(got))
    assert np.array_equal(R.decode(got)[fine], R.decode(want["k_cache"])[fine])
    assert nodes.read("k_scale")[0, 0] == 1.0 and nodes.read("v_scale")[0, 0] == 2.0 ** -40
    op.free()
    nodes.free()


def test_far_and_other_positions(device):
    """Keys turn by positions of their own, up to 2^31 - 1, while their slots go by the sequence's."""
    case = (2, 3, [3, 9], 4, 2, 4, 32, 16, "half")
    x, table, lengths, starts, page, f, layout = append_case(case, "single", False)
    positions = np.array([0, 2 ** 31 - 1, 123456789, -5, 1000003, 7], np.int64)
    want, off = R.append(x, "single", table, lengths, starts, page, f, layout, positions=positions)
    nodes = append_nodes(device, x, "single", table, lengths, starts, positions=("int32", (6,), positions))
    op = link_append(nodes, x, starts, f, layout, positions="positions")
    op.run()
    device.await_()
    check_append(nodes, want, off, False)
    op.free()
    nodes.free()


def test_queries_turn_in_place(device):
    case = (2, [4, 3], [10, 3], 8, 2, 4, 64, 32, "interleaved")
    x, table, lengths, starts, page, f, layout = append_case(case, "bfloat16", True)
    want, off = R.append(x, "bfloat16", table, lengths, starts, page, f, layout)
    nodes = append_nodes(device, x, "bfloat16", table, lengths, starts)
    op = nodes.context.cache_append("k", "v", "k_cache", "v_cache", "pages", "lengths", starts="starts", frequencies=f, layout=layout, k_scale="k_scale",
                                    v_scale="v_scale", q="q", q_out="q")
    op.run()
    device.await_()
    rows = slice(0, starts[-1])
    R.within(nodes.read("q")[rows], want["q_out"][rows], off["q_out"][rows], "q")
    assert np.array_equal(nodes.read("q")[starts[-1]:], x["q"][starts[-1]:])
    op.free()
    nodes.free()


# ------------------------------------------------------------------ attention
# (batch, new tokens, lengths, page, kv_heads, heads, d, window, sinks, cap, slopes)
ATTEND = [
    (3, 1, [1, 17, 32], 16, 2, 4, 64, 0, 0, 0.0, False),
    (2, 1, [700, 1], 32, 1, 1, 128, 0, 0, 0.0, False),
    (4, 1, [300, 0, -4, 90], 8, 2, 16, 64, 40, 4, 30.0, True),
    (2, [5, 3], [5, 90], 7, 3, 6, 40, 20, 3, 0.0, True),
    (3, [3, 0, 50], [2, 9, 80], 16, 1, 3, 24, 0, 0, 0.0, False),
    (2, [1, 33], [513, 129], 64, 2, 8, 128, 0, 0, 20.0, False),
    (1, 140, [300], 64, 1, 2, 128, 100, 16, 0.0, False),
    (2, 150, [150, 260], 8, 2, 2, 64, 0, 0, 0.0, True),
    (1, 20, [50], 1, 1, 1, 33, 7, 2, 5.0, False),
    (2, 2, [40, 260], 20, 1, 32, 80, 0, 0, 0.0, False),
    (1, 1, [100], 128, 1, 4, 1, 0, 0, 0.0, False),
    (1, 3, [2000], 16, 1, 20, 96, 64, 100, 0.0, False),
]


def attend_case(case, prec, coded, seed=11, stale=np.nan, extra=2):
    batch, new, lengths, page, hk, h, d, window, sinks, cap, slopes = case
    rng = np.random.default_rng(seed)
    counts = [new] * batch if isinstance(new, int) else new
    starts = None if isinstance(new, int) else np.concatenate([[0], np.cumsum(counts)])
    n = sum(counts) + (extra if starts is not None else 0)
    max_pages = -(-max(lengths) // page) + 1
    table, pages = pool(rng, batch, page, max_pages)
    held = np.zeros((pages, page), bool)
    for b in range(batch):
        for j in range(max(lengths[b], 0)):
            held[table[b, j // page], j % page] = True
    x = {"q": R.rounded(prec, rng.standard_normal((n, h, d)) * (2.0 if cap else 1.0))}
    for g in "kv":
        a = rng.standard_normal((pages, hk, page, d)) * np.exp(rng.standard_normal((pages, hk, 1, 1)))
        if coded:
            x[g + "_scale"] = 2.0 ** np.array([[R.exponent(np.abs(s).max()) for s in p] for p in a])
            x[g + "_cache"] = np.where(held[:, None, :, None], R.encode(a / x[g + "_scale"][:, :, None, None]), 0x7f if np.isnan(stale) else 0x7e)
        else:
            x[g + "_cache"] = R.rounded(prec, np.where(held[:, None, :, None], a, stale))
    t = dict(window=window, sinks=sinks, cap=cap)
    if slopes:
        x["slopes"] = 2.0 ** (-8.0 * np.arange(1, h + 1) / h)
    # pages that nobody sees any more are given back
    if window:
        for b in range(batch):
            first = lengths[b] - counts[b] - window + 1
            for i in range(max_pages):
                if (i + 1) * page <= first and i * page >= sinks:
                    table[b, i] = [-1, pages, 1 << 30][i % 3]
    return x, table, np.array(lengths), starts, page, t


def attend_nodes(device, x, prec, table, lengths, starts, packing="aligned", coded=None):
    coded = "k_scale" in x
    arrays = {g: ("byte" if coded and g.endswith("cache") else "single" if g.endswith("scale") or g == "slopes" else prec, a.shape, a) for g, a in x.items()}
    arrays.update(pages=("int32", table.shape, table), lengths=("int32", lengths.shape, lengths), out=(prec, x["q"].shape, None), lse=("single", x["q"].shape[:2], None))
    if starts is not None:
        arrays["starts"] = ("int32", starts.shape, starts)
    return R.Nodes(device, arrays, packing)


def link_attend(nodes, x, starts, t, lse="lse"):
    scales = dict(k_scale="k_scale", v_scale="v_scale") if "k_scale" in x else {}
    return nodes.context.cache_attention("q", "k_cache", "v_cache", "out", "pages", "lengths", starts=None if starts is None else "starts", lse=lse,
                                         slopes="slopes" if "slopes" in x else None, **scales, **t)


def want_attend(x, table, lengths, starts, page, prec, t):
    return R.attention(x["q"], x["k_cache"], x["v_cache"], table, lengths, starts, page, prec, x.get("k_scale"), x.get("v_scale"), slopes=x.get("slopes"), **t)


def check_attend(nodes, want):
    out, lse, off, lse_off = want
    R.within(nodes.read("out"), out, off, "out")
    R.within(nodes.read("lse"), lse, lse_off, "lse")


@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("case", ATTEND)
def test_attention_over_pages(device, case, prec, coded):
    """Slots that hold nothing, and pages given back, are undefined; rows of no sequence stay as they were."""
    x, table, lengths, starts, page, t = attend_case(case, prec, coded)
    want = want_attend(x, table, lengths, starts, page, prec, t)
    for packing in ("aligned", "tight"):
        nodes = attend_nodes(device, x, prec, table, lengths, starts, packing)
        op = link_attend(nodes, x, starts, t, lse="lse")
        op.run()
        device.await_()
        check_attend(nodes, want)
        first = nodes.raw("out")
        op.run()
        device.await_()
        assert nodes.raw("out").tobytes() == first.tobytes()
        op.free()
        nodes.free()


# prompts, in tiles of 16 rows
PROMPTS = [
    (1, 128, [128], 64, 2, 2, 128, 0, 0, 0.0, False),
    (2, [100, 300], [700, 300], 16, 2, 8, 128, 0, 0, 0.0, False),
    (3, [64, 0, 200], [64, 9, 1000], 32, 1, 5, 96, 150, 20, 0.0, True),
    (2, [90, 33], [513, 129], 64, 2, 6, 64, 0, 0, 20.0, False),
    (1, 260, [1000], 128, 1, 20, 80, 200, 70, 0.0, False),
    (2, [200, 70], [190, 300], 64, 1, 4, 48, 0, 0, 5.0, True),
    (5, 40, [40, 100, 300, 77, 64], 16, 4, 16, 64, 33, 2, 0.0, False),
    (1, 1, [50], 16, 1, 128, 64, 0, 0, 0.0, False),
    (2, [1300, 1100], [1300, 1900], 32, 2, 16, 64, 0, 0, 0.0, False),
    (3, [700, 800, 900], [700, 2000, 900], 64, 2, 16, 128, 300, 5, 30.0, False),
    (1, 130, [17000], 64, 1, 2, 64, 0, 0, 0.0, False),
    (1, 70, [34000], 16, 1, 2, 128, 0, 0, 0.0, False),
]
# key heads, and rows of them, enough for tiles of 128
TILES = [
    (1, 128, [128], 64, 72, 72, 64, 0, 0, 0.0, False),
    (2, [100, 300], [700, 300], 16, 12, 24, 128, 0, 0, 0.0, False),
    (3, [64, 0, 200], [64, 9, 1000], 32, 8, 40, 96, 150, 20, 0.0, True),
    (2, [90, 33], [513, 129], 64, 26, 78, 64, 0, 0, 20.0, False),
    (1, 260, [1000], 128, 2, 40, 80, 200, 70, 0.0, False),
    (2, [200, 70], [190, 300], 64, 9, 36, 48, 0, 0, 5.0, True),
    (5, 40, [40, 100, 300, 77, 64], 16, 12, 48, 64, 33, 2, 0.0, False),
    (1, 1, [50], 16, 72, 9216, 64, 0, 0, 0.0, False),
    (1, 140, [34000], 16, 34, 68, 16, 0, 0, 0.0, False),
    (2, [700, 900], [60, 900], 64, 4, 16, 112, 0, 0, 0.0, False),
]


@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("prec", ["bfloat16", "half"])
@pytest.mark.parametrize("case", PROMPTS + TILES)
def test_prompts_over_pages(device, case, prec, coded):
    x, table, lengths, starts, page, t = attend_case(case, prec, coded)
    want = want_attend(x, table, lengths, starts, page, prec, t)
    nodes = attend_nodes(device, x, prec, table, lengths, starts)
    op = link_attend(nodes, x, starts, t)
    op.run()
    device.await_()
    check_attend(nodes, want)
    first = nodes.raw("out")
    op.run()
    device.await_()
    assert nodes.raw("out").tobytes() == first.tobytes()
    op.free()
    nodes.free()


# ------------------------------------------------------------------ choosing a token
SAMPLE = [   # (rows, vocab, what the rows hold)
    (3, 1, "logits"), (7, 27, "logits"), (33, 27, "ties"), (5, 1000, "logits"), (4, 1023, "hidden"), (3, 5000, "ties"), (4, 4097, "flat"),
    (3, 33333, "logits"), (2, 70001, "hidden"), (2, 131072, "flat"), (2, 40000, "ties"), (1, 300007, "logits"), (1, 1 << 20, "flat"),
]


def logits(rng, prec, rows, vocab, what):
    x = rng.standard_normal((rows, vocab)) * np.exp(rng.standard_normal((rows, 1)) * 0.5 + 1.0)
    if what == "ties":
        x = np.round(x)
    if what == "flat":
        x = rng.standard_normal((rows, vocab)) * 0.01
    if what == "hidden":
        x = np.where(rng.random((rows, vocab)) < 0.7, -np.inf, x)
        x[:, ::5] = np.nan
        x[:, 1] = 0.0
        x[:, 2 % vocab] = -0.0
    return R.rounded(prec, x)


def settings(rng, rows):
    return dict(temperature=R.rounded("single", rng.choice([0.0, 0.7, 1.0, 1.3, 5.0], rows, p=[0.1, 0.3, 0.3, 0.2, 0.1])), top_k=rng.choice([0, 1, 2, 50, 1000, 30000], rows),
                top_p=R.rounded("single", rng.choice([1.0, 0.99, 0.9, 0.5, 0.0], rows)), min_p=R.rounded("single", rng.choice([0.0, 0.001, 0.1, 1.0, 2.0], rows)))


def run_sample(device, prec, x, u, given, packing="aligned"):
    """given: {setting: a number or one a row}."""
    rows = x.shape[0]
    arrays = dict(logits=(prec, x.shape, x), u=("single", (rows,), u), tokens=("int32", (rows,), None), logprob=("single", (rows,), None))
    for n, v in given.items():
        if np.ndim(v):
            arrays[n] = ("int32" if n == "top_k" else "single", (rows,), v)
    nodes = R.Nodes(device, arrays, packing)
    op = nodes.context.sample("logits", "u", "tokens", logprob="logprob", **{n: n if np.ndim(v) else v for n, v in given.items()})
    op.run()
    op.run()
    device.await_()
    got = nodes.read("tokens"), nodes.read("logprob")
    op.free()
    nodes.free()
    return got


def check_sample(got, x, u, given):
    tokens, logprob = got
    for r in range(x.shape[0]):
        token, lp = R.sample(x[r], u[r], **{n: v[r] if np.ndim(v) else v for n, v in given.items()})
        assert tokens[r] == token, (r, tokens[r], token)
        # weights are off by some 2^-22 (the exponent's size times 2^-24, and the exponential), the kept sum by as much; lp in single precision
        assert lp == logprob[r] or abs(lp - logprob[r]) <= 2.0 ** -18 + 2.0 ** -23 * abs(lp), (r, logprob[r], lp)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("case", SAMPLE)
def test_sample(device, case, prec):
    rows, vocab, what = case
    rng = np.random.default_rng(rows * vocab)
    x, u = logits(rng, prec, rows, vocab, what), R.rounded("single", rng.random(rows))
    for packing in ("aligned", "tight"):
        for _ in range(3):
            given = settings(rng, rows)
            check_sample(run_sample(device, prec, x, u, given, packing), x, u, given)
        check_sample(run_sample(device, prec, x, u, {}, packing), x, u, {})


@pytest.mark.parametrize("given", [dict(), dict(temperature=0.0), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.3), dict(top_k=40, top_p=0.9, min_p=0.01, temperature=1.7)])
def test_settings_as_numbers(device, given):
    rng = np.random.default_rng(8)
    x, u = logits(rng, "half", 40, 301, "logits"), R.rounded("single", rng.random(40))
    given = {n: float(np.float32(v)) if n != "top_k" else v for n, v in given.items()}
    check_sample(run_sample(device, "half", x, u, given), x, u, given)


def test_settings_that_are_undefined(device):
    """In a node: a temperature is 0 then, top_p 1, min_p 0; negative ones count as none."""
    rng = np.random.default_rng(12)
    x, u = logits(rng, "single", 8, 1500, "logits"), R.rounded("single", rng.random(8))
    nan, ones = np.full(8, np.nan), np.ones(8)
    for given, same in ((dict(temperature=nan), dict(temperature=0.0)), (dict(top_p=nan), {}), (dict(min_p=nan), {}), (dict(top_p=-ones, min_p=-ones, top_k=-ones), dict(top_p=0.0)),
                        (dict(temperature=-ones), dict(temperature=0.0)), (dict(top_k=2e9 * ones), {})):
        check_sample(run_sample(device, "single", x, u, given), x, u, same)


def test_random_numbers_at_the_ends(device):
    """0, just below 1, and those outside: the first and the last kept token."""
    rng = np.random.default_rng(9)
    x = logits(rng, "single", 6, 500, "logits")
    u = np.array([0.0, 1.0 - 2.0 ** -24, 1.0, -3.0, np.nan, np.inf])
    for given in (dict(), dict(top_k=20)):
        check_sample(run_sample(device, "single", x, u, given), x, u, given)


def test_rows_of_nothing_and_of_infinities(device):
    x = np.full((5, 70), -np.inf)
    x[1] = np.nan
    x[2, [7, 30, 69]] = np.inf
    x[2, 4] = 3.0
    x[3, 12] = -3e38
    x[4] = 0.0
    u = np.array([0.5, 0.5, 0.5, 0.9, 0.5])
    for given in (dict(), dict(top_k=2, top_p=0.9), dict(top_p=0.3), dict(temperature=0.0)):
        check_sample(run_sample(device, "single", x, u, given), x, u, given)


def test_the_shares_are_those_of_the_weights(device):
    """Many random numbers over one row: every kept token comes up as often as its weight says."""
    rng = np.random.default_rng(10)
    n = 4096
    x = np.repeat(logits(rng, "single", 1, 12, "logits"), n, 0)
    u = R.rounded("single", (np.arange(n) + 0.5) / n)
    tokens, _ = run_sample(device, "single", x, u, dict(top_k=7))
    order = np.argsort(-x[0])[:7]
    w = np.zeros(12)
    w[order] = np.exp(x[0, order] - x[0].max())
    # evenly spaced numbers: within one of the share at either end of a token's range
    assert np.all(np.abs(np.bincount(tokens, minlength=12) - n * w / w.sum()) <= 2)
