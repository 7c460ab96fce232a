"""Attention over a paged cache at the ends of its range: sequences of tens of millions of tokens and of 2^31, starts that fall, the widest windows."""
import numpy as np
import pytest

from tests import serving_reference as R
from tests.test_serving_gpu import attend_nodes, check_attend, link_attend, want_attend

pytestmark = pytest.mark.gpu


def repeated_page(q, k, v, length, prec, coded, scale):
    """(out, lse, bounds) of queries [h, d] that see `length` tokens, a page [page, d] again and again.  Bounds as in serving_reference.attention."""
    page = k.shape[0]
    times = length // page + (np.arange(page) < length % page)       # of every slot
    z = q @ k.T * scale
    top = np.where(times > 0, z, -np.inf).max(1, keepdims=True)
    w = np.where(times > 0, np.exp(z - top), 0.0) * times
    total = w.sum(1, keepdims=True)
    out, lse = w / total @ v, (top + np.log(total))[:, 0]
    half = R.EPS[prec] / 2
    of_weights = 0.0 if prec == "single" else 2.0 ** -11 if coded else half
    # (half weights below the normal range: 2^-25 of the largest, of all that a row sees)
    tiny = 2.0 ** -25 * (times @ np.abs(v) + 1) / total if prec == "half" or (coded and prec != "single") else 1e-30
    off = half * np.abs(out) + (of_weights + R.ARITH) * (w / total @ np.abs(v)) + tiny
    return out, lse, off, R.ARITH * (1 + np.abs(lse))


@pytest.mark.parametrize("lengths", [(17000011, 5000), (40000017, 3)])
@pytest.mark.parametrize("prec,coded,page,d,heads", [("bfloat16", True, 1024, 64, 2), ("bfloat16", False, 1024, 128, 16), ("half", False, 1000, 64, 3), ("half", True, 1 << 16, 128, 1),
                                                     ("single", False, 1000, 32, 2), ("single", True, 4096, 16, 9)])
def test_sequences_of_millions_of_tokens(device, prec, coded, page, d, heads, lengths):
    """More parts of a tile than are joined at once.  A table names one page throughout, so that the sums are known."""
    rng = np.random.default_rng(page + d)
    table = np.zeros((2, -(-max(lengths) // page) + 1), np.int64)
    x = {"q": R.rounded(prec, rng.standard_normal((2, heads, d)))}
    for g in "kv":
        a = rng.standard_normal((1, 1, page, d))
        if coded:
            x[g + "_scale"] = np.full((1, 1), 2.0 ** R.exponent(np.abs(a).max()))
            x[g + "_cache"] = R.encode(a / x[g + "_scale"][0, 0])
        else:
            x[g + "_cache"] = R.rounded(prec, a)
    kv = [R.decode(x[g + "_cache"][0, 0]) * x[g + "_scale"][0, 0] if coded else x[g + "_cache"][0, 0] for g in "kv"]
    nodes = attend_nodes(device, x, prec, table, np.array(lengths), None)
    op = link_attend(nodes, x, None, {})
    first = None
    for _ in range(2):
        op.run()
        device.await_()
        got, lse = nodes.read("out"), nodes.read("lse")
        for b, n in enumerate(lengths):
            want, want_lse, off, lse_off = repeated_page(x["q"][b], *kv, n, prec, coded, 1.0 / np.sqrt(d))
            R.within(got[b], want, off, "out")
            R.within(lse[b], want_lse, lse_off, "lse")
        first = nodes.raw("out") if first is None else first
        assert nodes.raw("out").tobytes() == first.tobytes()
    op.free()
    nodes.free()


@pytest.mark.parametrize("prec,coded,d", [("bfloat16", True, 128), ("half", True, 128), ("single", False, 64)])
def test_starts_that_fall_spoil_no_later_run(device, prec, coded, d):
    """What a run writes for them is not defined, but the runs behind it are as ever: no tile waits for parts of an earlier run.  (With three blocks on each of 148
    SMs, 444, the 32 tiles of 914432 tokens that falling starts make ask for 447, and the last of them begins in block 432; so does the last of eight
    tiles whose lengths are those below.)"""
    rng = np.random.default_rng(21)
    batch, n, page, width = 64, 8, 1024, 893
    x = {"q": R.rounded(prec, rng.standard_normal((n, 1, d)))}
    for g in "kv":
        a = rng.standard_normal((1, 1, page, d))
        if coded:
            x[g + "_scale"] = np.full((1, 1), 2.0 ** R.exponent(np.abs(a).max()))
            x[g + "_cache"] = R.encode(a / x[g + "_scale"][0, 0])
        else:
            x[g + "_cache"] = R.rounded(prec, a)
    kv = [R.decode(x[g + "_cache"][0, 0]) * x[g + "_scale"][0, 0] if coded else x[g + "_cache"][0, 0] for g in "kv"]
    most = page * width
    fine, falling = np.minimum(np.arange(batch + 1), n), np.where(np.arange(batch + 1) % 2, n, 0)
    lengths = np.full(batch, most)
    lengths[0], lengths[7] = most - 6400, 64 * 2300
    nodes = attend_nodes(device, x, prec, np.zeros((batch, width), np.int64), lengths, fine)
    op = link_attend(nodes, x, fine, {})
    for starts in (fine, falling, fine, fine):
        nodes.write("starts", starts)
        nodes.write("lengths", lengths if starts is fine else np.full(batch, most))
        nodes.write("out", np.full(x["q"].shape, np.nan))
        op.run()
        device.await_()
        if starts is fine:
            for b in range(n):
                out, lse, off, lse_off = repeated_page(x["q"][b], *kv, int(lengths[b]), prec, coded, 1.0 / np.sqrt(d))
                R.within(nodes.read("out")[b], out, off, "out")
                R.within(nodes.read("lse")[b], lse, lse_off, "lse")
    op.free()
    nodes.free()


def one_page(rng, prec, coded, page, d):
    """A cache of one page, and its values."""
    x, kv = {}, []
    for g in "kv":
        a = rng.standard_normal((1, 1, page, d))
        if coded:
            x[g + "_scale"] = np.full((1, 1), 2.0 ** R.exponent(np.abs(a).max()))
            x[g + "_cache"] = R.encode(a / x[g + "_scale"][0, 0])
        else:
            x[g + "_cache"] = R.rounded(prec, a)
        kv.append(R.decode(x[g + "_cache"][0, 0]) * x[g + "_scale"][0, 0] if coded else x[g + "_cache"][0, 0])
    return x, kv


@pytest.mark.parametrize("prec,coded,d", [("single", False, 1), ("half", True, 3), ("bfloat16", False, 8), ("half", True, 16)])
def test_as_many_tokens_as_there_are_positions(device, prec, coded, d):
    """2^31 - 1 tokens, and a few less, all of them seen."""
    rng = np.random.default_rng(d)
    page, lengths = 1 << 20, (2 ** 31 - 1, 2 ** 31 - 34)
    x, kv = one_page(rng, prec, coded, page, d)
    x["q"] = R.rounded(prec, rng.standard_normal((2, 2, d)))
    nodes = attend_nodes(device, x, prec, np.zeros((2, 2048), np.int64), np.array(lengths), None)
    op = link_attend(nodes, x, None, {})
    op.run()
    device.await_()
    for b, n in enumerate(lengths):
        out, lse, off, lse_off = repeated_page(x["q"][b], *kv, n, prec, coded, 1.0 / np.sqrt(d))
        R.within(nodes.read("out")[b], out, off, "out")
        R.within(nodes.read("lse")[b], lse, lse_off, "lse")
    op.free()
    nodes.free()


@pytest.mark.parametrize("prec,coded,new,heads,d", [("single", False, 5, 3, 20), ("half", True, 3, 4, 64), ("bfloat16", False, 300, 16, 64), ("bfloat16", True, 300, 32, 32)])
def test_windows_at_the_last_positions(device, prec, coded, new, heads, d):
    rng = np.random.default_rng(new)
    page, length, window = 4096, 2 ** 31 - 1, 500
    x, (k, v) = one_page(rng, prec, coded, page, d)
    x["q"] = R.rounded(prec, rng.standard_normal((new, heads, d)))
    nodes = attend_nodes(device, x, prec, np.zeros((1, 2 ** 31 // page), np.int64), np.array([length]), None)
    op = link_attend(nodes, x, None, dict(window=window))
    op.run()
    device.await_()
    got, lse = nodes.read("out"), nodes.read("lse")
    for r in range(new):
        pos = length - new + r
        at = np.arange(pos - window + 1, pos + 1) % page
        want, want_lse, off, lse_off = repeated_page(x["q"][r], k[at], v[at], window, prec, coded, 1.0 / np.sqrt(d))
        R.within(got[r], want, off, "out")
        R.within(lse[r], want_lse, lse_off, "lse")
    op.free()
    nodes.free()


@pytest.mark.parametrize("prec,coded", [("single", False), ("half", True), ("bfloat16", False)])
@pytest.mark.parametrize("window", [2 ** 31 - 2, 2 ** 31 - 1, 2 ** 62])
@pytest.mark.parametrize("case", [(1, 8, [3], 16, 1, 4, 64), (2, [300, 200], [200, 210], 64, 1, 16, 64)])
def test_the_widest_windows(device, case, window, prec, coded):
    """... beside rows that lie ahead of the first token, which see nothing."""
    from tests.test_serving_gpu import attend_case
    x, table, lengths, starts, page, t = attend_case(case + (0, 0, 0.0, False), prec, coded)
    t = dict(t, window=window)
    want = want_attend(x, table, lengths, starts, page, prec, t)
    nodes = attend_nodes(device, x, prec, table, lengths, starts)
    op = link_attend(nodes, x, starts, t)
    op.run()
    device.await_()
    check_attend(nodes, want)
    op.free()
    nodes.free()


@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("prec,page,d,pairs,layout", [("bfloat16", 256, 128, 64, "half"), ("single", 200, 256, 128, "half"), ("half", 700, 36, 13, "interleaved"),
                                                      ("bfloat16", 129, 128, 64, "interleaved"), ("single", 90, 512, 96, "interleaved")])
def test_pages_of_more_tokens_than_a_table(device, prec, page, d, pairs, layout, coded):
    """New tokens of a page whose cosines and sines are made in turns."""
    from tests.test_serving_gpu import append_case, append_nodes, check_append, link_append
    new = [page + 3, 1, 2 * page - 1, 128]
    x, table, lengths, starts, page, f, layout = append_case((4, new, [page + 3, 9, 2 * page + 40, 130], page, 3, 2, d, pairs, layout), prec, coded)
    want, off = R.append(x, prec, table, lengths, starts, page, f, layout)
    nodes = append_nodes(device, x, prec, table, lengths, starts)
    op = link_append(nodes, x, starts, f, layout)
    for _ in range(2):
        op.run()
        device.await_()
        check_append(nodes, want, off, coded)
    op.free()
    nodes.free()


@pytest.mark.parametrize("prec,coded,d,tokens,heads,length", [("bfloat16", False, 128, 130, 72, 17100), ("bfloat16", True, 128, 130, 72, 17100), ("half", False, 128, 130, 72, 17100),
                                                              ("half", True, 128, 130, 72, 17100), ("bfloat16", True, 72, 100, 96, 33100)])
def test_long_walks_of_tiles(device, prec, coded, d, tokens, heads, length):
    """More than 16384 tokens in tiles of 128 rows, heads of more than 64 elements: accumulators are added to sums beside them."""
    from tests.test_serving_gpu import attend_case
    x, table, lengths, starts, page, t = attend_case((1, tokens, [length], 64, 1, heads, d, 0, 0, 0.0, False), prec, coded)
    # (values of one sign add up: what an accumulator cuts off would show)
    x["v_cache"] = x["v_cache"] & 0x7f if coded else np.abs(x["v_cache"])
    x["q"] = R.rounded(prec, x["q"] * 0.05)
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


@pytest.mark.parametrize("prec,coded,page,d", [("bfloat16", True, 1024, 64), ("half", False, 1000, 40), ("single", False, 1024, 16)])
@pytest.mark.parametrize("there", [[0], [12000, 38000], [0, 1, 2, 20000, 38999, 39000], []])
def test_long_tables_of_few_pages(device, prec, coded, page, d, there):
    """Most parts of a tile see nothing, whole turns of their joining among them."""
    rng = np.random.default_rng(page + len(there))
    length, width = 39000 * page + 5, 39003
    x, kv = one_page(rng, prec, coded, page, d)
    x["q"] = R.rounded(prec, rng.standard_normal((1, 3, d)))
    table = np.full((1, width), -1)
    table[0, there] = 0
    seen = sum(5 if i == 39000 else page for i in there)
    nodes = attend_nodes(device, x, prec, table, np.array([length]), None)
    op = link_attend(nodes, x, None, {})
    op.run()
    device.await_()
    if not seen:
        assert np.all(nodes.read("out") == 0.0) and np.all(nodes.read("lse") == -np.inf)
    else:
        out, lse, off, lse_off = repeated_page(x["q"][0], *kv, seen, prec, coded, 1.0 / np.sqrt(d))
        R.within(nodes.read("out")[0], out, off, "out")
        R.within(nodes.read("lse")[0], lse, lse_off, "lse")
    op.free()
    nodes.free()
