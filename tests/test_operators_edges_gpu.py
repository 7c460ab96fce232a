"""The operators at values, sizes and arguments where a kernel could go wrong, against their definitions in 64 bits."""
import numpy as np
import pytest

from tests import operators_reference as R
from tests.test_operators_gpu import PRECS, attention_case, link_attention, out_bound

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
