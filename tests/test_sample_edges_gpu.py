"""Choices of a token over long rows where the border is hard to find: zeros of both signs as the largest logits, many equal logits, borders far down."""
import numpy as np
import pytest

from tests import serving_reference as R
from tests.test_serving_gpu import PRECS, check_sample, run_sample

pytestmark = pytest.mark.gpu


def repeated(rows, *arrays):
    """The same few rows again and again, up to `rows` of them: their number decides how many blocks a row has."""
    return [np.resize(a, (rows,) + a.shape[1:]) for a in arrays]


def check_repeated(got, few, rows, x, u, given):
    """The first `few` rows against the restatement, all others bit for bit against those."""
    check_sample([a[:few] for a in got], x[:few], u[:few], {n: v[:few] if np.ndim(v) else v for n, v in given.items()})
    for a in got:
        assert a.tobytes() == np.resize(a[:few], a.shape).tobytes()


# (vocab, rows): one to eight blocks a row
ZEROS = [(1500, 5), (5000, 5), (5000, 600), (20011, 150), (20011, 300), (20011, 600), (131072, 5)]


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("vocab,rows", ZEROS)
def test_zeros_are_the_largest(device, vocab, rows, prec):
    """Rows of -0 alone, of both zeros, of negated costs with thousands of zeros, and a -0 above all others."""
    rng = np.random.default_rng(vocab + rows)
    x = np.empty((5, vocab))
    x[0] = -0.0
    x[1] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    x[2] = -np.maximum(rng.standard_normal(vocab), 0.0)
    x[3] = -np.abs(rng.standard_normal(vocab))
    x[3, vocab // 3] = -0.0
    x[4] = np.where(rng.random(vocab) < 0.6, -0.0, -5.0)
    x, u = R.rounded(prec, x), R.rounded("single", rng.random(5))
    assert np.signbit(x[0]).all() and np.signbit(x[2][x[2] == 0]).all()
    x, u = repeated(rows, x, u)
    for given in (dict(top_k=50), dict(top_p=0.9), dict(top_k=1100, top_p=0.5, temperature=5.0), dict(min_p=0.5, temperature=0.5), dict(temperature=0.0)):
        given = {n: float(np.float32(v)) if n != "top_k" else v for n, v in given.items()}
        check_repeated(run_sample(device, prec, x, u, given), 5, rows, x, u, given)


@pytest.mark.parametrize("vocab,rows,prec", [(131072, 3, "single"), (131072, 600, "bfloat16"), (1 << 24, 1, "single"), (3 << 22, 1, "half")])
def test_one_logit_again_and_again_below_a_larger_one(device, vocab, rows, prec):
    """The kept count is known: n is the least with 1 + (n - 1) w >= p (1 + (vocab - 1) w).  A random number of 1 takes the last kept one, which is
    token n - 1, as equal logits are kept in the order of their indices."""
    x = np.full((1, vocab), -0.37)
    x[0, 0] = 0.0
    x = R.rounded(prec, x)
    w = np.exp(x[0, 1])
    x, u = repeated(rows, x, np.ones(1))
    for p in (0.3, 0.61, 0.9, 0.97):
        p = float(np.float32(p))
        need = (p * (1.0 + (vocab - 1) * w) - 1.0) / w
        # (weights in steps of 2^-44 move the sums by vocab * 2^-45 at most, `need` by less than 2^24 * 2^-45 / w < 10^-6; sums in 64 bits by less still)
        assert 0.001 < need % 1.0 < 0.999
        tokens, _ = run_sample(device, prec, x, u, dict(top_p=p))
        assert np.all(tokens == int(np.ceil(need))), (p, need, tokens[:4])


def test_the_same_bits_every_time(device):
    """Rows whose border is looked for in the blocks' lists, whose places are handed out in no order."""
    rng = np.random.default_rng(77)
    x, u = R.rounded("single", rng.standard_normal((40, 60000)) * 1.5), R.rounded("single", rng.random(40))
    for given in (dict(top_p=float(np.float32(0.8))), dict(top_k=5000, top_p=0.5)):
        first = run_sample(device, "single", x, u, given)
        for _ in range(10):
            again = run_sample(device, "single", x, u, given)
            assert all(a.tobytes() == b.tobytes() for a, b in zip(first, again))


@pytest.mark.parametrize("prec", PRECS)
def test_borders_lie_where_64_bits_have_them(device, prec):
    """Rows in falling order and a random number of 1: the token is the last kept one, the border itself."""
    rng = np.random.default_rng(91)
    rows, vocab = 24, 131072
    x = -np.sort(-rng.standard_normal((rows, vocab)) * np.linspace(0.3, 4.0, rows)[:, None], 1)
    x, u = R.rounded(prec, x), np.ones(rows)
    single = {"temperature": rng.uniform(0.6, 1.5, rows), "top_p": rng.uniform(0.2, 0.995, rows), "min_p": 10.0 ** rng.uniform(-4, -1, rows)}
    single = {n: R.rounded("single", v) for n, v in single.items()}
    for given in (dict(single, min_p=0.0), dict(single, top_p=1.0), dict(single, top_k=rng.integers(10000, 100000, rows), min_p=0.0)):
        check_sample(run_sample(device, prec, x, u, given), x, u, given)


@pytest.mark.parametrize("prec", PRECS)
def test_tokens_of_flat_rows(device, prec):
    """A hundred thousand tokens of nearly equal weights: running sums that are off by a few millionths would choose others."""
    rng = np.random.default_rng(92)
    rows, vocab = 120, 100003
    x = np.repeat(R.rounded(prec, rng.standard_normal((1, vocab)) * 2.0), rows, 0)
    u = R.rounded("single", rng.random(rows))
    for given in (dict(temperature=float(np.float32(3.3))), dict(top_p=float(np.float32(0.93)))):
        check_sample(run_sample(device, prec, x, u, given), x, u, given)


def test_differences_and_temperatures_at_the_ends(device):
    """Logits whose difference single precision cannot hold, temperatures from the least number to infinity."""
    x = np.tile(R.rounded("single", np.array([3e38, -3e38, 1e38, 0.0, -1e38, 2.9e38, 2e38])), (8, 1))
    x[4:] = R.rounded("single", np.array([0.0, -1e-38, -3e-39, 1e-45, -1.0, -0.0, -2e-38]))
    t = R.rounded("single", np.array([1e38, 3e38, 2e37, 1e30, 1e-45, 1e-38, 3e-39, 1.0]))
    for u in (0.0, 0.3, 0.6, 0.9, 1.0):
        u = R.rounded("single", np.full(8, u))
        for given in (dict(temperature=t), dict(temperature=t, top_p=float(np.float32(0.7))), dict(temperature=t, top_k=3), dict(temperature=t, min_p=float(np.float32(0.05)))):
            check_sample(run_sample(device, "single", x, u, given), x, u, given)
    x = np.tile(x[:4], (1, 400))                      # rows of several blocks' passes
    u, t = R.rounded("single", np.array([0.1, 0.4, 0.7, 1.0])), t[:4]
    for given in (dict(temperature=t, top_p=float(np.float32(0.7))), dict(temperature=t, top_k=1500), dict(temperature=np.full(4, np.inf))):
        check_sample(run_sample(device, "single", x, u, given), x, u, given)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("vocab", [1022, 1500, 9001])
def test_infinite_and_undefined_logits_of_long_rows(device, vocab, prec):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((7, vocab)) * 3.0
    x[0, [3, vocab // 2, vocab - 1]] = np.inf
    x[1, rng.random(vocab) < 0.9] = np.inf
    x[2] = np.where(rng.random(vocab) < 0.5, np.nan, -np.inf)
    x[3] = np.where(rng.random(vocab) < 0.9, np.nan, x[3])
    x[4] = np.where(rng.random(vocab) < 0.9, -np.inf, x[4])
    x[5] = np.where(rng.random(vocab) < 0.3, -np.nan, x[5])
    x[6, ::2] = -np.inf
    x, u = R.rounded(prec, x), R.rounded("single", rng.random(7))
    for given in ({}, dict(top_k=2), dict(top_k=1100, top_p=0.5), dict(top_p=0.75), dict(min_p=0.5), dict(temperature=0.0), dict(top_p=0.0, min_p=2.0), dict(temperature=1e-3, top_p=0.5)):
        given = {n: float(np.float32(v)) if n != "top_k" else v for n, v in given.items()}
        check_sample(run_sample(device, prec, x, u, given), x, u, given)


@pytest.mark.parametrize("vocab", [9, 700, 3000, 40000])
def test_masked_logits_beside_the_least_temperatures(device, vocab):
    """Finite masks (-10^9, the lowest value) where differences are multiplied: their weight is 0, as that of all but the largest few."""
    rng = np.random.default_rng(vocab)
    x = np.zeros((6, vocab))
    x[:, ::2] = -1e9
    x[:, ::7] = -3.4e38
    x[:, 1::2] = -np.abs(rng.standard_normal((6, len(x[0, 1::2])))) * np.array([1e-31, 1e-36, 1e-30, 0.5, 1e-29, 1e-40])[:, None]
    x[3, 1] = 1.0
    x, u = R.rounded("single", x), R.rounded("single", rng.random(6))
    t = R.rounded("single", np.array([1e-31, 1e-36, 9e-31, 1e-33, 1e-20, 1e-40]))
    for given in (dict(temperature=t), dict(temperature=t, top_k=3), dict(temperature=t, top_p=float(np.float32(0.6))), dict(temperature=t, top_p=float(np.float32(0.999)), min_p=float(np.float32(0.01)))):
        check_sample(run_sample(device, "single", x, u, given), x, u, given)
