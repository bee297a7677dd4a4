"""How far log probabilities and entropies are off, to the bound of their roundings.

m, l and t are a row's maximum, sum of e^d and sum of e^d d with d = x - m; p = e^d / l. A thread adds f32 exponentials of the
distance to its maximum so far; where that moves, and in the joins, its sums are multiplied by the exponential of the move.
- A logit's distances add up to |d| over all of these, and each has three roundings of half a step (of the difference, the
  constant and the product): 3 |d| 2^-24.
- Each exponential is off by a step of its result: 2^-23. There is the logit's own and one for each move: at most `rounds`, one
  for each 16 logits that a thread takes, and 4 in joins (lanes and waves of a split; lanes and waves over splits).
So a logit's term is off by e = 3 |d| 2^-24 + (1 + moves) 2^-23 of itself, log l by E0 = sum p e, and t / l by E0 D + E1 + 18 D 2^-24
with D = sum p |d| and E1 = sum p |d| e (16 additions in f32, d and its product rounded). Results are rounded once: half a
step, 2^-24 of them. Sums are f64.

All of these are independent: over many rows the root of the mean square is that of one rounding of each kind, at most a half
step each and (half a step / sqrt 3 evenly spread) less. Of a random order of n, ln n moves are expected. What is allowed for log
probabilities is 2^-24 (1 + sqrt(1 + ln rounds + 4) + D + |result|), each by its mean square."""
import numpy as np
import pytest

from . import kv_oracle as ko
from .test_gpu_logprobs import arguments, buffers, logits

pytestmark = pytest.mark.gpu


def rounds_of(rows, n, n_top, n_cu=256):
    """Of 16 logits that a thread takes: rows are split for two workgroups a CU, into no less than a round each."""
    granules = (n + 6) // 4
    splits = max(1, min(-(-2 * n_cu // rows), -(-granules // 1024), 64 if n_top else 256))
    return -(-(-(-granules // splits) + 3) // 1024)


def measure(dev, x, n_top):
    rows, n = x.shape
    rng = np.random.default_rng(n)
    token = rng.integers(0, n, (rows, 3))
    token[:, 0] = x.argmax(1)
    with ko.OnDevice(dev, **buffers(x, token, n_top)) as d:
        dev.logprobs_dev(arguments(d, x, token, n_top))
        dev.synchronize()
        lp, h = d.get("lp").astype(np.float64), d.get("h")[:-1].astype(np.float64)
    y = x.astype(np.float64)
    d = y - y.max(1, keepdims=True)
    e = np.exp(d)
    l = e.sum(1, keepdims=True)
    p, log_l = e / l, np.log(l)
    want, entropy = np.take_along_axis(d, token, 1) - log_l, log_l[:, 0] - (p * d).sum(1)
    moves = rounds_of(rows, n, n_top) + 4
    off = 3 * np.abs(d) * 2.0 ** -24 + (1 + moves) * 2.0 ** -23
    D, E0, E1 = ((p * a).sum(1) for a in (np.abs(d), off, off * np.abs(d)))
    return lp - want, want, E0, h - entropy, entropy, E0 * (1 + D) + E1 + 18 * D * 2.0 ** -24, D


SHAPES = [(1, 151936), (7, 1000), (64, 32003), (130, 100003), (2100, 517), (600, 20001)]


@pytest.mark.parametrize("rows,n", SHAPES)
@pytest.mark.parametrize("size", [0.3, 3.0, 12.0])
@pytest.mark.parametrize("n_top", [0, 20])
def test_random_rows(dev, rows, n, size, n_top):
    rng = np.random.default_rng(rows + n)
    off, want, e0, off_h, entropy, e1, D = measure(dev, logits(rng, rows, n, size, ties=False), n_top)
    assert (np.abs(off) <= e0[:, None] + 2.0 ** -24 * np.abs(want)).all()
    assert (np.abs(off_h) <= e1 + 2.0 ** -24 * np.abs(entropy)).all()
    if rows < 50:
        return
    rms = lambda a: np.sqrt(np.mean(np.square(a)))
    moves = 1 + np.log(rounds_of(rows, n, n_top)) + 4
    for i in range(want.shape[1]):
        assert rms(off[:, i]) <= 2.0 ** -24 * (1 + np.sqrt(moves) + rms(D) + rms(want[:, i]))


@pytest.mark.parametrize("n", [5000, 60000])
@pytest.mark.parametrize("size", [2.0, 60.0])
def test_rising_rows(dev, n, size):
    """Every round moves the maximum."""
    x = np.stack([np.linspace(0, size, n), np.linspace(-size, 0, n) ** 3 / size ** 2]).astype(np.float32)
    x = np.repeat(x, 300, 0)  # (so many that a row is not split)
    off, want, e0, off_h, entropy, e1, _ = measure(dev, x, 0)
    assert (np.abs(off) <= e0[:, None] + 2.0 ** -24 * np.abs(want)).all()
    assert (np.abs(off_h) <= e1 + 2.0 ** -24 * np.abs(entropy)).all()
