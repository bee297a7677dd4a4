"""Capped scores at the ends of what a cap may be: tanh of anything over a tiny
cap is -1, 0 or 1, and a cap that no score comes near changes nothing."""
import numpy as np
import pytest

from . import kv_oracle as ko, kv_scores as ks
from .test_gpu_attn_paged import queries, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("steps,large", [("single", 0), ("prompt", 0), ("prompt", 1)])
@pytest.mark.parametrize("cap", [1.4e-45, 1e-39, 1e-38, 1e-30, 1e-6, 1e6, 1e30, 3.4e38])
@pytest.mark.parametrize("hd", [64, 128])
def test_smallest_and_largest_caps(dev, option, steps, large, cap, hd):
    """Beside ordinary ones: queries of zeros and of large and tiny numbers, and
    keys that are zero by their codes or by their scale."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(hd)
    lengths, adds = ([200, 90, 16, 400], [1] * 4) if steps == "single" else ([90, 0, 30], [70, 150, 33])
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, 16, 2, hd)
    for r in range(len(adds)):
        cache.ks[table[r, 0]] = 0.0
        cache.k[table[r, 1]] = 0  # every request has two pages
    q = queries(rng, sum(adds), 4, hd)
    q[::7] = 0.0
    q[1::7] *= np.float32(1e-30)
    q[2::7] *= np.float32(30)
    if cap < 1:  # (their scores are past f32's integers, and their factors past its range)
        q[3::7] *= np.float32(1e36)
    cap = float(np.float32(cap))
    got = run(dev, cache, table, q_start, kv_len, q, 0.1, cap=cap)
    ks.check(got, cache, table, q_start, kv_len, q, 0.1, cap=cap)
