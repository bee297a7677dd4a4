"""Attention over pages whose value scales differ by far: a key weighs what its
probability times its value scale says, whatever the scales of other pages.
kv_scores.py has the bound, per row and head over the keys that a row sees."""
import numpy as np
import pytest

from . import kv_oracle as ko, kv_scores as ks
from .test_gpu_attn_paged import CHANGES, SHAPES, queries, run

pytestmark = pytest.mark.gpu

STEPS = [("single", 0), ("prompt", 0), ("prompt", 1)]


def one_large_page(rng, lengths, adds, block, n_kv, hd, heads, kq, at, log2_scale, log2_weight):
    """Requests whose block `at` (counted from the end if negative) has values
    2^log2_scale as large as the others' and keys that all queries score about
    log2_weight (in log2 units) above the others'."""
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, block, n_kv, hd)
    # alike scales elsewhere, so that what is lost is lost to the one page
    cache.vs[np.isfinite(cache.vs)] = 0.02
    u = rng.choice([-1, 1], (n_kv, hd))
    q = np.repeat(u, heads // n_kv, 0)[None] + 0.05 * rng.standard_normal((sum(adds), heads, hd))
    for r, n in enumerate(kv_len):
        page = table[r, at % ko.blocks_of(int(n), block)]
        cache.vs[page] = np.float32(0.02 * 2.0 ** log2_scale)
        cache.k[page] = np.sign(log2_weight) * 127 * u[:, None, :]
        cache.ks[page] = np.float32(abs(log2_weight) * np.log(2) / (kq * 127 * hd))
    return cache, table, q_start, kv_len, q.astype(np.float32)


@pytest.mark.parametrize("steps,large", STEPS)
@pytest.mark.parametrize("at", [0, 3, -1])
@pytest.mark.parametrize("log2_scale,log2_weight", [
    (20, -200), (24, -200), (30, -200), (36, -200), (60, -200), (100, -200),  # of no weight
    (24, -30), (30, -60),       # of little
    (24, -24), (30, -25), (60, -50), (100, -80),  # of weight as others', or more
    (-30, 0), (-60, 10), (-60, 70)])  # of less value, and the row's only key of weight
def test_a_page_of_large_values(dev, option, steps, large, at, log2_scale, log2_weight):
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(100 + log2_scale + at)
    lengths, adds = ([400, 150, 3000], [1, 1, 1]) if steps == "single" else ([200, 0, 70], [70, 150, 33])
    heads, n_kv, hd, block, kq = 8, 2, 64, 16, 0.125
    cache, table, q_start, kv_len, q = one_large_page(rng, lengths, adds, block, n_kv, hd, heads, kq, at, log2_scale, log2_weight)
    got = run(dev, cache, table, q_start, kv_len, q, kq)
    ks.check(got, cache, table, q_start, kv_len, q, kq)


@pytest.mark.parametrize("heads,n_kv,hd,block", SHAPES)
@pytest.mark.parametrize("steps,large", STEPS)
def test_scales_of_any_size(dev, option, steps, large, heads, n_kv, hd, block):
    """Value scales over 80 powers of two, rising and falling through a
    request's pages, and scores that favour now one page and now another."""
    if hd > 128 and large:
        pytest.skip("heads of more than 128 have no large row blocks")
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(hd + heads)
    lengths, adds = ([5, 300, 1000, 2200], [1] * 4) if steps == "single" else ([0, 500, 130], [150, 33, 70])
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, block, n_kv, hd)
    for r, n in enumerate(kv_len):
        for b in range(ko.blocks_of(int(n), block)):
            cache.vs[table[r, b]] = 2.0 ** rng.uniform(-40, 40, n_kv).astype(np.float32)
            cache.ks[table[r, b]] *= 2.0 ** rng.uniform(-6, 1.5, n_kv).astype(np.float32)
    q = queries(rng, sum(adds), heads, hd, 2.0)
    got = run(dev, cache, table, q_start, kv_len, q, 1 / np.sqrt(hd))
    ks.check(got, cache, table, q_start, kv_len, q, 1 / np.sqrt(hd))


@pytest.mark.parametrize("steps,large", STEPS)
@pytest.mark.parametrize("rising", [1, -1])
def test_scores_that_rise_while_values_fall(dev, option, steps, large, rising):
    """Every page outweighs the one before it by 2^4 and its values are 2^-4 as
    large, or the other way round: all contribute alike."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(31)
    heads, n_kv, hd, block, kq = 4, 2, 64, 16, 0.125
    lengths, adds = ([310, 170], [1, 1]) if steps == "single" else ([150, 0], [150, 129])
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, block, n_kv, hd)
    u = rng.choice([-1, 1], (n_kv, hd))
    for r, n in enumerate(kv_len):
        blocks = ko.blocks_of(int(n), block)
        for b in range(blocks):
            page, log2 = table[r, b], 4.0 * rising * (b - blocks / 2)
            cache.k[page] = np.sign(log2) * 127 * u[:, None, :]
            cache.ks[page] = np.float32(abs(log2) * np.log(2) / (kq * 127 * hd))
            cache.vs[page] = np.float32(2.0 ** -log2)
    q = (np.repeat(u, heads // n_kv, 0)[None] + 0.01 * rng.standard_normal((sum(adds), heads, hd))).astype(np.float32)
    got = run(dev, cache, table, q_start, kv_len, q, kq)
    ks.check(got, cache, table, q_start, kv_len, q, kq)


@pytest.mark.parametrize("steps,large", STEPS)
@pytest.mark.parametrize("change", CHANGES)
def test_masks_per_row(dev, option, change, steps, large):
    """Scores of every kind, and a bound of each row and head of its own."""
    option("ATTNP_LARGE", large)
    heads, n_kv, hd, block = 8, 2, 128, 16
    rng = np.random.default_rng(len(change))
    lengths = [0, 1, 63, 64, 200, 450, 1300] if steps == "single" else [0, 40, 0, 333, 100]
    adds = [1] * 7 if steps == "single" else [70, 129, 1, 33, 200]
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, block, n_kv, hd)
    o = dict(CHANGES[change])
    if o.pop("slopes", False):
        o["slopes"] = (2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)).astype(np.float32)
    if o.pop("prefix", False):
        o["prefix"] = np.array([0, 20, 64, 70, 10 ** 6, -5, 400][:len(adds)], np.int32)
    q = queries(rng, sum(adds), heads, hd, 2.0)
    got = run(dev, cache, table, q_start, kv_len, q, 1 / np.sqrt(hd), **dict(o))
    ks.check(got, cache, table, q_start, kv_len, q, 1 / np.sqrt(hd), **o)


@pytest.mark.parametrize("steps,large", STEPS)
def test_garbage_that_no_row_sees_per_row(dev, option, steps, large):
    """Scales of NaN and infinity behind the window, of 10^30 to 10^-38 and zero
    in the last page: the bound of a row is that of the scales it sees."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(14)
    lengths, adds = ([700, 300], [1, 1]) if steps == "single" else ([400, 0], [200, 150])
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, 16, 2, 64)
    q = queries(rng, sum(adds), 4, 64)
    window = 100
    first = [max(0, n - window) // 16 for n in lengths]
    for r in range(2):
        for b in range(first[r]):
            cache.ks[table[r, b]], cache.vs[table[r, b]] = np.nan, [np.inf, np.nan]
    last = [int(table[r, kv_len[r] // 16 - 1]) for r in range(2)]
    cache.vs[last[0]], cache.ks[last[0]] = [1e30, 1e-30], [0.0, 1e-37]
    cache.vs[last[1]], cache.ks[last[1]] = [0.0, 3e-38], [1e-3, 0.0]
    got = run(dev, cache, table, q_start, kv_len, q, 0.2, window=window)
    assert np.isfinite(got).all()
    ks.check(got, cache, table, q_start, kv_len, q, 0.2, window=window)
