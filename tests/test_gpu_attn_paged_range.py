"""Attention over the paged caches at the ends of their range (kv_scores has the bound)."""
import numpy as np
import pytest

from . import kv4_oracle as k4
from . import kv_oracle as ko
from . import kv_scores as ks
from . import test_gpu_attn_paged as eight
from .test_gpu_attn_paged4 import queries, run

pytestmark = pytest.mark.gpu

# (query heads of a KV head, requests, large row blocks): of 4 bits the kernel for the fewest rows, the one for few, the one for many
KERNELS = {"fewest": (1, ([0, 2, 299, 1500], [1] * 4), 0), "few": (10, ([0, 2, 299, 1500], [1] * 4), 0),
           "many": (3, ([0, 37, 700], [1, 129, 70]), 1)}


def filled(bits, lengths, adds, block, k, v, rng):
    """A cache that holds the rows k and v [token of all requests, KV head, dim], written as an append writes them."""
    make = (k4 if bits == 4 else ko).requests
    cache, pages, q_start, kv_len = make(rng, lengths, adds, block, k.shape[1], k.shape[2])
    cache.append(pages, np.concatenate([[0], np.cumsum(kv_len)]), kv_len, k, v)
    return cache, pages, q_start, kv_len


def attend(bits, *a, **o):
    return (run if bits == 4 else eight.run)(*a, **o)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("hd,block", [(128, 16), (64, 64), (96, 32), (256, 32)])
@pytest.mark.parametrize("log2", [117, 122, 126])
@pytest.mark.parametrize("row_waves,splits", [(1, 1), (4, 1), (1, 5), (4, 5)])
def test_large_values(dev, option, bits, kernel, hd, block, log2, row_waves, splits):
    """Values up to 2^126, the largest that the 4-bit cache tells apart: means of them are numbers, however many there are and
    whatever the sums of their weights times values."""
    group, (lengths, adds), large = KERNELS[kernel]
    for name, value in (("LARGE", large), ("ROW_WAVES", row_waves), ("SPLITS", splits)):
        option("ATTNP_" + name, value)
    rng = np.random.default_rng(hd + log2)
    n, n_kv = sum(lengths) + sum(adds), 2
    k, v = rng.standard_normal((n, n_kv, hd)), rng.uniform(-1, 1, (n, n_kv, hd)) * 2.0 ** log2
    v[:, :, ::5] = np.abs(v[:, :, ::5])  # dims whose values do not cancel
    cache, pages, q_start, kv_len = filled(bits, lengths, adds, block, k.astype(np.float32), v.astype(np.float32), rng)
    q = queries(rng, sum(adds), group * n_kv, hd, 2.0)
    got = attend(bits, dev, cache, pages, q_start, kv_len, q, 1 / np.sqrt(hd))
    ks.check(got, cache, pages, q_start, kv_len, q, 1 / np.sqrt(hd))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("hd,block", [(128, 16), (64, 64), (96, 32), (256, 32)])
@pytest.mark.parametrize("log2_q,log2_k,change", [
    (110, -90, "none"), (118, -98, "none"), (124, -98, "slopes"), (126.5, -98, "none"), (126.5, -98, "cap"), (126.5, -60, "none"),
    (-10, 80, "none"), (-60, 60, "none")])
def test_sizes_of_queries_and_keys(dev, option, bits, kernel, hd, block, log2_q, log2_k, change):
    """Queries and keys of any size whose scores are of ordinary size, among them the largest that sums of products can have:
    keys whose dims all have the largest magnitude and the queries' signs."""
    group, (lengths, adds), large = KERNELS[kernel]
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(hd + int(log2_q) % 256)
    n, n_kv = sum(lengths) + sum(adds), 2
    u = rng.choice([-1, 1], (n_kv, hd))
    k = rng.uniform(-1, 1, (n, n_kv, hd)) * u
    k[::3] = rng.choice([-1, 1], (len(k[::3]), 1, 1)) * u
    v = rng.standard_normal((n, n_kv, hd))
    cache, pages, q_start, kv_len = filled(bits, lengths, adds, block, (k * 2.0 ** log2_k).astype(np.float32), v.astype(np.float32), rng)
    q = np.repeat(u, group, 0)[None] * rng.uniform(0.7, 1.3, (sum(adds), group * n_kv, hd))
    q = (q * 2.0 ** log2_q).astype(np.float32)
    kq = 20 / hd * 2.0 ** -(log2_q + log2_k)
    o = dict(none={}, cap=dict(cap=10.0), slopes=dict(slopes=2.0 ** -np.arange(group * n_kv, dtype=np.float32)))[change]
    got = attend(bits, dev, cache, pages, q_start, kv_len, q, kq, **dict(o))
    ks.check(got, cache, pages, q_start, kv_len, q, float(np.float32(kq)), **o)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("hd,block", [(128, 16), (64, 64), (96, 32), (256, 32)])
@pytest.mark.parametrize("log2_q,log2_k,change", [(-10, 126, "none"), (-60, 117, "none"), (-100, 122, "slopes"), (-120, 126, "cap"),
                                                  (-124, 126, "none")])
def test_the_largest_keys(dev, option, kernel, hd, block, log2_q, log2_k, change):
    """The same with keys up to the largest that 4 bits hold."""
    test_sizes_of_queries_and_keys(dev, option, 4, kernel, hd, block, log2_q, log2_k, change)
