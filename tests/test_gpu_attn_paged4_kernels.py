"""Attention over the paged 4-bit cache of single and drafted tokens, in shapes that between them reach each kernel for few
rows with each number of waves, against its definition in 64 bits (kv_scores)."""
import numpy as np
import pytest

from . import kv4_oracle as k4
from . import kv_scores as ks
from .test_gpu_attn_paged4 import queries, run

pytestmark = pytest.mark.gpu


def requests(*a):
    """Of kv4_oracle, with subs as an append writes them, which are never 0: a key of all the weight whose values are zeros
    says nothing, and kv_scores takes no such row."""
    made = k4.requests(*a)
    for sub in (made[0].ksub, made[0].vsub):
        sub[sub == 0] = 1
    return made


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("group,adds", [(1, 1), (2, 1), (3, 1), (4, 1), (8, 1), (9, 1), (1, 2), (2, 2)])
@pytest.mark.parametrize("row_waves", [1, 4])
@pytest.mark.parametrize("splits", [-1, 3])
def test_few_rows(dev, option, hd, group, adds, row_waves, splits):
    """Rows up to and past the border between the two kernels for few, at each width."""
    option("ATTNP_ROW_WAVES", row_waves)
    option("ATTNP_SPLITS", splits)
    rng = np.random.default_rng(hd + 10 * group + adds)
    lengths = [0, 1, 62, 63, 64, 300, 1500]
    cache, pages, q_start, kv_len = requests(rng, lengths, [adds] * 7, 32, 2, hd)
    q = queries(rng, 7 * adds, 2 * group, hd, 2.0)
    got = run(dev, cache, pages, q_start, kv_len, q, 1 / np.sqrt(hd))
    ks.check(got, cache, pages, q_start, kv_len, q, 1 / np.sqrt(hd))


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("n_req", [130, 257, 300])
@pytest.mark.parametrize("change", ["none", "masks"])
def test_single_tokens_of_many_requests(dev, hd, n_req, change):
    """Batches that need no split, and of more requests than are dealt to workgroups, some of them waiting."""
    rng = np.random.default_rng(hd + n_req)
    lengths = [int(x) for x in np.exp(rng.uniform(0, 6.5, n_req))]
    adds = [int(x) for x in rng.choice([0, 1, 1, 1], n_req)]
    cache, pages, q_start, kv_len = requests(rng, lengths, adds, 16, 4, hd)
    q = queries(rng, sum(adds), 4, hd, 2.0)
    o = {} if change == "none" else dict(cap=20.0, window=100, slopes=2.0 ** -np.arange(4, dtype=np.float32))
    got = run(dev, cache, pages, q_start, kv_len, q, 1 / np.sqrt(hd), **dict(o))
    ks.check(got, cache, pages, q_start, kv_len, q, 1 / np.sqrt(hd), **o)
