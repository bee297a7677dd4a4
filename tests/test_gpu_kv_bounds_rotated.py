"""What a rotated append into the paged 8-bit cache leaves as it was: rows that are not to be written, bit for bit."""
import numpy as np
import pytest

from . import kv4_oracle as k4
from . import kv_oracle as ko
from .test_gpu_kv4_cache import Append, check, positions, same, step_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("max_q,max_kv", [(25, 43), (30, 44), (1, 44), (30, 11)])
def test_rows_that_are_not_written8(dev, block, max_q, max_kv):
    """Tokens past max_q, from max_kv on and behind the last: no keys, no values, no queries. A page outside the cache loses
    its keys and values and not its queries."""
    rng = np.random.default_rng(block)
    cache, pages, q_start, kv_len = ko.requests(rng, [10, 40, 0, 7], [30, 5, 9, 1], block, 2, 64)
    n = int(q_start[-1]) + 3
    k, v, q = (step_rows(rng, n, h, 64) for h in (2, 2, 4))
    pages[0, 1], pages[2, 0] = -3, cache.n_pages
    rope = k4.table(44, 64)
    got = Append(dev, cache, pages, q_start, kv_len, k, v, q, rope, max_q=max_q, max_kv=max_kv)
    pos = np.full(n, 2 ** 31)
    pos[:45] = positions(q_start, kv_len, 45)
    turned = np.minimum(pos, 43)
    cache.append(pages, q_start, kv_len, k4.rotate(k, turned, rope, False), v, max_q=max_q, max_kv=max_kv)
    check(got, cache)
    want = k4.rotate(q, turned, rope, False)
    late = np.concatenate([np.arange(b - a) >= max_q for a, b in zip(q_start, q_start[1:])] + [np.ones(3, bool)])
    want[late | (pos >= max_kv)] = 77
    assert same(got.q, want)


def test_requests_of_impossible_numbers8(dev):
    """They take part in nothing."""
    rng = np.random.default_rng(6)
    cache, pages, q_start, kv_len = ko.requests(rng, [10, 40, 0, 7], [30, 5, 9, 1], 16, 2, 64)
    n = int(q_start[-1]) + 3
    k, v, q = (step_rows(rng, n, h, 64) for h in (2, 2, 4))
    rope = k4.table(44, 64)
    for q0, end in (([0, 60, 60, 60, 60], [70, 0, 0, 0]), ([-1, 1, 1, 1, 1], [42, 0, 0, 0]), ([2, 0, 0, 0, 0], [42, 22, 0, 0]),
                    ([0, 3, 3, 3, 3], [2, 0, 0, 0]), ([0, 1, 1, 1, 1], [-1, 0, 0, 0])):
        got = Append(dev, cache, pages, np.array(q0), np.array(end), k, v, q, rope, max_q=25, max_kv=43)
        check(got, cache)
        assert (got.q == 77).all()
