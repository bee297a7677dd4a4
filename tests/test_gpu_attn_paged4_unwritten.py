"""Attention over the paged 4-bit cache beside memory that nothing was written to (kv_scores has the bound)."""
import numpy as np
import pytest

from . import kv4_oracle as k4
from . import kv_scores as ks
from .test_gpu_attn_paged4 import queries, run

pytestmark = pytest.mark.gpu

SHAPES = [(128, 16), (64, 64), (96, 32)]


def unwritten(cache, pages, r, first, end):
    """What a cache may hold of tokens that nothing was written to."""
    junk = [0x7fc0, 0x7f80, 0xff80, 0xffff]  # NaN, infinities, another NaN
    for t in range(first, end):
        page, at = pages[r, t // cache.block], t % cache.block
        cache.ks[page, :, at], cache.vb[page, :, at] = junk[t % 4], junk[t // 4 % 4]


@pytest.mark.parametrize("large", [0, 1])
@pytest.mark.parametrize("hd,block", SHAPES)
@pytest.mark.parametrize("max_q", [1, 2, 9, 50, 64, 97])
@pytest.mark.parametrize("o", [{}, {"window": 40}, {"prefix": 30}])
def test_tokens_that_were_never_written(dev, option, large, hd, block, max_q, o):
    """A request of more new tokens than max_q: those past it are written by no append, so their
    scales may be anything, also in the chunk and the page of the last row that there is."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(hd + max_q)
    lengths, adds, heads = [37, 500, 0], [70, 129, 98], 4
    cache, pages, q_start, kv_len = k4.requests(rng, lengths, adds, block, 2, hd)
    q = queries(rng, sum(adds), heads, hd, 2.0)
    for r, (n, a) in enumerate(zip(lengths, adds)):
        unwritten(cache, pages, r, n + max_q, n + a)
    o = dict(o)
    if "prefix" in o:
        o["prefix"] = np.array([30, 500, 0], np.int32)
    got = run(dev, cache, pages, q_start, kv_len, q, 0.1, bounds=dict(max_q=max_q), **o)
    # the same requests, of as many tokens as are written
    some = np.concatenate([np.arange(a, min(a + max_q, b)) for a, b in zip(q_start, q_start[1:])])
    short = [min(a, max_q) for a in adds]
    ends = np.array([n + a for n, a in zip(lengths, short)])
    ks.check(got[some], cache, pages, np.concatenate([[0], np.cumsum(short)]), ends, q[some], 0.1, **o)
    got[some] = 55.0
    assert (got == 55.0).all()
