"""The bounds max_q and max_kv of a batch, below what the device's numbers say:
tokens past them are not written, and neither are the scales of their pages."""
import numpy as np
import pytest

from . import kv_oracle as ko
from .test_gpu_kv_cache import bits, step_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block,hd", [(16, 32), (64, 80), (256, 16)])
@pytest.mark.parametrize("max_q,max_kv", [(8, None), (1, None), (17, None), (40, None), (None, 1), (None, 30), (None, 64), (None, 100),
                                          (8, 30), (20, 70), (3, 0), (0, 50), (10 ** 6, 2 ** 31 - 1)])
def test_append_stops_at_its_bounds(dev, block, hd, max_q, max_kv):
    rng = np.random.default_rng(block)
    lengths, adds = [0, 13, 29, 60, 96, 0, 65], [20, 7, 40, 5, 40, 1, 33]
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, block, 2, hd)
    fresh = [int(table[r, b]) for r in range(7) for b in range(ko.blocks_of(lengths[r], block), table.shape[1])
             if b < ko.blocks_of(int(kv_len[r]), block)]
    cache.ks[fresh], cache.vs[fresh] = np.nan, np.nan  # written by this step first, or not at all
    n, width = sum(adds), 2 * hd
    k, v = step_rows(rng, n, 2, hd), step_rows(rng, n, 2, hd)
    with ko.OnDevice(dev, kn=k, vn=v) as d:
        c = ko.put_cache(d, cache)
        b = ko.put_batch(d, table, q_start, kv_len, n, max_q=n if max_q is None else max_q, max_kv=max_kv)
        dev.kv_append_dev(c, b, d.ptr("kn"), width, d.ptr("vn"), width)
        dev.synchronize()
        got = {x: d.get(x) for x in ("k", "v", "ks", "vs")}
    for r in range(7):
        m = min(adds[r], n if max_q is None else max_q, (2 ** 31 if max_kv is None else max_kv) - lengths[r])
        if m > 0:
            cache.append(table[r:r + 1], [q_start[r], q_start[r] + m], [lengths[r] + m], k, v)
    for name in ("k", "v"):
        assert np.array_equal(got[name], getattr(cache, name)), name
        assert np.array_equal(bits(got[name + "s"]), bits(getattr(cache, name + "s"))), name + " scales"
