"""Positions up to the last that max_blocks allows, 2^31 - 16, and chunks and
heads whose product passes 2^31. Requests share pages, or have only the last of
them, so that the caches are small."""
import numpy as np
import pytest

import siphon_amd as sa

from . import kv_oracle as ko, kv_scores as ks
from .test_gpu_attn_paged import queries

pytestmark = pytest.mark.gpu


def htod(dev, ptr, a):
    a = np.ascontiguousarray(a)
    dev._check(dev.L.sihip_memcpy_htod(dev.ctx, ptr, a.ctypes.data, a.nbytes))


@pytest.mark.parametrize("block", [16, 32, 256])
@pytest.mark.parametrize("new,large", [(1, 0), (5, 0), (150, 0), (150, 1)])
@pytest.mark.parametrize("before_end", [0, 1, 17, 40])
def test_the_last_positions(dev, option, block, new, large, before_end):
    """A window's worth of keys, and new ones, at the end of a full table row,
    beside a short request. The result is that of the same pages at the
    beginning of a row; table entries before the window are never read."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(block + new)
    heads, n_kv, hd, window = 6, 2, 64, 100
    end = 1024 - before_end
    cache, table, q_start, kv_len = ko.requests(rng, [end - new, 20], [new, 2], block, n_kv, hd)
    held = ko.blocks_of(1024, block)
    if ko.blocks_of(end, block) < held:
        table = np.pad(table, ((0, 0), (0, held)))
    cache.vs[np.isnan(cache.vs)] = 1.0
    max_blocks = (2 ** 31 - 1) // block
    far = kv_len.copy()
    far[0] += (max_blocks - held) * block
    q = queries(rng, new + 2, heads, hd, 2.0)
    rows = dev.alloc(2 * max_blocks * 4)
    try:
        htod(dev, rows.ptr + 4 * (max_blocks - held), table[0, :held])
        htod(dev, rows.ptr + 4 * max_blocks, table[1, :held])
        k, v = rng.standard_normal((2, new + 2, n_kv, hd)).astype(np.float32)
        with ko.OnDevice(dev, q=q, out=np.full_like(q, 55), kn=k, vn=v, q_start=q_start, kv_len=far) as d:
            c = ko.put_cache(d, cache)
            b = sa.KvBatch(q_start=d.ptr("q_start"), kv_len=d.ptr("kv_len"), table=rows.ptr, n_req=2, max_blocks=max_blocks,
                           n_tok=new + 2, max_q=max(new, 2), max_kv=max_blocks * block)
            a = sa.AttnPaged(q=d.ptr("q"), ldq=heads * hd, out=d.ptr("out"), ldo=heads * hd, n_head=heads, kq_scale=0.1, window=window)
            dev.kv_append_dev(c, b, d.ptr("kn"), n_kv * hd, d.ptr("vn"), n_kv * hd)
            dev.attn_paged_dev(c, b, a)
            dev.synchronize()
            got = {x: d.get(x) for x in ("k", "v", "out")}
    finally:
        rows.free()
    cache.append(table, q_start, kv_len, k, v)
    assert np.array_equal(got["k"], cache.k) and np.array_equal(got["v"], cache.v)
    ks.check(got["out"], cache, table, q_start, kv_len, q, 0.1, window=window)


def test_chunks_and_heads_past_32_bits(dev):
    """4096 KV heads over 33.6 million keys: 2^31 + 4096 chunks. Two pages take
    turns; in each one key of 256 has all the weight, and all repeats of a page
    add equal numbers: 131100 / 4 of them a lane at most, each rounded by 2^-24,
    and 2^-20 for the rest; the other keys' weight is below 2^-25 a page."""
    heads, hd, block, blocks = 4096, 16, 256, 131100
    rng = np.random.default_rng(3)
    k = np.zeros((2, heads, block, hd), np.int8)
    v = rng.integers(-127, 128, (2, heads, hd, block)).astype(np.int8)
    peak = rng.integers(0, block, (2, heads))
    for p in range(2):
        k[p, np.arange(heads), peak[p]] = 100
    ones = np.ones((2, heads), np.float32)
    kv_len = blocks * block
    assert heads * (kv_len // 64) > 1 << 31
    q = np.ones((1, heads, hd), np.float32)
    with ko.OnDevice(dev, q=q, out=np.full_like(q, 55), k=k, v=v, ks=ones, vs=ones, table=(np.arange(blocks) % 2).astype(np.int32),
                     q_start=np.array([0, 1], np.int32), kv_len=np.array([kv_len], np.int32)) as d:
        c = sa.KvCache(k=d.ptr("k"), v=d.ptr("v"), k_scale=d.ptr("ks"), v_scale=d.ptr("vs"), n_pages=2, n_head_kv=heads, head_dim=hd,
                       block=block)
        b = sa.KvBatch(q_start=d.ptr("q_start"), kv_len=d.ptr("kv_len"), table=d.ptr("table"), n_req=1, max_blocks=blocks, n_tok=1,
                       max_q=1, max_kv=kv_len)
        # a score of 1600 kq = 17.6 natural units above the others
        a = sa.AttnPaged(q=d.ptr("q"), ldq=heads * hd, out=d.ptr("out"), ldo=heads * hd, n_head=heads, kq_scale=0.011)
        dev.attn_paged_dev(c, b, a)
        dev.synchronize()
        got = d.get("out")[0].astype(np.float64)
    w = np.exp(np.where(np.arange(block) == peak[..., None], 0.0, -1600 * 0.011))
    w /= w.sum((0, 2))[None, :, None]
    x = v.astype(np.float64)
    want, size = np.einsum("pht,phdt->hd", w, x), np.einsum("pht,phdt->hd", w, np.abs(x))
    assert (np.abs(got - want) <= 2 * (blocks / 4 * 2.0 ** -24 + 2.0 ** -20) * size).all()
