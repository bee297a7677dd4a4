"""The 4-bit cache and the rotation at positions up to the last that max_blocks allows, 2^31 - 16, and chunks and heads whose
product passes 2^31 (as test_gpu_kv_far has them for 8 bits)."""
import numpy as np
import pytest

import siphon_amd as sa

from . import kv4_oracle as k4
from . import kv_oracle as ko
from . import kv_scores as ks
from .test_gpu_attn_paged4 import queries
from .test_gpu_kv4_cache import positions, same
from .test_gpu_kv_far import htod

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", [16, 32, 256])
@pytest.mark.parametrize("new,large", [(1, 0), (5, 0), (150, 0), (150, 1)])
@pytest.mark.parametrize("before_end", [0, 1, 17, 40])
@pytest.mark.parametrize("heads,hd", [(2, 64), (6, 64), (6, 128), (4, 160)])
def test_the_last_positions(dev, option, block, new, large, before_end, heads, hd):
    """A window's worth of keys, and new ones, at the end of a full table row, beside a short request. The result is that of the
    same pages at the beginning of a row; table entries before the window are never read."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(block + new + hd)
    n_kv, window = 2, 100
    end = 1024 - before_end
    cache, table, q_start, kv_len = k4.requests(rng, [end - new, 20], [new, 2], block, n_kv, hd)
    held = ko.blocks_of(1024, block)
    if ko.blocks_of(end, block) < held:
        table = np.pad(table, ((0, 0), (0, held)))
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
            c = k4.put_cache(d, cache)
            b = sa.KvBatch(q_start=d.ptr("q_start"), kv_len=d.ptr("kv_len"), table=rows.ptr, n_req=2, max_blocks=max_blocks,
                           n_tok=new + 2, max_q=max(new, 2), max_kv=max_blocks * block)
            a = sa.AttnPaged(q=d.ptr("q"), ldq=heads * hd, out=d.ptr("out"), ldo=heads * hd, n_head=heads, kq_scale=0.1, window=window)
            dev.kv4_append_dev(c, b, sa.KvRows(k=d.ptr("kn"), v=d.ptr("vn"), ldk=n_kv * hd, ldv=n_kv * hd))
            dev.attn_paged4_dev(c, b, a)
            dev.synchronize()
            got = {x: d.get(x) for x in ("k", "v", "ksub", "vsub", "ks", "vb", "out")}
    finally:
        rows.free()
    cache.append(table, q_start, kv_len, k, v)
    for name, x in cache.arrays().items():
        assert same(got[name], x), name
    ks.check(got["out"], cache, table, q_start, kv_len, q, 0.1, window=window)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("neighbours", [0, 1])
def test_rotation_at_the_last_positions(dev, bits, neighbours):
    """A table of 2^31 - 16 rows of one pair, of which the last are written."""
    rng = np.random.default_rng(bits)
    block, n_kv, hd, heads, new, end = 16, 2, 32, 4, 40, 1024
    mod = k4 if bits == 4 else ko
    cache, table, q_start, kv_len = mod.requests(rng, [end - new], [new], block, n_kv, hd)
    held, max_blocks = end // block, (2 ** 31 - 1) // block
    length = max_blocks * block
    angle = rng.uniform(-4, 4, end)
    tail = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)[:, None]  # of the positions that the pages stand for
    rows, rope = dev.alloc(max_blocks * 4), dev.alloc(length * 8)
    k, v, q = (rng.standard_normal((new, h, hd)).astype(np.float32) for h in (n_kv, n_kv, heads))
    try:
        htod(dev, rows.ptr + 4 * (max_blocks - held), table[0, :held])
        htod(dev, rope.ptr + 8 * (length - end), tail)
        with ko.OnDevice(dev, q=q, kn=k, vn=v, q_start=q_start, kv_len=np.array([length], np.int32)) as d:
            c = mod.put_cache(d, cache)
            b = sa.KvBatch(q_start=d.ptr("q_start"), kv_len=d.ptr("kv_len"), table=rows.ptr, n_req=1, max_blocks=max_blocks, n_tok=new,
                           max_q=new, max_kv=length)
            r = sa.KvRows(k=d.ptr("kn"), v=d.ptr("vn"), ldk=n_kv * hd, ldv=n_kv * hd, q=d.ptr("q"), q_out=d.ptr("q"), ldq=heads * hd,
                          ldq_out=heads * hd, n_head=heads, rope=rope.ptr, rope_len=length, rope_dim=2, rope_neighbours=neighbours)
            (dev.kv4_append_dev if bits == 4 else dev.kv_append_rope_dev)(c, b, r)
            dev.synchronize()
            names = ("k", "v", "ksub", "vsub", "ks", "vb") if bits == 4 else ("k", "v", "ks", "vs")
            got = {x: d.get(x) for x in (*names, "q")}
    finally:
        rows.free()
        rope.free()
    pos = positions(q_start, kv_len, new)
    cache.append(table, q_start, kv_len, k4.rotate(k, pos, tail, neighbours), v)
    for name in names:
        assert same(got[name], cache.arrays()[name] if bits == 4 else getattr(cache, name)), name
    assert same(got["q"], k4.rotate(q, pos, tail, neighbours))


def test_chunks_and_heads_past_32_bits(dev):
    """4096 KV heads over 33.6 million keys: 2^31 + 4096 chunks. Two pages take turns; in each one key of 256 has all the weight,
    and all repeats of a page add equal numbers: 131100 / 4 of them a lane at most, each rounded by 2^-24, and 2^-20 for the
    rest; the other keys' weight is below 2^-25 a page."""
    heads, hd, block, blocks = 4096, 32, 256, 131100
    rng = np.random.default_rng(3)
    cache = k4.Cache(rng, 2, heads, hd, block)
    peak = rng.integers(0, block, (2, heads))
    cache.k[:] = 0
    for p in range(2):
        cache.k[p, np.arange(heads), peak[p]] = 5
    cache.ksub[:], cache.vsub[:], cache.ks[:], cache.vb[:] = 10, 16, 0x3f80, 0x3f80
    kv_len = blocks * block
    assert heads * (kv_len // 64) > 1 << 31
    q = np.ones((1, heads, hd), np.float32)
    with ko.OnDevice(dev, q=q, out=np.full_like(q, 55), table=(np.arange(blocks) % 2).astype(np.int32), q_start=np.array([0, 1], np.int32),
                     kv_len=np.array([kv_len], np.int32)) as d:
        c = k4.put_cache(d, cache)
        b = sa.KvBatch(q_start=d.ptr("q_start"), kv_len=d.ptr("kv_len"), table=d.ptr("table"), n_req=1, max_blocks=blocks, n_tok=1,
                       max_q=1, max_kv=kv_len)
        # a score of 1600 kq = 17.6 natural units above the others
        a = sa.AttnPaged(q=d.ptr("q"), ldq=heads * hd, out=d.ptr("out"), ldo=heads * hd, n_head=heads, kq_scale=0.011)
        dev.attn_paged4_dev(c, b, a)
        dev.synchronize()
        got = d.get("out")[0].astype(np.float64)
    w = np.exp(np.where(np.arange(block) == peak[..., None], 0.0, -1600 * 0.011))
    w /= w.sum((0, 2))[None, :, None]
    x = cache.v.astype(np.float64) * 16
    want = (w[:, :, None] * x).sum((0, 3))
    size = (w[:, :, None] * np.abs(x)).sum((0, 3))
    assert (np.abs(got - want) <= 2 * (blocks / 4 * 2.0 ** -24 + 2.0 ** -20) * size).all()
