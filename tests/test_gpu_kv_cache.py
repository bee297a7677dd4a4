"""The paged 8-bit KV cache on the device against its restatement in numpy
(kv_oracle.py): plans, writes and reads are exact, bit for bit."""
import numpy as np
import pytest

import siphon_amd as sa

from . import kv_oracle as ko

pytestmark = pytest.mark.gpu


# ---- plans -------------------------------------------------------------------


def run_plan(dev, length, add, free, n_free, table, n_tok, block):
    n = len(length)
    with ko.OnDevice(dev, len=np.asarray(length, np.int32), add=np.asarray(add, np.int32), free=free,
                     n_free=np.array([n_free], np.int32), table=table, q_start=np.full(n + 1, 77, np.int32),
                     kv_len=np.full(n, 77, np.int32), slot=np.full(n_tok + 1, 77, np.int64),
                     pos=np.full(n_tok + 1, 77, np.int32), n_out=np.full(1, 77, np.int32),
                     status=np.full(1, 77, np.int32)) as d:
        dev.kv_plan_dev(sa.KvPlan(len=d.ptr("len"), add=d.ptr("add"), free_pages=d.ptr("free"), n_free=d.ptr("n_free"),
                                  n_req=n, n_tok=n_tok, n_pages=len(free), max_blocks=table.shape[1], block=block,
                                  table=d.ptr("table"), q_start=d.ptr("q_start"), kv_len=d.ptr("kv_len"),
                                  slot=d.ptr("slot"), pos=d.ptr("pos"), n_free_out=d.ptr("n_out"), status=d.ptr("status")))
        dev.synchronize()
        assert d.get("slot")[n_tok] == 77 and d.get("pos")[n_tok] == 77  # nothing past the arrays
        return (d.get("table"), d.get("q_start"), d.get("kv_len"), d.get("slot")[:n_tok], d.get("pos")[:n_tok],
                d.get("free"), int(d.get("n_out")[0]), int(d.get("status")[0]))


def check_plan(dev, length, add, free, n_free, table, n_tok, block, status=0):
    want = ko.plan(length, add, free, n_free, table, n_tok, block)
    got = run_plan(dev, length, add, free, n_free, table, n_tok, block)
    assert want[-1] == status == got[-1]
    for name, a, b in zip(("table", "q_start", "kv_len", "slot", "pos", "free", "n_free"), got, want):
        assert np.array_equal(a, b), name
    return got


def pool(rng, length, block, max_blocks, spare):
    """A table of requests with `length` tokens and the free list of the rest."""
    held = [ko.blocks_of(n, block) for n in length]
    order = rng.permutation(sum(held) + spare).astype(np.int32)
    table, at = np.full((len(length), max_blocks), -5, np.int32), 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    free = np.full(len(order), -9, np.int32)
    free[:spare] = order[at:]
    return table, free, spare


@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("n_req", [1, 2, 65, 1023, 1025, 4096])
def test_plan(dev, block, n_req):
    rng = np.random.default_rng(n_req * 7 + block)
    length = rng.integers(0, 5 * block, n_req)
    length[rng.random(n_req) < 0.3] //= block
    length[rng.random(n_req) < 0.3] *= 0
    length = np.minimum(length // (1 + 3 * (rng.random(n_req) < 0.2)), 5 * block)
    add = np.where(rng.random(n_req) < 0.5, 1, rng.integers(-1, 3 * block, n_req))
    add[rng.random(n_req) < 0.2] = 0
    table, free, n_free = pool(rng, length, block, 9, 4 * n_req + 3)
    total = int(add[add > 0].sum())
    for n_tok in (total, total + 1, total + 1500):
        check_plan(dev, length, add, free, n_free, table, n_tok, block)


def test_plan_ends_and_pages_change_hands(dev):
    """Pages of ended requests are taken again in the same step when the list
    is empty, and lengthen it when few are taken."""
    rng = np.random.default_rng(4)
    length, block = [100, 0, 64, 33, 1, 16], 16
    table, free, n_free = pool(rng, length, block, 12, 0)
    check_plan(dev, length, [-1, 90, 1, 0, -1, 16], free, n_free, table, 107, block)  # all 8 pages of the ended
    check_plan(dev, length, [-1, 16, 0, 0, -1, 1], free, n_free, table, 20, block)
    check_plan(dev, length, [-1] * 6, free, n_free, table, 0, block)  # nobody stays
    check_plan(dev, length, [0] * 6, free, n_free, table, 3, block)
    check_plan(dev, [0] * 6, [-1] * 6, free, n_free, table, 3, block)


@pytest.mark.parametrize("status,change", [
    (1, dict(length=[-1, 5, 20])), (1, dict(add=[1, -2, 3])), (2, dict(add=[1, 1, 16 * 9 - 19])),
    (2, dict(length=[16 * 9 + 1, 5, 20])), (2, dict(length=[2 ** 31 - 1, 5, 20])), (2, dict(add=[2 ** 31 - 1, 1, 1])),
    (4, dict(n_tok=2)), (8, dict(add=[1, 90, 90], n_tok=200)), (16, dict(n_free=-1)), (16, dict(n_free=100)),
    (16, dict(add=[-1, 1, 3], n_free=8)), (1 + 4, dict(add=[-7, 30, 30])), (4 + 8, dict(add=[1, 90, 90])),
])
def test_plan_that_cannot_be(dev, status, change):
    """Nothing is taken, given back or overwritten, and the outputs describe
    a step without tokens."""
    a = {"length": [3, 5, 20], "add": [1, 1, 3], "n_tok": 9, "n_free": None, **change}
    table, free, n_free = pool(np.random.default_rng(1), [3, 5, 20], 16, 9, 4)
    n_free = n_free if a["n_free"] is None else a["n_free"]
    got = check_plan(dev, a["length"], a["add"], free, n_free, table, a["n_tok"], 16, status)
    assert np.array_equal(got[0], table) and np.array_equal(got[5], free)
    assert not got[1].any() and (got[3] == -1).all() and (got[4] == -1).all()


def test_plan_with_foreign_pages(dev):
    """Page numbers outside the pool in the list or the table give no slot."""
    table, free, n_free = pool(np.random.default_rng(2), [3, 16], 16, 4, 3)
    table[0, 0], free[2] = 99, -4
    got = check_plan(dev, [3, 16], [2, 1], free, n_free, table, 3, 16)
    assert list(got[3]) == [-1, -1, -1]


# ---- writes and reads --------------------------------------------------------------


def step_rows(rng, n, n_kv, hd):
    """Rows whose sizes differ between tokens and heads, some exact ties."""
    x = rng.standard_normal((n, n_kv, hd)) * np.exp(rng.normal(0, 0.7, (n, n_kv, 1)))
    x[rng.random((n, n_kv)) < 0.1] *= 1e-3
    return x.astype(np.float32)


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32)


def append_both(dev, cache, table, q_start, kv_len, k, v, ldk=None, ldv=None, shift=0, **bounds):
    """One append on the device and on the host's copy; every byte of the
    cache and of the scales is compared."""
    n, width = k.shape[0], cache.n_kv * cache.hd
    ldk, ldv = ldk or width, ldv or width
    kp, vp = np.full(shift + n * ldk, np.nan, np.float32), np.full(shift + n * ldv, np.nan, np.float32)
    for t in range(n):
        kp[shift + t * ldk:shift + t * ldk + width] = k[t].reshape(-1)
        vp[shift + t * ldv:shift + t * ldv + width] = v[t].reshape(-1)
    with ko.OnDevice(dev, kp=kp, vp=vp) as d:
        c = ko.put_cache(d, cache)
        b = ko.put_batch(d, table, q_start, kv_len, n, **bounds)
        dev.kv_append_dev(c, b, d.ptr("kp") + 4 * shift, ldk, d.ptr("vp") + 4 * shift, ldv)
        dev.synchronize()
        got = {x: d.get(x) for x in ("k", "v", "ks", "vs")}
    cache.append(table, q_start, kv_len, k, v)
    for name in ("k", "v"):
        assert np.array_equal(got[name], getattr(cache, name)), name
        assert np.array_equal(bits(got[name + "s"]), bits(getattr(cache, name + "s"))), name + " scales"


@pytest.mark.parametrize("block,n_kv,hd", [(16, 8, 128), (32, 2, 64), (64, 1, 80), (128, 3, 256), (256, 2, 16), (16, 1, 16),
                                           (64, 2, 112)])
def test_append_steps(dev, block, n_kv, hd):
    """Steps of single tokens and of chunks that start and end anywhere in a
    page, one behind the other on the same cache."""
    rng = np.random.default_rng(block * hd)
    adds = [[block + 3, 1, 0, 2 * block, 5], [1] * 5, [1, 0, 7, 1, 2 * block - 1], [block, block - 1, 1, 1, block + 1]]
    cache, table, _, _ = ko.requests(rng, [sum(a[r] for a in adds) for r in range(5)], [0] * 5, block, n_kv, hd)
    cache.ks[:], cache.vs[:] = np.nan, np.nan  # nothing is written yet
    kv_len = np.zeros(5, np.int32)
    for add in adds:
        kv_len = kv_len + np.array(add, np.int32)
        q_start = np.concatenate([[0], np.cumsum(add)]).astype(np.int32)
        n = int(q_start[-1])
        append_both(dev, cache, table, q_start, kv_len, step_rows(rng, n, n_kv, hd), step_rows(rng, n, n_kv, hd))


def test_append_rows_with_gaps_and_at_odd_addresses(dev):
    rng = np.random.default_rng(8)
    cache, table, q_start, kv_len = ko.requests(rng, [9, 0], [30, 17], 16, 2, 64)
    append_both(dev, cache, table, q_start, kv_len, step_rows(rng, 47, 2, 64), step_rows(rng, 47, 2, 64), ldk=131,
                ldv=128 + 64, shift=1)


def test_append_ties_and_extremes(dev):
    """Values on the border between two codes, zeros, the smallest and largest
    magnitudes, infinities and NaN."""
    rng = np.random.default_rng(9)
    block, hd = 16, 64
    cache, table, _, _ = ko.requests(rng, [0] * 9, [24] * 9, block, 1, hd)
    cache.ks[:], cache.vs[:] = np.nan, np.nan
    k = np.zeros((9 * 8, 1, hd), np.float32)
    rows = k.reshape(9, 8, hd)
    rows[0, :, :] = np.arange(8 * hd).reshape(8, hd) * 0.5 - 127  # scale 1 or so: halves
    rows[0, 0, 0] = 127.0
    rows[1] = 0.0
    rows[2] = rng.standard_normal((8, hd)) * 1e-38
    rows[3] = rng.standard_normal((8, hd)) * np.float32(2.0 ** -100)
    rows[4] = rng.standard_normal((8, hd)) * 1e37
    rows[4, 3, 3] = np.finfo(np.float32).max
    rows[5] = rng.standard_normal((8, hd))
    rows[5, 1, :5] = [np.inf, -np.inf, np.nan, 0.0, -0.0]
    rows[6, 2, 7] = np.inf
    rows[7] = np.nan
    rows[8] = (np.arange(hd) - 32) * 1.5
    q_start = np.arange(0, 73, 8).astype(np.int32)
    for step, factor in enumerate((1.0, 2.0, 1.0)):  # old codes: requantized by two, then kept
        kk = k.copy()
        kk[np.arange(72) // 8 != 4] *= np.float32(factor)
        append_both(dev, cache, table, q_start, np.full(9, 8 * (step + 1), np.int32), kk, kk[::-1].copy())


def test_append_leaves_others_alone(dev):
    """Requests without rows, with impossible numbers, with pages outside the
    pool; rows behind the last token; bounds that are too small."""
    rng = np.random.default_rng(10)
    cache, table, q_start, kv_len = ko.requests(rng, [9, 5, 0, 20], [2, 0, 3, 20], 16, 2, 32)
    k, v = step_rows(rng, 40, 2, 32), step_rows(rng, 40, 2, 32)
    table[3, 2] = cache.n_pages
    append_both(dev, cache, table, q_start, kv_len, k, v)
    before = [x.copy() for x in (cache.k, cache.v, cache.ks, cache.vs)]
    with ko.OnDevice(dev, kp=k, vp=v) as d:
        c = ko.put_cache(d, cache)
        for q0, end in (([5, 4, 4, 4, 4], kv_len),          # q_start falls
                        ([0, 41, 41, 41, 41], kv_len),      # past n_tok
                        ([-3, 2, 2, 2, 2], kv_len),
                        ([0, 3, 3, 3, 3], [2, 5, 3, 40]),   # more new tokens than tokens
                        ([0, 1, 1, 1, 1], [-5, 0, 0, 0]),
                        ([0, 1, 1, 1, 1], [16 * 40, 0, 0, 0]),  # past its table row
                        ([0, 1, 2, 2, 2], [0, 2 ** 31 - 1, 0, 0])):
            b = ko.put_batch(d, table, q0, end, 40, max_q=40)
            dev.kv_append_dev(c, b, d.ptr("kp"), 64, d.ptr("vp"), 64)
        dev.synchronize()
        for name, was in zip(("k", "v", "ks", "vs"), before):
            assert np.array_equal(d.get(name).view(np.uint8), was.view(np.uint8)), name


@pytest.mark.parametrize("block,n_kv,hd,ld", [(16, 8, 128, 1024), (64, 2, 80, 163), (256, 1, 256, 256), (32, 3, 16, 50)])
def test_read(dev, block, n_kv, hd, ld):
    """Any slots in any order, the same one twice, and slots outside the
    cache, whose rows stay as they were."""
    rng = np.random.default_rng(hd + ld)
    cache, table, _, _ = ko.requests(rng, [3 * block], [0], block, n_kv, hd)
    k, v = cache.rows(table[0], 3 * block)
    at = np.concatenate([np.arange(3 * block), rng.integers(0, 3 * block, 37)])
    slots = table[0, at // block].astype(np.int64) * block + at % block
    wrong = rng.random(len(slots)) < 0.1
    slots[wrong] = rng.choice([-1, cache.n_pages * block, 2 ** 62, -2 ** 63, 2 ** 40], wrong.sum())
    marker = np.full(len(slots) * ld + 3, 55.0, np.float32)
    with ko.OnDevice(dev, slots=slots, ko=marker, vo=marker) as d:
        dev.kv_read_dev(ko.put_cache(d, cache), d.ptr("slots"), len(slots), d.ptr("ko") + 12, ld, d.ptr("vo") + 12, ld)
        dev.synchronize()
        for name, x in (("ko", k), ("vo", v)):
            want = np.full((len(slots), ld), 55.0, np.float32)
            want[~wrong, :n_kv * hd] = x.swapaxes(0, 1)[at[~wrong]].reshape(-1, n_kv * hd).astype(np.float32)
            assert np.array_equal(bits(d.get(name)[3:].reshape(len(slots), ld)), bits(want))
