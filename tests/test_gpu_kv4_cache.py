"""Writes into the paged caches with the rotation on the way, and the 4-bit
cache's writes and reads, against their restatements in numpy (kv4_oracle, kv_oracle):
exact, bit for bit."""
import numpy as np
import pytest

import siphon_amd as sa

from . import kv4_oracle as k4
from . import kv_oracle as ko

pytestmark = pytest.mark.gpu


def same(a, b):
    """Whether two arrays are equal bit for bit."""
    a, b = (np.ascontiguousarray(x) for x in (a, b))
    return a.shape == b.shape and bool((a.view(np.uint8) == b.view(np.uint8)).all())


def step_rows(rng, n, heads, hd):
    x = rng.standard_normal((n, heads, hd)) * np.exp(rng.normal(0, 0.7, (n, heads, 1)))
    x[rng.random((n, heads)) < 0.1] *= 1e-3
    x[rng.random((n, heads)) < 0.05] = 0
    return x.astype(np.float32)


def strided(x, ld, shift):
    """Rows at a distance of ld, from `shift` values on; the rest marked."""
    n = x.shape[0]
    out = np.full(shift + n * ld, 55.0, np.float32)
    rows = out[shift:].reshape(n, ld)
    rows[:, :x[0].size] = x.reshape(n, -1)
    return out


class Append:
    """One append of a batch, and everything it may and may not write."""

    def __init__(self, dev, cache, pages, q_start, kv_len, k, v, q=None, rope=None, neighbours=False, gap=4, shift=4, in_place=False,
                 max_q=None, max_kv=None, stream=None, n_tok=None):
        n, width = len(k), cache.n_kv * cache.hd
        heads = 0 if q is None else q.shape[1]
        ld, ldq = width + gap, heads * cache.hd + gap
        four = isinstance(cache, k4.Cache)
        arrays = dict(nk=strided(k, ld, shift), nv=strided(v, ld, shift))
        if rope is not None:
            arrays["rope"] = rope
        if q is not None:
            arrays["q"] = strided(q, ldq, shift)
            arrays["qo"] = np.full_like(arrays["q"], 77.0)
        with ko.OnDevice(dev, **arrays) as d:
            c = (k4 if four else ko).put_cache(d, cache)
            b = ko.put_batch(d, pages, q_start, kv_len, n_tok or n, max_q=max_q, max_kv=max_kv)
            rows = sa.KvRows(k=d.ptr("nk") + 4 * shift, v=d.ptr("nv") + 4 * shift, ldk=ld, ldv=ld)
            if q is not None:
                rows.q, rows.ldq, rows.ldq_out, rows.n_head = d.ptr("q") + 4 * shift, ldq, ldq, heads
                rows.q_out = rows.q if in_place else d.ptr("qo") + 4 * shift
            if rope is not None:
                rows.rope, rows.rope_len, rows.rope_dim, rows.rope_neighbours = d.ptr("rope"), len(rope), 2 * rope.shape[1], neighbours
            (dev.kv4_append_dev if four else dev.kv_append_rope_dev)(c, b, rows, stream)
            dev.synchronize()
            names = ("k", "v", "ksub", "vsub", "ks", "vb") if four else ("k", "v", "ks", "vs")
            self.cache = {name: d.get(name) for name in names}
            assert same(d.get("nk"), arrays["nk"]) and same(d.get("nv"), arrays["nv"])
            if q is not None:
                got = d.get("q" if in_place else "qo")
                assert (got[:shift] == (55 if in_place else 77)).all()
                got = got[shift:].reshape(n, ldq)
                assert (got[:, heads * cache.hd:] == (55 if in_place else 77)).all()
                self.q = got[:, :heads * cache.hd].reshape(q.shape)


def positions(q_start, kv_len, n):
    pos = np.zeros(n, np.int64)
    for r, end in enumerate(kv_len):
        q0, q1 = q_start[r], q_start[r + 1]
        pos[q0:q1] = np.arange(end - (q1 - q0), end)
    return pos


def check(got, cache):
    want = cache.arrays() if isinstance(cache, k4.Cache) else {n: getattr(cache, n) for n in ("k", "v", "ks", "vs")}
    for name, a in want.items():
        assert same(got.cache[name], a), name


def make(bits_, rng, lengths, adds, block, n_kv, hd):
    return (k4.requests if bits_ == 4 else ko.requests)(rng, lengths, adds, block, n_kv, hd)


@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("n_kv,hd", [(2, 128), (1, 64), (3, 32), (2, 96), (1, 160), (1, 256), (1, 192), (1, 224)])
def test_append4(dev, block, n_kv, hd):
    """Tokens that begin and end anywhere in words, chunks and pages; the rest
    of every word stays."""
    rng = np.random.default_rng(block + hd)
    lengths = [0, 1, 5, block - 1, block, 2 * block + 7, 3, 70, 9]
    adds = [1, 1, 2, 1, block, block + 3, 2 * block + 60, 130, 0]
    cache, pages, q_start, kv_len = k4.requests(rng, lengths, adds, block, n_kv, hd)
    k, v = (step_rows(rng, sum(adds), n_kv, hd) for _ in range(2))
    got = Append(dev, cache, pages, q_start, kv_len, k, v)
    cache.append(pages, q_start, kv_len, k, v)
    check(got, cache)


ROPES = [(128, 128), (64, 64), (96, 48), (64, 38), (32, 2), (256, 256), (96, 94), (160, 72)]


@pytest.mark.parametrize("bits_", [4, 8])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("hd,dim", ROPES)
@pytest.mark.parametrize("aligned", [True, False])
def test_rotated_append(dev, bits_, neighbours, hd, dim, aligned):
    """Keys and queries turned by the positions, values as they are; rows at any
    address; every query head of a KV head; rotations of part of a head."""
    rng = np.random.default_rng(hd + dim + bits_)
    lengths, adds = [0, 40, 15, 333, 3], [50, 1, 3, 1, 0]
    cache, pages, q_start, kv_len = make(bits_, rng, lengths, adds, 16, 2, hd)
    n = sum(adds)
    k, v, q = (step_rows(rng, n, h, hd) for h in (2, 2, 6))
    rope = k4.table(int(kv_len.max()) + 3, dim)
    got = Append(dev, cache, pages, q_start, kv_len, k, v, q, rope, neighbours, *((4, 4) if aligned else (3, 1)), in_place=not aligned)
    pos = positions(q_start, kv_len, n)
    cache.append(pages, q_start, kv_len, k4.rotate(k, pos, rope, neighbours), v)
    check(got, cache)
    assert same(got.q, k4.rotate(q, pos, rope, neighbours))


@pytest.mark.parametrize("bits_", [4, 8])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("hd,dim", ROPES)
@pytest.mark.parametrize("in_place", [False, True])
def test_rotated_queries_of_large_steps(dev, bits_, neighbours, hd, dim, in_place):
    """A step of so many rows, as far as the host's bound says, that queries are written past the caches."""
    rng = np.random.default_rng(hd + dim + bits_)
    cache, pages, q_start, kv_len = make(bits_, rng, [0, 40, 15], [50, 1, 33], 16, 2, hd)
    k, v, q = (step_rows(rng, 84, h, hd) for h in (2, 2, 6))
    rope = k4.table(int(kv_len.max()), dim)
    got = Append(dev, cache, pages, q_start, kv_len, k, v, q, rope, neighbours, in_place=in_place, max_q=60,
                 n_tok=(64 << 20) // (4 * 6 * hd) + 1)
    pos = positions(q_start, kv_len, 84)
    cache.append(pages, q_start, kv_len, k4.rotate(k, pos, rope, neighbours), v)
    check(got, cache)
    assert same(got.q, k4.rotate(q, pos, rope, neighbours))


@pytest.mark.parametrize("block,hd,n_kv", [(256, 256, 1), (128, 256, 2), (64, 128, 2), (32, 80, 2), (256, 16, 3), (64, 48, 1)])
def test_rotated_append8_of_any_page(dev, block, hd, n_kv):
    """Every number of threads that a page takes."""
    rng = np.random.default_rng(block + hd)
    cache, pages, q_start, kv_len = ko.requests(rng, [0, block - 1, 9], [2 * block + 5, 2, 1], block, n_kv, hd)
    n = int(q_start[-1])
    k, v, q = (step_rows(rng, n, h, hd) for h in (n_kv, n_kv, 4 * n_kv))
    rope = k4.table(int(kv_len.max()), hd)
    got = Append(dev, cache, pages, q_start, kv_len, k, v, q, rope)
    pos = positions(q_start, kv_len, n)
    cache.append(pages, q_start, kv_len, k4.rotate(k, pos, rope, False), v)
    check(got, cache)
    assert same(got.q, k4.rotate(q, pos, rope, False))


@pytest.mark.parametrize("bits_", [4, 8])
def test_far_positions(dev, bits_):
    """A table row is its own position's, however far; the last row of the table is the last position."""
    rng = np.random.default_rng(3)
    cache, pages, q_start, kv_len = make(bits_, rng, [99_990], [10], 64, 1, 64)
    k, v, q = (step_rows(rng, 10, h, 64) for h in (1, 1, 4))
    rope = k4.table(100_000, 64)
    got = Append(dev, cache, pages, q_start, kv_len, k, v, q, rope)
    pos = positions(q_start, kv_len, 10)
    cache.append(pages, q_start, kv_len, k4.rotate(k, pos, rope, False), v)
    check(got, cache)
    assert same(got.q, k4.rotate(q, pos, rope, False))


@pytest.mark.parametrize("bits_", [4, 8])
def test_keys_alone(dev, bits_):
    rng = np.random.default_rng(4)
    cache, pages, q_start, kv_len = make(bits_, rng, [20, 3], [2, 30], 16, 2, 64)
    k, v = (step_rows(rng, 32, 2, 64) for _ in range(2))
    rope = k4.table(64, 64)
    got = Append(dev, cache, pages, q_start, kv_len, k, v, None, rope, True)
    cache.append(pages, q_start, kv_len, k4.rotate(k, positions(q_start, kv_len, 32), rope, True), v)
    check(got, cache)


def test_values_at_the_ends4(dev):
    """Zeros, ties between steps, infinities, NaN, the smallest and the largest numbers."""
    rng = np.random.default_rng(5)
    cache, pages, q_start, kv_len = k4.requests(rng, [3], [40], 16, 2, 64)
    k, v = (step_rows(rng, 40, 2, 64) for _ in range(2))
    for x in (k, v):
        x[0], x[1, 0, :4] = 0, [np.inf, -np.inf, np.nan, 2]
        x[2] = (rng.integers(-16, 16, (2, 64)) / 2).astype(np.float32)  # ties between steps
        x[2, :, ::32] = -8 * 127 / 127
        x[3], x[4] = x[3] * np.float32(1e-32), x[4] * np.float32(1e-38)
        x[5, 0, 0], x[6] = 3e38, x[6] * np.float32(1e35)
        x[7], x[8, 0], x[8, 1] = np.nan, np.inf, -np.inf
        x[9, 0, 32:] *= np.float32(1e-6)  # a group far smaller than the other
        x[10, 1, :2] = [1.5, -1.5]
    got = Append(dev, cache, pages, q_start, kv_len, k, v)
    cache.append(pages, q_start, kv_len, k, v)
    check(got, cache)


@pytest.mark.parametrize("bits_", [4, 8])
def test_rows_that_are_not_written(dev, bits_):
    """Tokens past max_q, from max_kv on, behind the last, and of requests whose
    numbers are impossible: no keys, no values, no queries. A page outside the cache
    loses its keys and values and not its queries."""
    rng = np.random.default_rng(6)
    cache, pages, q_start, kv_len = make(bits_, rng, [10, 40, 0, 7], [30, 5, 9, 1], 16, 2, 64)
    n = int(q_start[-1]) + 3
    k, v, q = (step_rows(rng, n, h, 64) for h in (2, 2, 4))
    pages[0, 1], pages[2, 0] = -3, cache.n_pages
    rope = k4.table(44, 64)
    if bits_ == 4:
        got = Append(dev, cache, pages, q_start, kv_len, k, v, q, rope, max_q=25, max_kv=43)
        pos = np.clip(positions(q_start, kv_len, n), 0, 43)
        cache.append(pages, q_start, kv_len, k4.rotate(k, pos, rope, False), v, max_q=25, max_kv=43)
        check(got, cache)
    else:
        got = Append(dev, cache, pages, q_start, kv_len, k, v, q, rope, max_q=25, max_kv=43)
        pos = np.clip(positions(q_start, kv_len, n), 0, 43)
    want = k4.rotate(q, pos, rope, False)
    want[25:30], want[33:35], want[45:] = 77, 77, 77
    assert same(got.q, want)
    for q0, end in (([0, 60, 60, 60, 60], [70, 0, 0, 0]), ([-1, 1, 1, 1, 1], [42, 0, 0, 0]), ([2, 0, 0, 0, 0], [42, 22, 0, 0]),
                    ([0, 3, 3, 3, 3], [2, 0, 0, 0]), ([0, 1, 1, 1, 1], [-1, 0, 0, 0])):
        got = Append(dev, cache, pages, np.array(q0), np.array(end), k, v, q, rope, max_q=25, max_kv=43)
        check(got, cache) if bits_ == 4 else None
        assert (got.q == 77).all()


# ---- reads ------------------------------------------------------------------------


def read(dev, cache, slots, wide):
    n, width = len(slots), cache.n_kv * cache.hd
    ld, shift = (width + 4, 4) if wide else (width + 1, 1)
    marker = np.full(n * ld + shift, 55.0, np.float32)
    with ko.OnDevice(dev, slots=np.asarray(slots, np.int64), ro=marker, vo=marker) as d:
        dev.kv4_read_dev(k4.put_cache(d, cache), d.ptr("slots"), n, d.ptr("ro") + 4 * shift, ld, d.ptr("vo") + 4 * shift, ld)
        dev.synchronize()
        out = []
        for name in ("ro", "vo"):
            got = d.get(name)
            rows = got[shift:].reshape(n, ld)
            assert (got[:shift] == 55).all() and (rows[:, width:] == 55).all()
            out.append(rows[:, :width].reshape(n, cache.n_kv, cache.hd))
    return out


@pytest.mark.parametrize("start", [0, 1, 7, 8, 15, 16, 41])
@pytest.mark.parametrize("block,n_kv,hd,wide", [(16, 2, 64, True), (32, 1, 32, True), (64, 2, 96, False), (128, 1, 256, False),
                                                (32, 16, 64, True), (256, 1, 160, True)])
def test_read_runs(dev, block, n_kv, hd, wide, start):
    rng = np.random.default_rng(block + hd + start)
    n = 2100 if n_kv == 16 else 205
    cache, pages, _, _ = k4.requests(rng, [start + n], [0], block, n_kv, hd)
    at = np.arange(start, start + n)
    got = read(dev, cache, pages[0, at // block].astype(np.int64) * block + at % block, wide)
    for a, b in zip(got, cache.rows(pages[0], start + n)):
        assert same(a, b.swapaxes(0, 1)[start:].astype(np.float32))


@pytest.mark.parametrize("n", [1, 2, 17, 100])
def test_read_any_slots(dev, n):
    """Slots in any order, the same one twice, and slots that are none."""
    rng = np.random.default_rng(n)
    cache, pages, _, _ = k4.requests(rng, [300], [0], 32, 2, 64)
    at = rng.integers(0, 300, n)
    slots = pages[0, at // 32].astype(np.int64) * 32 + at % 32
    none = rng.random(n) < 0.2
    slots[none] = rng.choice([-1, cache.n_pages * 32, 2 ** 62, -2 ** 63], none.sum())
    for a, b in zip(read(dev, cache, slots, True), cache.rows(pages[0], 300)):
        want = b.swapaxes(0, 1)[at].astype(np.float32)
        want[none] = 55
        assert same(a, want)
