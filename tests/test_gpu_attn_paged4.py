"""Attention over the paged 4-bit KV cache against its definition in 64 bits
(kv_oracle.attention over kv4_oracle.Cache, with its bound of the roundings)."""
import numpy as np
import pytest

import siphon_amd as sa

from . import kv4_oracle as k4
from . import kv_oracle as ko

pytestmark = pytest.mark.gpu


def queries(rng, n, heads, hd, size=1.0):
    return (rng.standard_normal((n, heads, hd)) * size).astype(np.float32)


def run(dev, cache, pages, q_start, kv_len, q, kq, ldq=None, ldo=None, shift=0, bounds=None, **o):
    """The call's rows, and that nothing else of its output was written."""
    n, heads, hd = q.shape
    ldq, ldo = ldq or heads * hd, ldo or heads * hd
    qp = np.full(shift + n * ldq, np.nan, np.float32)
    for t in range(n):
        qp[shift + t * ldq:shift + t * ldq + heads * hd] = q[t].reshape(-1)
    arrays = {name: o.pop(name) for name in ("slopes", "prefix") if o.get(name) is not None}
    with ko.OnDevice(dev, q=qp, out=np.full(shift + n * ldo, 55.0, np.float32), **arrays) as d:
        c = k4.put_cache(d, cache)
        b = ko.put_batch(d, pages, q_start, kv_len, n, **(bounds or {}))
        a = sa.AttnPaged(q=d.ptr("q") + 4 * shift, ldq=ldq, out=d.ptr("out") + 4 * shift, ldo=ldo, n_head=heads, kq_scale=kq,
                         softcap=o.get("cap", 0.0), window=o.get("window", 0), **{x: d.ptr(x) for x in arrays})
        dev.attn_paged4_dev(c, b, a)
        dev.synchronize()
        out = d.get("out")
    rows = out[shift:].reshape(n, ldo)
    assert (out[:shift] == 55.0).all() and (rows[:, heads * hd:] == 55.0).all()
    return rows[:, :heads * hd].reshape(n, heads, hd)


def check(dev, cache, pages, q_start, kv_len, q, kq, **o):
    args = {k: o[k] for k in ("cap", "slopes", "prefix", "window") if k in o}
    want, err, seen = ko.attention(cache, pages, q_start, kv_len, q, kq, **args)
    got = run(dev, cache, pages, q_start, kv_len, q, kq, **o)
    assert (got[~seen] == 55.0).all()  # rows of no request
    off = np.abs(got.astype(np.float64) - want)[seen]
    worst = np.max(off / (err[seen] + 1e-30), initial=0.0)
    assert worst <= 1.0, f"{worst:.3g} times the bound"
    # all roundings together: independent, so their norm is far below the sum that the bound is
    # (an f16 operand alone would be 2e-4)
    assert np.linalg.norm(off) <= 1e-5 * np.linalg.norm(want[seen])
    return got


SHAPES = [(32, 8, 128, 16), (14, 2, 64, 32), (4, 4, 96, 64), (8, 1, 96, 16), (40, 8, 128, 128), (16, 8, 256, 32),
          (3, 3, 32, 256), (32, 1, 64, 16), (10, 2, 160, 64), (6, 2, 192, 16), (24, 1, 32, 128), (5, 1, 224, 16)]


@pytest.mark.parametrize("heads,n_kv,hd,block", SHAPES)
def test_single_tokens(dev, heads, n_kv, hd, block):
    """Lengths from one token, around chunks, pages and splits, to long ones."""
    rng = np.random.default_rng(heads * hd + block)
    lengths = [0, 1, 15, 16, 17, 62, 63, 64, 127, 128, 254, 255, 256, 300, 600, 1000, 2500]
    n = len(lengths)
    cache, pages, q_start, kv_len = k4.requests(rng, lengths, [1] * n, block, n_kv, hd)
    check(dev, cache, pages, q_start, kv_len, queries(rng, n, heads, hd, 2.0), 1 / np.sqrt(hd))


@pytest.mark.parametrize("heads,n_kv,hd,block", SHAPES)
@pytest.mark.parametrize("large", [0, 1])
def test_prompts(dev, option, heads, n_kv, hd, block, large):
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(heads + hd + block)
    lengths, adds = [0, 0, 37, 500, 64, 9, 0], [1, 300, 65, 17, 64, 0, 129]
    cache, pages, q_start, kv_len = k4.requests(rng, lengths, adds, block, n_kv, hd)
    check(dev, cache, pages, q_start, kv_len, queries(rng, sum(adds), heads, hd, 2.0), 1 / np.sqrt(hd))


CHANGES = {
    "cap": dict(cap=5.0), "wide_cap": dict(cap=50.0), "window_1": dict(window=1), "window_63": dict(window=63),
    "window_64": dict(window=64), "window_100": dict(window=100), "window_past": dict(window=10 ** 12),
    "slopes": dict(slopes=True), "prefix": dict(prefix=True), "all": dict(cap=20.0, window=70, slopes=True, prefix=True),
    "prefix_window": dict(window=17, prefix=True), "slopes_window": dict(slopes=True, window=200),
}


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("heads,n_kv,hd,block", [(8, 2, 128, 16), (5, 1, 64, 64), (4, 4, 96, 128), (2, 1, 256, 32)])
@pytest.mark.parametrize("steps,large", [("single", 0), ("prompt", 0), ("prompt", 1)])
def test_masks_and_scores(dev, option, change, heads, n_kv, hd, block, steps, large):
    if hd > 128 and large:
        pytest.skip("heads of more than 128 have no large row blocks")
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(len(change) * 100 + hd)
    lengths = [0, 1, 63, 64, 200, 450, 1300] if steps == "single" else [0, 40, 0, 333, 100]
    adds = [1] * 7 if steps == "single" else [70, 129, 1, 33, 200]
    cache, pages, q_start, kv_len = k4.requests(rng, lengths, adds, block, n_kv, hd)
    o = dict(CHANGES[change])
    if o.pop("slopes", False):
        o["slopes"] = (2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)).astype(np.float32)
    if o.pop("prefix", False):
        # none, some, a chunk, past the row, past the request, negative
        o["prefix"] = np.array([0, 20, 64, 70, 10 ** 6, -5, 400][:len(adds)], np.int32)
    check(dev, cache, pages, q_start, kv_len, queries(rng, sum(adds), heads, hd, 2.0), 1 / np.sqrt(hd), **o)


@pytest.mark.parametrize("kq", [-0.25, 0.0, 1e-30, 3.0])
@pytest.mark.parametrize("cap", [0.0, 10.0])
@pytest.mark.parametrize("large", [0, 1])
def test_score_factors(dev, option, kq, cap, large):
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(17)
    cache, pages, q_start, kv_len = k4.requests(rng, [400, 0, 90], [1, 60, 3], 32, 2, 64)
    check(dev, cache, pages, q_start, kv_len, queries(rng, 64, 4, 64), kq, cap=cap)
    check(dev, cache, pages, [0, 1, 1, 4], kv_len, queries(rng, 4, 4, 64), kq, cap=cap)


@pytest.mark.parametrize("splits", [1, 3, 64])
@pytest.mark.parametrize("row_waves", [1, 4])
@pytest.mark.parametrize("heads,n_kv,hd", [(8, 2, 128), (3, 3, 64), (6, 2, 256), (20, 1, 96), (4, 2, 160)])
def test_pieces(dev, option, heads, n_kv, hd, row_waves, splits):
    """Pieces of any number, joined by the last workgroup to arrive."""
    option("ATTNP_ROW_WAVES", row_waves)
    option("ATTNP_SPLITS", splits)
    rng = np.random.default_rng(row_waves * splits + hd)
    cache, pages, q_start, kv_len = k4.requests(rng, [3000, 1, 64, 700, 0, 129], [1, 1, 2, 1, 3, 0], 32, n_kv, hd)
    check(dev, cache, pages, q_start, kv_len, queries(rng, 8, heads, hd, 2.0), 0.09)


@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("hd", [128, 64, 96])
def test_splits_of_large_blocks(dev, option, hd, splits):
    option("ATTNP_LARGE", 1)
    option("ATTNP_SPLITS", splits)
    rng = np.random.default_rng(splits)
    cache, pages, q_start, kv_len = k4.requests(rng, [900, 0, 3000, 5], [150, 100, 129, 40], 64, 2, hd)
    check(dev, cache, pages, q_start, kv_len, queries(rng, 419, 4, hd, 2.0), 0.09)


@pytest.mark.parametrize("hd", [128, 64])
def test_prompts_beside_single_tokens(dev, option, hd):
    option("ATTNP_LARGE", 1)
    rng = np.random.default_rng(hd)
    lengths, adds = [1500, 0, 333, 70, 40, 2000, 9], [1, 200, 1, 16, 17, 90, 5]
    cache, pages, q_start, kv_len = k4.requests(rng, lengths, adds, 32, 2, hd)
    check(dev, cache, pages, q_start, kv_len, queries(rng, sum(adds), 8, hd, 2.0), 0.09)


@pytest.mark.parametrize("n_req", [64, 65, 256, 257])
@pytest.mark.parametrize("large", [0, 1])
def test_many_requests(dev, option, n_req, large):
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(n_req)
    lengths = [int(x) for x in np.exp(rng.uniform(0, 6.5, n_req))]
    adds = [int(x) for x in rng.choice([0, 1, 1, 1, 4, 40], n_req)]
    cache, pages, q_start, kv_len = k4.requests(rng, lengths, adds, 16, 1, 32)
    check(dev, cache, pages, q_start, kv_len, queries(rng, sum(adds), 3, 32, 2.0), 0.2)


def test_long_context(dev):
    """100 000 tokens in one request beside a short one, with a peak that comes late."""
    rng = np.random.default_rng(5)
    cache, pages, q_start, kv_len = k4.requests(rng, [99_999, 70], [1, 1], 64, 2, 64)
    q = queries(rng, 2, 4, 64, 1.0)
    page = pages[0, 1500]
    cache.k[page, :, 3], cache.ksub[page, :, :, 3] = np.where(q[0, ::2] > 0, 7, -7), 127
    cache.ks[page, :, 3] = 0x3b80  # 2^-8
    check(dev, cache, pages, q_start, kv_len, q, 0.5)


def test_offsets_past_32_bits(dev):
    """Pages whose codes, and whose subs, lie more than 2^32 bytes into their arrays."""
    rng = np.random.default_rng(6)
    block, n_kv, hd = 256, 8, 256
    small, pages, q_start, kv_len = k4.requests(rng, [1000, 300], [1, 2], block, n_kv, hd)
    sizes = {name: a[0].nbytes for name, a in small.arrays().items()}
    n_pages = (1 << 32) // sizes["ksub"] + 40
    held = [int(p) for r, n in enumerate(kv_len) for p in pages[r, :ko.blocks_of(int(n), block)]]
    far = {p: n_pages - 1 - 3 * i for i, p in enumerate(held)}
    assert min(far.values()) * sizes["ksub"] > 1 << 32
    moved = pages.copy()
    for r, n in enumerate(kv_len):
        for b in range(ko.blocks_of(int(n), block)):
            moved[r, b] = far[int(pages[r, b])]
    big = {}
    try:
        for name, size in sizes.items():
            big[name] = dev.alloc(n_pages * size)
        for p, f in far.items():
            for name, a in small.arrays().items():
                row = np.ascontiguousarray(a[p])
                dev._check(dev.L.sihip_memcpy_htod(dev.ctx, big[name].ptr + f * sizes[name], row.ctypes.data, row.nbytes))
        q = queries(rng, 3, 16, hd, 2.0)
        want, err, _ = ko.attention(small, pages, q_start, kv_len, q, 0.07)
        k, v = rng.standard_normal((2, 3, n_kv, hd)).astype(np.float32)
        w = n_kv * hd
        at = np.array([0, 1000, 299])
        slots = np.array([moved[0, 0] * block, moved[0, 3] * block + 1000 % block, moved[1, 1] * block + 299 % block], np.int64)
        with ko.OnDevice(dev, q=q, out=np.zeros_like(q), kn=k, vn=v, slots=slots, ro=np.zeros((2, 3, n_kv, hd), np.float32)) as d:
            c = sa.Kv4Cache(k=big["k"].ptr, v=big["v"].ptr, k_sub=big["ksub"].ptr, v_sub=big["vsub"].ptr, k_scale=big["ks"].ptr,
                            v_scale=big["vb"].ptr, n_pages=n_pages, n_head_kv=n_kv, head_dim=hd, block=block)
            b = ko.put_batch(d, moved, q_start, kv_len, 3)
            dev.attn_paged4_dev(c, b, sa.AttnPaged(q=d.ptr("q"), ldq=16 * hd, out=d.ptr("out"), ldo=16 * hd, n_head=16, kq_scale=0.07))
            dev.synchronize()
            assert (np.abs(d.get("out") - want) <= err + 1e-30).all()
            # and a write there: the step's rows again, read back in values
            dev.kv4_append_dev(c, b, sa.KvRows(k=d.ptr("kn"), ldk=w, v=d.ptr("vn"), ldv=w))
            dev.kv4_read_dev(c, d.ptr("slots"), 3, d.ptr("ro"), w, d.ptr("ro") + 12 * w, w)
            dev.synchronize()
            small.append(pages, q_start, kv_len, k, v)
            (k0, v0), (k1, v1) = (small.rows(pages[r], int(kv_len[r])) for r in (0, 1))
            want = [np.stack([a[:, 0], a[:, 1000], b[:, 299]]) for a, b in ((k0, k1), (v0, v1))]
            assert np.array_equal(d.get("ro"), np.stack(want).astype(np.float32))
    finally:
        for b in big.values():
            b.free()


def test_rows_at_odd_addresses_with_gaps(dev):
    rng = np.random.default_rng(11)
    cache, pages, q_start, kv_len = k4.requests(rng, [90, 7], [1, 40], 16, 2, 96)
    check(dev, cache, pages, q_start, kv_len, queries(rng, 41, 6, 96, 2.0), 0.1, ldq=6 * 96 + 7, ldo=6 * 96 + 1, shift=3)


@pytest.mark.parametrize("large", [0, 1])
def test_rows_that_see_nothing(dev, option, large):
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(12)
    cache, pages, q_start, kv_len = k4.requests(rng, [40, 20, 30, 9], [2, 2, 2, 2], 16, 2, 64)
    q = queries(rng, 9, 4, 64)
    whole = check(dev, cache, pages, q_start, kv_len, q[:8], 0.2)
    torn = pages.copy()
    torn[0, :3], torn[1, 0] = [-1, cache.n_pages, 2 ** 31 - 1], -7
    got = run(dev, cache, torn, q_start, kv_len, q[:8], 0.2)
    assert not got[0:2].any()
    # request 1 sees positions 16 .. only: as a window of its rows would
    for i, n in ((2, 5), (3, 6)):
        want, err, _ = ko.attention(cache, pages, np.array([0, 0, 1, 1, 1]), np.array([0, 16 + n, 0, 0]), q[i:i + 1], 0.2, window=n)
        assert (np.abs(got[i] - want[0]) <= err[0]).all()
    assert np.array_equal(got[4:], whole[4:])
    for q0, end in (([0, 3, 3, 3, 3], [2, 0, 0, 0]), ([0, 10, 10, 10, 10], [42, 0, 0, 0]), ([-1, 1, 1, 1, 1], [42, 0, 0, 0]),
                    ([2, 0, 0, 0, 0], [42, 22, 0, 0]), ([0, 0, 0, 0, 0], [42, 22, 32, 11]), ([0, 1, 1, 1, 1], [-1, 0, 0, 0])):
        got = run(dev, cache, pages, np.array(q0), np.array(end), q, 0.2, bounds=dict(max_q=9, max_kv=64))
        assert (got == 55.0).all(), (q0, end)


def test_bounds_cut(dev):
    rng = np.random.default_rng(13)
    cache, pages, q_start, kv_len = k4.requests(rng, [200, 10], [1, 20], 16, 1, 64)
    q = queries(rng, 21, 2, 64)
    got = run(dev, cache, pages, q_start, kv_len, q, 0.2, bounds=dict(max_q=8, max_kv=100))
    assert (got[9:] == 55.0).all()
    want, err, _ = ko.attention(cache, pages, np.array([0, 1, 1]), np.array([100, 0]), q[:1], 0.2)
    assert (np.abs(got[0] - want[0]) <= err[0]).all()
    want, err, _ = ko.attention(cache, pages, q_start, kv_len, q, 0.2)
    assert (np.abs(got[1:9] - want[1:9]) <= err[1:9]).all()


@pytest.mark.parametrize("steps,large", [("single", 0), ("prompt", 0), ("prompt", 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_garbage_that_no_row_sees(dev, option, steps, large, hd):
    """NaN and infinite scales behind the window and past the length; large,
    tiny and zero scales of what is seen."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(14)
    lengths, adds = ([700, 300], [1, 1]) if steps == "single" else ([400, 0], [200, 150])
    cache, pages, q_start, kv_len = k4.requests(rng, lengths, adds, 16, 2, hd)
    q = queries(rng, sum(adds), 4, hd)
    window = 100
    for r in range(2):
        for b in range(max(0, lengths[r] - window) // 16):
            cache.ks[pages[r, b]], cache.vb[pages[r, b]] = 0x7fc0, [[0x7f80], [0xff80]]
    bf = lambda x: int(np.float32(x).view(np.uint32)) >> 16
    last = [int(pages[r, kv_len[r] // 16 - 1]) for r in range(2)]
    cache.vb[last[0], :, :9], cache.ks[last[0], 0, :9], cache.ks[last[0], 1, 3:] = bf(1e28), 0, bf(1e-33)
    cache.vb[last[1], 0, 2:], cache.vb[last[1], 1], cache.ks[last[1], 1, ::2] = 0, bf(1e-33), 0
    got = run(dev, cache, pages, q_start, kv_len, q, 0.2, window=window)
    assert np.isfinite(got).all()
    want, err, _ = ko.attention(cache, pages, q_start, kv_len, q, 0.2, window=window)
    assert (np.abs(got - want) <= err + 1e-30).all()


def test_large_values_that_a_row_hardly_sees(dev):
    """A value scale of 2^40 times the others', on a key of no weight, takes no bits from them
    (what its key weighs is e^-60)."""
    rng = np.random.default_rng(18)
    cache, pages, q_start, kv_len = k4.requests(rng, [200], [1], 16, 1, 64)
    q = np.ones((1, 1, 64), np.float32)
    page = int(pages[0, 3])
    cache.k[page, 0, 5], cache.ksub[page, 0, :, 5], cache.ks[page, 0, 5] = -8, 100, 0x3f80  # score -64 * 800 * kq
    cache.vb[page, 0, 5] += 40 << 7
    kq = 70 / (64 * 800)
    want, err, _ = ko.attention(cache, pages, q_start, kv_len, q, kq)
    got = run(dev, cache, pages, q_start, kv_len, q, kq)
    # the bound of kv_oracle counts the largest scale; here: what is held to 2^-34 of the largest product
    k, v = cache.rows(pages[0], 201)
    s = kq * k[0].sum(1)
    w = np.exp(s - s.max())
    product = (w[:, None] * np.abs(v[0])).max()
    assert (np.abs(got - want) <= 2.0 ** -18 * (w @ np.abs(v[0])) / w.sum() + 201 * 2.0 ** -34 * 128 * product).all()


def test_sizes_of_queries(dev):
    rng = np.random.default_rng(15)
    cache, pages, q_start, kv_len = k4.requests(rng, [300] * 6, [1] * 6, 32, 1, 64)
    q = queries(rng, 6, 2, 64)
    q[0], q[1], q[2] = 0.0, q[1] * np.float32(1e-38), q[2] * 40
    q[3] *= np.exp(rng.normal(0, 4, 64)).astype(np.float32)
    q[4, 1, 5] = np.nan
    got = run(dev, cache, pages, q_start, kv_len, q, 0.125)
    want, err, _ = ko.attention(cache, pages, q_start, kv_len, np.nan_to_num(q), 0.125)
    assert np.isnan(got[4, 1]).all()
    got[4, 1], want[4, 1] = 0, 0
    assert (np.abs(got - want) <= err + 1e-30).all()


@pytest.mark.parametrize("row_waves", [1, 4])
def test_same_bits_every_time(dev, option, row_waves):
    option("ATTNP_ROW_WAVES", row_waves)
    rng = np.random.default_rng(16)
    cache, pages, q_start, kv_len = k4.requests(rng, [5000, 3000, 64, 900], [1, 1, 1, 1], 32, 2, 128)
    q = queries(rng, 4, 8, 128)
    first = run(dev, cache, pages, q_start, kv_len, q, 0.09)
    for _ in range(4):
        assert np.array_equal(run(dev, cache, pages, q_start, kv_len, q, 0.09).view(np.uint32), first.view(np.uint32))
