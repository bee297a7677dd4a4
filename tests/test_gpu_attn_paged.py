"""Attention over the paged 8-bit KV cache against its definition in 64 bits
(kv_oracle.attention, which also counts the roundings that a result may
differ by)."""
import numpy as np
import pytest

import siphon_amd as sa

from . import kv_oracle as ko

pytestmark = pytest.mark.gpu


def queries(rng, n, heads, hd, size=1.0):
    return (rng.standard_normal((n, heads, hd)) * size).astype(np.float32)


def run(dev, cache, table, q_start, kv_len, q, kq, stream=None, ldq=None, ldo=None, shift=0, bounds=None, **o):
    """The call's rows, and that nothing else of its output was written."""
    n, heads, hd = q.shape
    ldq, ldo = ldq or heads * hd, ldo or heads * hd
    qp = np.full(shift + n * ldq, np.nan, np.float32)
    for t in range(n):
        qp[shift + t * ldq:shift + t * ldq + heads * hd] = q[t].reshape(-1)
    arrays = {name: o.pop(name) for name in ("slopes", "prefix") if o.get(name) is not None}
    with ko.OnDevice(dev, q=qp, out=np.full(shift + n * ldo, 55.0, np.float32), **arrays) as d:
        c = ko.put_cache(d, cache)
        b = ko.put_batch(d, table, q_start, kv_len, n, **(bounds or {}))
        a = sa.AttnPaged(q=d.ptr("q") + 4 * shift, ldq=ldq, out=d.ptr("out") + 4 * shift, ldo=ldo, n_head=heads, kq_scale=kq,
                         softcap=o.get("cap", 0.0), window=o.get("window", 0), **{x: d.ptr(x) for x in arrays})
        dev.attn_paged_dev(c, b, a, stream)
        dev.synchronize()
        out = d.get("out")
    rows = out[shift:].reshape(n, ldo)
    assert (out[:shift] == 55.0).all() and (rows[:, heads * hd:] == 55.0).all()
    return rows[:, :heads * hd].reshape(n, heads, hd)


def check(dev, cache, table, q_start, kv_len, q, kq, **o):
    args = {k: o[k] for k in ("cap", "slopes", "prefix", "window") if k in o}
    want, err, seen = ko.attention(cache, table, q_start, kv_len, q, kq, **args)
    got = run(dev, cache, table, q_start, kv_len, q, kq, **o)
    assert (got[~seen] == 55.0).all()  # rows of no request
    off = np.abs(got.astype(np.float64) - want)[seen]
    worst = np.max(off / (err[seen] + 1e-30), initial=0.0)
    assert worst <= 1.0, f"{worst:.3g} times the bound"
    # all roundings together: they are independent, so their norm is far below
    # the sum that the bound is (1e-5: an f16 operand alone would be 2e-4)
    assert np.linalg.norm(off) <= 1e-5 * np.linalg.norm(want[seen])
    return got


SHAPES = [(32, 8, 128, 16), (14, 2, 64, 32), (4, 4, 80, 64), (8, 1, 96, 16), (40, 8, 128, 128), (16, 8, 256, 32),
          (3, 3, 16, 256), (32, 1, 64, 16), (10, 2, 112, 64), (6, 2, 192, 16), (24, 1, 48, 128), (5, 1, 240, 16)]


@pytest.mark.parametrize("heads,n_kv,hd,block", SHAPES)
def test_single_tokens(dev, heads, n_kv, hd, block):
    """Lengths from one token, around chunks, pages and splits, to long ones."""
    rng = np.random.default_rng(heads * hd + block)
    lengths = [0, 1, 15, 16, 17, 62, 63, 64, 127, 128, 254, 255, 256, 300, 600, 1000, 2500]
    n = len(lengths)
    cache, table, q_start, kv_len = ko.requests(rng, lengths, [1] * n, block, n_kv, hd)
    check(dev, cache, table, q_start, kv_len, queries(rng, n, heads, hd, 2.0), 1 / np.sqrt(hd))


@pytest.mark.parametrize("heads,n_kv,hd,block", SHAPES)
@pytest.mark.parametrize("large", [0, 1])
def test_prompts(dev, option, heads, n_kv, hd, block, large):
    """Requests of 0 to 300 new tokens, behind nothing or behind a context, in
    blocks of 16, 128 and 256 rows (the large ones: heads up to 128, and the
    requests of more than 64 rows)."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(heads + hd + block)
    lengths, adds = [0, 0, 37, 500, 64, 9, 0], [1, 300, 65, 17, 64, 0, 129]
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, block, n_kv, hd)
    check(dev, cache, table, q_start, kv_len, queries(rng, sum(adds), heads, hd, 2.0), 1 / np.sqrt(hd))


CHANGES = {
    "cap": dict(cap=5.0), "wide_cap": dict(cap=50.0), "window_1": dict(window=1), "window_63": dict(window=63),
    "window_64": dict(window=64), "window_100": dict(window=100), "window_past": dict(window=10 ** 12),
    "slopes": dict(slopes=True), "prefix": dict(prefix=True), "all": dict(cap=20.0, window=70, slopes=True, prefix=True),
    "prefix_window": dict(window=17, prefix=True), "slopes_window": dict(slopes=True, window=200),
}


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("heads,n_kv,hd,block", [(8, 2, 128, 16), (5, 1, 64, 64), (4, 4, 80, 128), (2, 1, 256, 32)])
@pytest.mark.parametrize("steps,large", [("single", 0), ("prompt", 0), ("prompt", 1)])
def test_masks_and_scores(dev, option, change, heads, n_kv, hd, block, steps, large):
    if hd > 128 and large:
        pytest.skip("heads of more than 128 have no large row blocks")
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(len(change) * 100 + hd)
    lengths = [0, 1, 63, 64, 200, 450, 1300] if steps == "single" else [0, 40, 0, 333, 100]
    adds = [1] * 7 if steps == "single" else [70, 129, 1, 33, 200]
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, block, n_kv, hd)
    o = dict(CHANGES[change])
    if o.pop("slopes", False):
        o["slopes"] = (2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)).astype(np.float32)
    if o.pop("prefix", False):
        # none, some, a chunk, past the row, past the request, negative
        o["prefix"] = np.array([0, 20, 64, 70, 10 ** 6, -5, 400][:len(adds)], np.int32)
    check(dev, cache, table, q_start, kv_len, queries(rng, sum(adds), heads, hd, 2.0), 1 / np.sqrt(hd), **o)


@pytest.mark.parametrize("kq", [-0.25, 0.0, 1e-30, 3.0])
@pytest.mark.parametrize("cap", [0.0, 10.0])
@pytest.mark.parametrize("large", [0, 1])
def test_score_factors(dev, option, kq, cap, large):
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(17)
    cache, table, q_start, kv_len = ko.requests(rng, [400, 0, 90], [1, 60, 3], 32, 2, 64)
    check(dev, cache, table, q_start, kv_len, queries(rng, 64, 4, 64), kq, cap=cap)
    check(dev, cache, table, [0, 1, 1, 4], kv_len, queries(rng, 4, 4, 64), kq, cap=cap)


@pytest.mark.parametrize("splits", [1, 3, 64])
@pytest.mark.parametrize("row_waves", [1, 4])
@pytest.mark.parametrize("heads,n_kv,hd", [(8, 2, 128), (3, 3, 64), (6, 2, 256), (20, 1, 96)])
def test_pieces(dev, option, heads, n_kv, hd, row_waves, splits):
    """Pieces of any number, joined by the last workgroup to arrive; lengths
    from less than a piece to many."""
    option("ATTNP_ROW_WAVES", row_waves)
    option("ATTNP_SPLITS", splits)
    rng = np.random.default_rng(row_waves * splits + hd)
    cache, table, q_start, kv_len = ko.requests(rng, [3000, 1, 64, 700, 0, 129], [1, 1, 2, 1, 3, 0], 32, n_kv, hd)
    check(dev, cache, table, q_start, kv_len, queries(rng, 8, heads, hd, 2.0), 0.09)


@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("hd", [128, 64, 96])
def test_splits_of_large_blocks(dev, option, hd, splits):
    option("ATTNP_LARGE", 1)
    option("ATTNP_SPLITS", splits)
    rng = np.random.default_rng(splits)
    cache, table, q_start, kv_len = ko.requests(rng, [900, 0, 3000, 5], [150, 100, 129, 40], 64, 2, hd)
    check(dev, cache, table, q_start, kv_len, queries(rng, 419, 4, hd, 2.0), 0.09)


@pytest.mark.parametrize("hd", [128, 64])
def test_prompts_beside_single_tokens(dev, option, hd):
    """Both row blocks in one call, in any order of the requests."""
    option("ATTNP_LARGE", 1)
    rng = np.random.default_rng(hd)
    lengths, adds = [1500, 0, 333, 70, 40, 2000, 9], [1, 200, 1, 16, 17, 90, 5]
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, 32, 2, hd)
    check(dev, cache, table, q_start, kv_len, queries(rng, sum(adds), 8, hd, 2.0), 0.09)


@pytest.mark.parametrize("n_req", [63, 64, 65, 200, 256, 257, 300])
@pytest.mark.parametrize("large", [0, 1])
def test_many_requests(dev, option, n_req, large):
    """More than the 64 requests that a wave keeps in one register, and more
    than the 256 that are listed on the device."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(n_req)
    lengths = [int(x) for x in np.exp(rng.uniform(0, 6.5, n_req))]
    adds = [int(x) for x in rng.choice([0, 1, 1, 1, 4, 40], n_req)]
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, 16, 1, 32)
    check(dev, cache, table, q_start, kv_len, queries(rng, sum(adds), 3, 32, 2.0), 0.2)


@pytest.mark.parametrize("adds", [[2, 3, 8], [4] * 5, [5, 1, 16, 2]])
def test_a_few_tokens_each(dev, adds):
    """Drafted tokens: more rows than a 16-row block, fewer than a prompt's."""
    rng = np.random.default_rng(len(adds))
    cache, table, q_start, kv_len = ko.requests(rng, [700, 90, 2000, 31, 8][:len(adds)], adds, 32, 2, 128)
    check(dev, cache, table, q_start, kv_len, queries(rng, sum(adds), 10, 128, 2.0), 1 / np.sqrt(128))


def test_long_context(dev):
    """100 000 tokens in one request beside a short one: many splits, and
    scores with a peak, so that the maximum moves late."""
    rng = np.random.default_rng(5)
    cache, table, q_start, kv_len = ko.requests(rng, [99_999, 70], [1, 1], 64, 2, 64)
    q = queries(rng, 2, 4, 64, 1.0)
    cache.k[table[0, 1500], :, 3] = np.sign(q[0, ::2]).astype(np.int8) * 127
    check(dev, cache, table, q_start, kv_len, q, 0.5)


def test_offsets_past_32_bits(dev):
    """Pages whose codes lie more than 2^32 bytes into the cache."""
    rng = np.random.default_rng(6)
    block, n_kv, hd = 256, 4, 256
    page = block * n_kv * hd
    n_pages = (1 << 32) // page + 40
    small, table, q_start, kv_len = ko.requests(rng, [1000, 300], [1, 2], block, n_kv, hd)
    held = [int(p) for r, n in enumerate(kv_len) for p in table[r, :ko.blocks_of(int(n), block)]]
    far = {p: n_pages - 1 - 3 * i for i, p in enumerate(held)}
    assert min(far.values()) * page > 1 << 32
    big = [dev.alloc(n_pages * page), dev.alloc(n_pages * page), dev.alloc(n_pages * n_kv * 4), dev.alloc(n_pages * n_kv * 4)]
    try:
        moved = table.copy()
        for r, n in enumerate(kv_len):
            for b in range(ko.blocks_of(int(n), block)):
                moved[r, b] = far[int(table[r, b])]
        for p, f in far.items():
            for buf, src, size in zip(big, (small.k, small.v, small.ks, small.vs), (page, page, n_kv * 4, n_kv * 4)):
                row = np.ascontiguousarray(src[p])
                dev._check(dev.L.sihip_memcpy_htod(dev.ctx, buf.ptr + f * size, row.ctypes.data, row.nbytes))
        q = queries(rng, 3, 8, hd, 2.0)
        want, err, _ = ko.attention(small, table, q_start, kv_len, q, 0.07)
        k, v = rng.standard_normal((2, 3, n_kv, hd)).astype(np.float32)
        with ko.OnDevice(dev, q=q, out=np.zeros_like(q), kn=k, vn=v, slots=moved[0, :1].astype(np.int64) * block + 5,
                         ro=np.zeros((2, n_kv * hd), np.float32)) as d:
            c = sa.KvCache(k=big[0].ptr, v=big[1].ptr, k_scale=big[2].ptr, v_scale=big[3].ptr, n_pages=n_pages,
                           n_head_kv=n_kv, head_dim=hd, block=block)
            b = ko.put_batch(d, moved, q_start, kv_len, 3)
            dev.attn_paged_dev(c, b, sa.AttnPaged(q=d.ptr("q"), ldq=8 * hd, out=d.ptr("out"), ldo=8 * hd, n_head=8, kq_scale=0.07))
            dev.kv_read_dev(c, d.ptr("slots"), 1, d.ptr("ro"), n_kv * hd, d.ptr("ro") + 4 * n_kv * hd, n_kv * hd)
            dev.synchronize()
            assert (np.abs(d.get("out") - want) <= err + 1e-30).all()
            kr, vr = small.rows(table[0], 6)
            assert np.array_equal(d.get("ro"), np.stack([kr[:, 5].reshape(-1), vr[:, 5].reshape(-1)]).astype(np.float32))
            # and a write there: the step's rows again, read back in values
            dev.kv_append_dev(c, b, d.ptr("kn"), n_kv * hd, d.ptr("vn"), n_kv * hd)
            dev.kv_read_dev(c, d.put("s2", np.array([moved[0, 3] * block + 1000 % block], np.int64)), 1, d.ptr("ro"), n_kv * hd,
                            d.ptr("ro") + 4 * n_kv * hd, n_kv * hd)
            dev.synchronize()
            small.append(table, q_start, kv_len, k, v)
            kr, vr = small.rows(table[0], 1001)
            assert np.array_equal(d.get("ro"), np.stack([kr[:, 1000].reshape(-1), vr[:, 1000].reshape(-1)]).astype(np.float32))
    finally:
        for b in big:
            b.free()


def test_rows_at_odd_addresses_with_gaps(dev):
    rng = np.random.default_rng(11)
    cache, table, q_start, kv_len = ko.requests(rng, [90, 7], [1, 40], 16, 2, 80)
    check(dev, cache, table, q_start, kv_len, queries(rng, 41, 6, 80, 2.0), 0.1, ldq=6 * 80 + 7, ldo=6 * 80 + 1, shift=3)


@pytest.mark.parametrize("large", [0, 1])
def test_rows_that_see_nothing(dev, option, large):
    """Requests with impossible numbers write nothing; keys in pages outside
    the pool are not seen, and a row that sees none is zero."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(12)
    cache, table, q_start, kv_len = ko.requests(rng, [40, 20, 30, 9], [2, 2, 2, 2], 16, 2, 64)
    q = queries(rng, 9, 4, 64)
    whole = check(dev, cache, table, q_start, kv_len, q[:8], 0.2)
    torn = table.copy()
    torn[0, :3], torn[1, 0] = [-1, cache.n_pages, 2 ** 31 - 1], -7
    got = run(dev, cache, torn, q_start, kv_len, q[:8], 0.2)
    assert not got[0:2].any()
    # request 1 sees positions 16 .. only: as a window of its rows would
    for i, n in ((2, 5), (3, 6)):
        want, err, _ = ko.attention(cache, table, np.array([0, 0, 1, 1, 1]), np.array([0, 16 + n, 0, 0]), q[i:i + 1], 0.2, window=n)
        assert (np.abs(got[i] - want[0]) <= err[0]).all()
    assert np.array_equal(got[4:], whole[4:])
    for q0, end in (([0, 3, 3, 3, 3], [2, 0, 0, 0]), ([0, 10, 10, 10, 10], [42, 0, 0, 0]), ([-1, 1, 1, 1, 1], [42, 0, 0, 0]),
                    ([2, 0, 0, 0, 0], [42, 22, 0, 0]), ([0, 0, 0, 0, 0], [42, 22, 32, 11]), ([0, 1, 1, 1, 1], [-1, 0, 0, 0])):
        got = run(dev, cache, table, np.array(q0), np.array(end), q, 0.2, bounds=dict(max_q=9, max_kv=64))
        assert (got == 55.0).all(), (q0, end)


def test_bounds_cut(dev):
    """max_q and max_kv below the device's numbers: nothing past them is
    written or seen."""
    rng = np.random.default_rng(13)
    cache, table, q_start, kv_len = ko.requests(rng, [200, 10], [1, 20], 16, 1, 64)
    q = queries(rng, 21, 2, 64)
    got = run(dev, cache, table, q_start, kv_len, q, 0.2, bounds=dict(max_q=8, max_kv=100))
    assert (got[9:] == 55.0).all()
    short = kv_len.copy()
    want, err, _ = ko.attention(cache, table, np.array([0, 1, 1]), np.array([100, 0]), q[:1], 0.2)
    assert (np.abs(got[0] - want[0]) <= err[0]).all()
    want, err, _ = ko.attention(cache, table, q_start, short, q, 0.2)
    assert (np.abs(got[1:9] - want[1:9]) <= err[1:9]).all()


@pytest.mark.parametrize("steps,large", [("single", 0), ("prompt", 0), ("prompt", 1)])
def test_garbage_that_no_row_sees(dev, option, steps, large):
    """NaN scales and any codes behind the window and past the length, and
    large, tiny and zero scales of what is seen."""
    option("ATTNP_LARGE", large)
    rng = np.random.default_rng(14)
    lengths, adds = ([700, 300], [1, 1]) if steps == "single" else ([400, 0], [200, 150])
    cache, table, q_start, kv_len = ko.requests(rng, lengths, adds, 16, 2, 64)
    q = queries(rng, sum(adds), 4, 64)
    window = 100
    first = [max(0, n - window) // 16 for n in lengths]  # blocks before it: no row sees them
    for r in range(2):
        for b in range(first[r]):
            cache.ks[table[r, b]], cache.vs[table[r, b]] = np.nan, [np.inf, np.nan]
    last = [int(table[r, kv_len[r] // 16 - 1]) for r in range(2)]
    cache.vs[last[0]], cache.ks[last[0]] = [1e30, 1e-30], [0.0, 1e-37]
    cache.vs[last[1]], cache.ks[last[1]] = [0.0, 3e-38], [1e-3, 0.0]
    got = run(dev, cache, table, q_start, kv_len, q, 0.2, window=window)
    assert np.isfinite(got).all()
    want, err, _ = ko.attention(cache, table, q_start, kv_len, q, 0.2, window=window)
    assert (np.abs(got - want) <= err + 1e-30).all()


def test_sizes_of_queries(dev):
    """Rows of zeros, of the smallest and of large numbers, and rows whose
    values differ by far in size; NaN stays in its own row and head."""
    rng = np.random.default_rng(15)
    cache, table, q_start, kv_len = ko.requests(rng, [300] * 6, [1] * 6, 32, 1, 64)
    q = queries(rng, 6, 2, 64)
    q[0], q[1], q[2] = 0.0, q[1] * np.float32(1e-38), q[2] * 40
    q[3] *= np.exp(rng.normal(0, 4, 64)).astype(np.float32)
    q[4, 1, 5] = np.nan
    got = run(dev, cache, table, q_start, kv_len, q, 0.125)
    want, err, _ = ko.attention(cache, table, q_start, kv_len, np.nan_to_num(q), 0.125)
    assert np.isnan(got[4, 1]).all()
    got[4, 1], want[4, 1] = 0, 0
    assert (np.abs(got - want) <= err + 1e-30).all()


@pytest.mark.parametrize("row_waves", [1, 4])
def test_same_bits_every_time(dev, option, row_waves):
    """The order in which workgroups arrive does not show."""
    option("ATTNP_ROW_WAVES", row_waves)
    rng = np.random.default_rng(16)
    cache, table, q_start, kv_len = ko.requests(rng, [5000, 3000, 64, 900], [1, 1, 1, 1], 32, 2, 128)
    q = queries(rng, 4, 8, 128)
    first = run(dev, cache, table, q_start, kv_len, q, 0.09)
    for _ in range(4):
        assert np.array_equal(run(dev, cache, table, q_start, kv_len, q, 0.09).view(np.uint32), first.view(np.uint32))


def test_overlapping_spans_leave_the_workspace_clean(dev, option):
    """Numbers that give the same rows to several requests are more blocks than
    the grid was made for: what it cannot join is not begun, and the next call
    finds its counters at zero."""
    option("ATTNP_LARGE", 0)
    rng = np.random.default_rng(17)
    lengths = [2000, 0] * 6
    cache, table, q_start, kv_len = ko.requests(rng, lengths, [64, 0] * 6, 32, 2, 64)
    q = queries(rng, 64, 2, 64)
    with ko.OnDevice(dev, q=q, out=np.zeros_like(q)) as d:
        c = ko.put_cache(d, cache)
        b = ko.put_batch(d, table, [0, 64] * 6 + [0], kv_len, 64, max_q=64)
        a = sa.AttnPaged(q=d.ptr("q"), ldq=128, out=d.ptr("out"), ldo=128, n_head=2, kq_scale=0.1)
        n = dev.attn_paged_workspace(c, b, a)
        assert n > 0
        d.put("ws", np.zeros(n, np.uint8))
        a.workspace, a.workspace_bytes = d.ptr("ws"), n
        dev.attn_paged_dev(c, b, a)
        dev.synchronize()
        assert not d.get("ws")[:256 << 10].any()
