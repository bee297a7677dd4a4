"""Log probabilities, entropies and the most likely tokens of rows of logits
against their definition in 64 bits.

The bound, relative to the sum l of e^(x - m): 2^-22 for an f32 exponential, 3 |x - m| 2^-24
for the three roundings of its argument, weighted by p: 3 D 2^-24 with D = sum p |x - m|; a running
maximum that moves R times (at most one for each of 16 logits that a thread takes, and once for each
of 6 + 2 + 9 joins) the same again for each; the f64 sums add nothing. Of t = sum e^(x - m) (x - m): the same and
2^-24 for each of 16 additions. A random order of n logits moves a thread's maximum some ln n times; sorted rows up to
n / 4096 times. The result is rounded once more."""
import numpy as np
import pytest

import siphon_amd as sa

from . import kv_oracle as ko
from .test_gpu_slices import _HipGraph
from .test_gpu_streams import _Streams

pytestmark = pytest.mark.gpu


def definition(x, token, n_top):
    """(logprob, entropy, top ids, top logprobs, D) in f64."""
    y = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = y.max(1, keepdims=True)
        none = np.isneginf(m[:, 0])
        d = y - np.where(none[:, None], 0, m)
        e = np.exp(d)
        l = e.sum(1, keepdims=True)
        p = e / l
        spread = -np.where(p > 0, p * d, 0).sum(1)
        entropy = np.where(none, 0, np.log(l[:, 0]) + spread)
        lp = d - np.log(l)
        bad = np.isnan(y).any(1) | np.isposinf(y).any(1)
        lp[none], lp[bad], entropy[bad] = -np.inf, np.nan, np.nan
        # the result is f32: what is half a step or more past its largest number (2^128 - 2^103) is infinite in it
        lp[lp <= -(2.0 ** 128 - 2.0 ** 103)] = -np.inf
    order = np.argsort(-np.where(np.isnan(y), -np.inf, y), axis=1, kind="stable")[:, :n_top]
    given = np.take_along_axis(lp, np.clip(token, 0, x.shape[1] - 1), 1)
    top = np.take_along_axis(lp, order, 1)
    top[np.isnan(np.take_along_axis(y, order, 1))] = np.nan
    return given, entropy, order, top, np.nan_to_num(spread, nan=0, posinf=0)


def buffers(x, token, n_top, gap=0, shift=0):
    rows, n = x.shape
    flat = np.full(shift + rows * (n + gap), 1e9, np.float32)
    flat[shift:].reshape(rows, n + gap)[:, :n] = x
    return dict(x=flat, token=token.astype(np.int32), lp=np.full(token.shape, 55.0, np.float32), h=np.full(rows + 1, 55.0, np.float32),
                ti=np.full((rows, max(n_top, 1)), 77, np.int32), tl=np.full((rows, max(n_top, 1)), 55.0, np.float32))


def arguments(d, x, token, n_top, gap=0, shift=0, /, **o):
    return sa.Logprobs(**{**dict(logits=d.ptr("x") + 4 * shift, ld=x.shape[1] + gap, n_rows=x.shape[0], n_vocab=x.shape[1],
                                 token=d.ptr("token"), n_token=token.shape[1], logprob=d.ptr("lp"), entropy=d.ptr("h"), n_top=n_top,
                                 top_id=d.ptr("ti"), top_logprob=d.ptr("tl")), **o})


def compare(d, x, token, n_top, raises=64):
    given, entropy, ids, top, spread = definition(x, token, n_top)
    bound = (2.0 ** -22 + 3 * spread * 2.0 ** -24) * (1 + raises)
    lp, h = d.get("lp").astype(np.float64), d.get("h").astype(np.float64)
    valid = (token >= 0) & (token < x.shape[1])
    assert (lp[~valid] == 55).all() and h[-1] == 55
    pairs = [(lp[valid], given[valid], np.broadcast_to(bound[:, None], lp.shape)[valid]),
             (h[:-1], entropy, bound * (2 + spread) + 16 * 2.0 ** -24 * spread)]
    if n_top:
        assert np.array_equal(d.get("ti"), ids)
        pairs.append((d.get("tl").astype(np.float64), top, np.broadcast_to(bound[:, None], top.shape)))
    for got, want, b in pairs:
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
        got, want, b = got[fine], want[fine], b[fine]
        assert (np.abs(got - want) <= b + 2.0 ** -24 * np.abs(want)).all()


def check(dev, x, token, n_top, gap=0, shift=0, raises=64, stream=None):
    with ko.OnDevice(dev, **buffers(x, token, n_top, gap, shift)) as d:
        dev.logprobs_dev(arguments(d, x, token, n_top, gap, shift), stream)
        dev.synchronize()
        compare(d, x, token, n_top, raises)


def logits(rng, rows, n, size=3.0, ties=True):
    x = rng.standard_normal((rows, n)) * size
    return (np.round(x * 16) / 16 if ties else x).astype(np.float32)


def tokens(rng, rows, n, given=2):
    t = rng.integers(0, n, (rows, given))
    t[rng.random(t.shape) < 0.1] = rng.choice([-1, n, -100, 2 ** 31 - 1])
    return t


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 2), (3, 5), (2, 63), (5, 64), (1, 4096), (2, 4097), (7, 1000), (1, 32003), (64, 2049),
                                    (1, 100003), (1, 151936), (2, 262147), (40, 5000), (300, 4099), (2100, 517)])
@pytest.mark.parametrize("n_top", [0, 1, 5, 20, 64])
def test_rows(dev, rows, n, n_top):
    rng = np.random.default_rng(rows + n)
    check(dev, logits(rng, rows, n), tokens(rng, rows, n), min(n_top, n))


@pytest.mark.parametrize("gap,shift", [(0, 1), (1, 0), (3, 2), (4, 3), (5, 1)])
def test_rows_at_any_address(dev, gap, shift):
    """Rows that begin anywhere in a granule; what lies around them is not read as logits."""
    rng = np.random.default_rng(gap)
    for n in (1, 2, 3, 4, 5, 1023, 9001):
        check(dev, logits(rng, 5, n), tokens(rng, 5, n), min(n, 7), gap, shift)


@pytest.mark.parametrize("order", ["equal", "rising", "falling", "rising_steps", "two_values"])
@pytest.mark.parametrize("n", [300, 20000])
def test_orders(dev, order, n):
    """Rows in which every logit passes the threshold so far, and rows of ties."""
    rng = np.random.default_rng(1)
    i = np.arange(n, dtype=np.float32)
    x = dict(equal=i * 0 + 2, rising=i / 64, falling=-i / 64, rising_steps=np.floor(i / 100), two_values=(i % 7 == 3) * np.float32(1))[order]
    for n_top in (1, 20, 64):
        check(dev, np.stack([x, x * np.float32(0.25)]).astype(np.float32), tokens(rng, 2, n), n_top, raises=n / 64 + 64)


def test_masks(dev):
    """-inf for what is not allowed: all, all but one, nearly all; the type's lowest value in its place;
    +inf and NaN; -0 and 0 are equal."""
    rng = np.random.default_rng(2)
    n = 9000
    x = logits(rng, 12, n)
    x[0] = -np.inf
    x[1], x[1, 777] = -np.inf, -3.0
    x[2, rng.random(n) < 0.999] = -np.inf
    x[3] = np.finfo(np.float32).min
    x[4, 100:] = np.finfo(np.float32).min
    x[5, 5000] = np.nan
    x[6, 1] = np.inf
    x[7], x[7, ::2] = 0.0, -0.0
    x[8], x[8, 5], x[8, 9] = -np.inf, np.nan, 1.0
    x[9] = np.nan
    x[10, :10] = np.finfo(np.float32).max
    x[11] = np.finfo(np.float32).min
    x[11, 8000] = np.finfo(np.float32).max
    for n_top in (0, 3, 64):
        check(dev, x, tokens(rng, 12, n, 5), n_top)


def test_nearly_certain(dev):
    """Where one token has all but 2^-30 of the probability its log probability is that small
    rest, and not zero."""
    rng = np.random.default_rng(3)
    x = logits(rng, 4, 50000, 1.0, ties=False)
    at = rng.integers(0, 50000, 4)
    x[np.arange(4), at] = 32.0
    want, entropy, _, _, _ = definition(x, at[:, None], 0)
    with ko.OnDevice(dev, **buffers(x, at[:, None], 1)) as d:
        dev.logprobs_dev(arguments(d, x, at[:, None], 1))
        dev.synchronize()
        assert (want < 0).all() and (want > -2.0 ** -20).all()
        # e^-d with d about 32: 3 * 32 roundings of 2^-24 and the exponential's own, of l - 1 itself
        assert np.allclose(d.get("lp"), want, rtol=2.0 ** -16, atol=0)
        assert np.allclose(d.get("h")[:4], entropy, rtol=2.0 ** -16, atol=0)
        assert np.array_equal(d.get("ti")[:, 0], at) and np.allclose(d.get("tl"), want, rtol=2.0 ** -16, atol=0)


def test_parts_that_are_not_asked_for(dev):
    rng = np.random.default_rng(4)
    x, token = logits(rng, 3, 5000), tokens(rng, 3, 5000)
    for gone in (dict(entropy=0), dict(n_token=0), dict(token=0, logprob=0), dict(n_top=0, top_id=0, top_logprob=0)):
        with ko.OnDevice(dev, **buffers(x, token, 5)) as d:
            dev.logprobs_dev(arguments(d, x, token, 5, **gone))
            dev.synchronize()
            want = buffers(x, token, 5)
            kept = dict(entropy=["h"], n_token=["lp"], token=["lp"], n_top=["ti", "tl"])[next(iter(gone))]
            for name in ("lp", "h", "ti", "tl"):
                assert np.array_equal(d.get(name), want[name]) == (name in kept), (gone, name)
    with ko.OnDevice(dev, **buffers(x, token, 5)) as d:
        dev.logprobs_dev(arguments(d, x, token, 5, n_rows=0))
        dev.synchronize()
        assert (d.get("lp") == 55).all() and (d.get("ti") == 77).all()


def test_rows_past_32_bits(dev):
    """Rows whose logits lie more than 2^32 bytes into the array."""
    rng = np.random.default_rng(5)
    n, ld, rows = 3001, 600_000_001, 3
    x, token = logits(rng, rows, n), tokens(rng, rows, n)
    big = dev.alloc(4 * ((rows - 1) * ld + n))
    try:
        for r in range(rows):
            dev._check(dev.L.sihip_memcpy_htod(dev.ctx, big.ptr + 4 * r * ld, x[r].ctypes.data, x[r].nbytes))
        with ko.OnDevice(dev, **buffers(x, token, 5)) as d:
            dev.logprobs_dev(arguments(d, x, token, 5, logits=big.ptr, ld=ld))
            dev.synchronize()
            compare(d, x, token, 5)
    finally:
        big.free()


@pytest.mark.parametrize("n_top", [0, 5, 64])
def test_the_longest_row(dev, n_top):
    """2^31 - 1 logits, of which the last few are not all alike."""
    rng = np.random.default_rng(9)
    n, piece, far = 2 ** 31 - 1, 1 << 26, 3000
    fill, tail = np.full(piece, -5, np.float32), logits(rng, 1, far)
    tail[0, -1] = tail.max() + 1
    big = dev.alloc(4 * n)
    try:
        for at in range(0, n, piece):
            dev._check(dev.L.sihip_memcpy_htod(dev.ctx, big.ptr + 4 * at, fill.ctypes.data, 4 * min(piece, n - at)))
        dev._check(dev.L.sihip_memcpy_htod(dev.ctx, big.ptr + 4 * (n - far), tail.ctypes.data, tail.nbytes))
        token = np.array([[0, n - 1, n - far, -1]])
        with ko.OnDevice(dev, **buffers(tail, token, n_top)) as d:
            dev.logprobs_dev(arguments(d, tail, token, n_top, logits=big.ptr, ld=n, n_vocab=n))
            dev.synchronize()
            y = tail[0].astype(np.float64)
            m, e = y.max(), np.exp(y - y.max())
            rest = (n - far) * np.exp(-5 - m)
            l = rest + e.sum()
            spread = ((m - y) * e).sum() / l + rest / l * (m + 5)
            lp = lambda x: x - m - np.log(l)
            # a thread's maximum may be raised at each of its runs of the tail
            bound = (2.0 ** -22 + 3 * spread * 2.0 ** -24) * 66
            got = d.get("lp")[0]
            assert got[3] == 55
            for g, x in zip(got, (-5.0, y[-1], y[0])):
                assert abs(g - lp(x)) <= bound + 2.0 ** -24 * abs(lp(x))
            assert abs(d.get("h")[0] - (np.log(l) + spread)) <= bound * (2 + spread) + 2.0 ** -20 * spread
            if n_top:
                order = np.argsort(-y, kind="stable")[:n_top]
                assert np.array_equal(d.get("ti")[0], n - far + order)
                assert (np.abs(d.get("tl")[0] - lp(y[order])) <= bound + 2.0 ** -24 * np.abs(lp(y[order]))).all()
    finally:
        big.free()


def test_streams_workspaces_and_graphs(dev):
    """Two calls at once with workspaces of their own; captured ones replayed with other
    logits and eager calls between."""
    rng = np.random.default_rng(6)
    shapes = [(2, 30000, 7), (3, 9001, 20)]
    x = [logits(rng, r, n) for r, n, _ in shapes]
    token = [tokens(rng, r, n) for r, n, _ in shapes]
    ss, graphs, held = _Streams(), [], []
    try:
        for (r, n, top), a, t in zip(shapes, x, token):
            d = ko.OnDevice(dev, **buffers(a, t, top))
            held.append(d)
            args = arguments(d, a, t, top)
            size = dev.logprobs_workspace(args)
            assert size > 0
            args.workspace, args.workspace_bytes = d.put("ws", np.zeros(size, np.uint8)), size
            d.args = args
        streams = [ss.create() for _ in held]
        for _ in range(3):
            for d, s in zip(held, streams):
                dev.logprobs_dev(d.args, s)
        for s in streams:
            ss.sync(s)
        for d, a, t, (_, _, top) in zip(held, x, token, shapes):
            compare(d, a, t, top)
            assert not d.get("ws")[:1 << 18].any()
        for d in held:
            g = _HipGraph()
            graphs.append(g)
            g.begin()
            dev.logprobs_dev(d.args, g.stream.value)
            g.end()
        for step in range(4):
            x = [logits(rng, r, n) for r, n, _ in shapes]
            for d, a in zip(held, x):
                d.bufs["x"][0].fill(a)
            check(dev, x[0], token[0], 3)  # an eager call on the context's workspace
            for g in graphs:
                g._ok(g.hip.hipGraphLaunch(g.exec, g.stream))
            for g in graphs:
                g._ok(g.hip.hipStreamSynchronize(g.stream))
            for d, a, t, (_, _, top) in zip(held, x, token, shapes):
                compare(d, a, t, top)
    finally:
        dev.synchronize()
        for g in graphs:
            g.close()
        ss.close()
        for d in held:
            d.__exit__()


def test_same_bits_every_time(dev):
    rng = np.random.default_rng(7)
    x, token = logits(rng, 2, 100000, ties=False), tokens(rng, 2, 100000)
    seen = set()
    with ko.OnDevice(dev, **buffers(x, token, 64)) as d:
        for _ in range(5):
            dev.logprobs_dev(arguments(d, x, token, 64))
            dev.synchronize()
            seen.add(tuple(d.get(n).tobytes() for n in ("lp", "h", "ti", "tl")))
    assert len(seen) == 1
