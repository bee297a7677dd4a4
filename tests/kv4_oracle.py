"""The paged 4-bit KV cache and the rotation of rows restated in numpy (test
infrastructure; kv_oracle has the plans, the device side and attention, which takes
this cache as well)."""
import numpy as np

import siphon_amd as sa

from . import kv_oracle as ko

ORDER = [0, 2, 4, 6, 1, 3, 5, 7]  # elements of a word, from the lowest nibble up


def pack(codes):
    """Codes along the last axis to bytes."""
    n = (codes.astype(np.int64) + 8).reshape(*codes.shape[:-1], -1, 8)[..., ORDER]
    word = sum(n[..., i] << (4 * i) for i in range(8)).astype(np.uint32)
    return word.view(np.uint8).reshape(*codes.shape[:-1], -1)


def unpack(data):
    word = np.ascontiguousarray(data).view(np.uint32)
    out = np.zeros((*word.shape, 8), np.int8)
    for i, e in enumerate(ORDER):
        out[..., e] = (word >> (4 * i) & 15).astype(np.int8) - 8
    return out.reshape(*data.shape[:-1], -1)


def bf16(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def quantize(x):
    """(codes, subs, scale bits) of rows [..., head_dim], f32: what include/sihip.h defines."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, 32)
    a = np.clip(np.where(np.isfinite(g), g, np.float32(0)), np.float32(-2.0 ** 126), np.float32(2.0 ** 126))
    top, low = np.maximum(a.max(-1), 0), np.maximum(-a.min(-1), 0)
    size = np.maximum(top, low) * np.float32(0.125)
    most = size.max(-1)
    bits = ((most / np.float32(127)).view(np.uint32).astype(np.uint64) + 0xffff >> 16).astype(np.uint16)
    bits = np.where(most < np.float32(2.0 ** -103), np.uint16(0), bits)
    scale = bf16(bits).astype(np.float64)[..., None]
    with np.errstate(all="ignore"):
        n = np.where(scale > 0, np.clip(np.ceil(size.astype(np.float64) / scale), 1, 127), 1)
        sub = np.where(low >= top, n, -n)
        step = (sub * scale)[..., None]
        q = np.clip(np.rint(g.astype(np.float64) / step), -8, 7)
        q = np.where(np.isnan(g) | (step == 0), 0, q)
    return q.reshape(x.shape).astype(np.int8), sub.astype(np.int8), bits


def rotate(x, pos, rope, neighbours):
    """Rows [token, head, dim] by the table [position, pair, 2], rounded once."""
    x, pairs = np.asarray(x, np.float32), rope.shape[1]
    out = x.copy()
    c, s = (rope[pos, :, i].astype(np.float64)[:, None] for i in (0, 1))
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if neighbours else (slice(0, pairs), slice(pairs, 2 * pairs))
    y, z = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
    with np.errstate(invalid="ignore"):
        out[..., a], out[..., b] = (y * c - z * s).astype(np.float32), (y * s + z * c).astype(np.float32)
    return out


def table(n, dim, base=10000.0):
    """Cosines and sines of n positions, f32 [n, dim / 2, 2]."""
    angle = np.arange(n)[:, None] * base ** (-np.arange(0, dim, 2) / dim)
    return np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)


class Cache:
    """One layer's cache on the host: codes unpacked, NaN scales where nothing was written."""

    def __init__(self, rng, n_pages, n_kv, hd, block):
        self.n_pages, self.n_kv, self.hd, self.block = n_pages, n_kv, hd, block
        self.k = rng.integers(-8, 8, (n_pages, n_kv, block, hd)).astype(np.int8)
        self.v = rng.integers(-8, 8, (n_pages, n_kv, hd, block)).astype(np.int8)
        self.ksub, self.vsub = (rng.integers(-128, 128, (n_pages, n_kv, hd // 32, block)).astype(np.int8) for _ in range(2))
        self.ks, self.vb = (np.full((n_pages, n_kv, block), 0x7fc0, np.uint16) for _ in range(2))

    @property
    def vs(self):
        """Of each page and head, what times 128 is no less than any value (for kv_oracle's bounds)."""
        s = bf16(self.vb)
        return np.where(np.isfinite(s), s, 0).max(2) * 8

    def values(self, page):
        """(keys, values) [head, token, dim] of a page, f64."""
        with np.errstate(invalid="ignore"):
            k, v = (np.repeat(sub[page].astype(np.float64) * bf16(s[page])[:, None], 32, 1).swapaxes(1, 2)
                    for sub, s in ((self.ksub, self.ks), (self.vsub, self.vb)))
            return self.k[page] * k, self.v[page].swapaxes(1, 2) * v

    def rows(self, table, n):
        pages = [self.values(int(p)) for p in table[:ko.blocks_of(n, self.block)]]
        if not pages:
            return (np.zeros((self.n_kv, 0, self.hd)),) * 2
        return tuple(np.concatenate(x, 1)[:, :n] for x in zip(*pages))

    def append(self, table, q_start, kv_len, k, v, max_q=2 ** 31, max_kv=2 ** 31):
        for r, end in enumerate(int(x) for x in kv_len):
            q0, q1 = int(q_start[r]), int(q_start[r + 1])
            start = end - (q1 - q0)
            for t in range(q0, min(q1, q0 + max_q)):
                pos = start + t - q0
                page, off = int(table[r, pos // self.block]) if pos < max_kv else -1, pos % self.block
                if not 0 <= page < self.n_pages:
                    continue
                self.k[page, :, off], self.ksub[page, :, :, off], self.ks[page, :, off] = quantize(k[t])
                self.v[page, :, :, off], self.vsub[page, :, :, off], self.vb[page, :, off] = quantize(v[t])

    def arrays(self):
        return dict(k=pack(self.k), v=pack(self.v), ksub=self.ksub, vsub=self.vsub, ks=self.ks, vb=self.vb)


def put_cache(d, cache):
    p = {name: d.put(name, a) for name, a in cache.arrays().items()}
    return sa.Kv4Cache(k=p["k"], v=p["v"], k_sub=p["ksub"], v_sub=p["vsub"], k_scale=p["ks"], v_scale=p["vb"],
                       n_pages=cache.n_pages, n_head_kv=cache.n_kv, head_dim=cache.hd, block=cache.block)


def requests(rng, lengths, adds, block, n_kv, hd, spare_blocks=2):
    """As kv_oracle.requests: (cache, table, q_start, kv_len)."""
    ends = [n + a for n, a in zip(lengths, adds)]
    held = [ko.blocks_of(e, block) for e in ends]
    n_pages = sum(held) + 3
    order = rng.permutation(n_pages)
    cache = Cache(rng, n_pages, n_kv, hd, block)
    junk = np.array([-1, n_pages, 2 ** 31 - 1, -2 ** 31, int(order[-1])])
    pages = rng.choice(junk, (len(ends), max(held) + spare_blocks)).astype(np.int32)
    at = 0
    for r, n in enumerate(held):
        pages[r, :n] = order[at:at + n]
        for b in range(n):
            page, fill = int(order[at + b]), min(block, ends[r] - b * block)
            for s, spread in ((cache.ks, 1.0), (cache.vb, 1.5)):
                x = np.exp(rng.normal(0, spread, (n_kv, fill))).astype(np.float32) * np.float32(0.0025)
                s[page, :, :fill] = (x.view(np.uint32) >> 16).astype(np.uint16)
        at += n
    q_start = np.concatenate([[0], np.cumsum(adds)]).astype(np.int32)
    return cache, pages, q_start, np.array(ends, np.int32)
