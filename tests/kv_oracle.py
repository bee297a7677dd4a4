"""The paged 8-bit KV cache restated in numpy, in 64 bits (test
infrastructure), and the device side of a test: buffers and argument
structures of include/sihip.h."""
import numpy as np

import siphon_amd as sa


def blocks_of(tokens, block):
    return -(-tokens // block)


def plan(length, add, free, n_free, table, n_tok, block):
    """(table, q_start, kv_len, slot, pos, free, n_free, status) after a step."""
    n_pages, max_blocks = len(free), table.shape[1]
    length, add = [int(x) for x in length], [int(x) for x in add]
    ok = [n >= 0 and a >= -1 for n, a in zip(length, add)]
    before = [blocks_of(n, block) for n in length]
    fits = [o and b <= max_blocks and blocks_of(n + max(a, 0), block) <= max_blocks
            for o, n, a, b in zip(ok, length, add, before)]
    rows = [f and a or 0 for f, a in zip(fits, add)]
    back = [p for r, a in enumerate(add) if fits[r] and a == -1 for p in table[r, :before[r]]]
    need = sum(blocks_of(n + a, block) - b for n, a, b, f in zip(length, add, before, fits) if f and a > 0)
    total = sum(x for x in rows if x > 0)
    status = (not all(ok)) + 2 * any(o and not f for o, f in zip(ok, fits)) + 4 * (total > n_tok)
    if not 0 <= n_free <= n_pages or n_free + len(back) > n_pages:
        status += 16
    elif n_free + len(back) < need:
        status += 8
    table, free = table.copy(), free.copy()
    slot, pos = np.full(n_tok, -1, np.int64), np.full(n_tok, -1, np.int32)
    if status:
        return table, np.zeros(len(length) + 1, np.int32), np.array(length, np.int32), slot, pos, free, n_free, status
    stack = list(free[:n_free]) + back
    q_start, kv_len, t = [0], [], 0
    for r, (n, a) in enumerate(zip(length, add)):
        kv_len.append(0 if a < 0 else n + a)
        for p in range(n, n + max(a, 0)):
            if p % block == 0:
                table[r, p // block] = stack.pop()
            page = int(table[r, p // block])
            slot[t] = page * block + p % block if 0 <= page < n_pages else -1
            pos[t] = p
            t += 1
        q_start.append(t)
    keep = min(n_free, len(stack))
    assert list(free[:keep]) == stack[:keep]
    free[:len(stack)] = stack
    return table, np.array(q_start, np.int32), np.array(kv_len, np.int32), slot, pos, free, len(stack), status


def round_even(x):
    return np.rint(x)  # ties to even


def append_page(codes, scale, x, lo):
    """Codes [token, dim] (f64) and scale of a page whose tokens lo .. get x
    (f32): what sihip_kv_append_dev defines, and the bounds it keeps."""
    x = x.astype(np.float64)
    size = np.abs(x)
    top = np.max(size[np.isfinite(size)], initial=0.0)
    was = float(scale) if lo else 0.0
    now = max(was, 0.0 if top < 2.0 ** -100 else float(np.float32(top) / np.float32(127)))
    out = codes.astype(np.float64).copy()
    if now > was:
        out[:lo] = round_even(out[:lo] * was / now)
    if now > 0:
        with np.errstate(all="ignore"):
            q = np.clip(round_even(x / now), -127, 127)
        q[np.isnan(x)] = 0
    else:
        q = np.zeros_like(x)
    out[lo:lo + len(x)] = q
    return out, np.float32(now if now > was or lo == 0 else scale)


class Cache:
    """One layer's cache on the host: random pages, NaN scales where nothing
    was written."""

    def __init__(self, rng, n_pages, n_kv, hd, block):
        self.n_pages, self.n_kv, self.hd, self.block = n_pages, n_kv, hd, block
        self.k = rng.integers(-128, 128, (n_pages, n_kv, block, hd)).astype(np.int8)
        self.v = rng.integers(-128, 128, (n_pages, n_kv, hd, block)).astype(np.int8)
        self.ks = np.full((n_pages, n_kv), np.nan, np.float32)
        self.vs = np.full((n_pages, n_kv), np.nan, np.float32)

    def rows(self, table, n):
        """(keys, values) [head, position, dim] in f64 of positions 0 .. n - 1."""
        pages = [int(p) for p in table[:blocks_of(n, self.block)]]
        with np.errstate(invalid="ignore"):  # of scales that nothing was written to
            k = [self.k[p].astype(np.float64) * self.ks[p].astype(np.float64)[:, None, None] for p in pages]
            v = [self.v[p].swapaxes(1, 2).astype(np.float64) * self.vs[p].astype(np.float64)[:, None, None] for p in pages]
        if not pages:
            return (np.zeros((self.n_kv, 0, self.hd)),) * 2
        return np.concatenate(k, 1)[:, :n], np.concatenate(v, 1)[:, :n]

    def append(self, table, q_start, kv_len, k, v, max_q=2 ** 31, max_kv=2 ** 31):
        """The step's rows [token, head, dim] into the pages."""
        for r, end in enumerate(int(x) for x in kv_len):
            q0, q1 = int(q_start[r]), int(q_start[r + 1])
            start = end - (q1 - q0)
            end = min(start + min(q1 - q0, max_q), max_kv)  # of what is written
            for b in range(start // self.block, blocks_of(end, self.block) if end > start else 0):
                p, first = int(table[r, b]), max(start - b * self.block, 0)
                if not 0 <= p < self.n_pages:
                    continue
                t0 = q0 + b * self.block + first - start
                t1 = q0 + min(end, (b + 1) * self.block) - start
                for h in range(self.n_kv):
                    got, s = append_page(self.k[p, h], self.ks[p, h], k[t0:t1, h], first)
                    self.k[p, h], self.ks[p, h] = got.astype(np.int8), s
                    got, s = append_page(self.v[p, h].T, self.vs[p, h], v[t0:t1, h], first)
                    self.v[p, h], self.vs[p, h] = got.T.astype(np.int8), s


def attention(cache, table, q_start, kv_len, q, kq_scale, cap=0.0, slopes=None, prefix=None, window=0):
    """(out, error) [token, head, dim] in f64. The error bound counts, per
    score, the f32 sum of 2 hd products (2 hd 2^-24 of the sum of their
    magnitudes), the split of q into two f16 halves (2^-22) and a handful of
    f32 roundings of the factors and of the tanh (2^-21 of the score, 2^-21
    of the cap, 2^-23 of a bias) and of the running maximum it is taken from;
    twice the largest of them for a quotient of sums of exponentials, plus
    2^-20 for the exponentials and their split, and 2^-24 for each of the
    2 n + 64 additions of an output's chain: relative to sum p |v|. A key's
    weight times its value scale is held in f16 halves whose last one is off by
    at most 2^-34 of the row's largest such product. The bound has 2^-34 of the
    largest scale of all the request's pages and heads, times codes up to 128,
    for each key, which is more: kv_scores has a bound for each row and head."""
    T, H, hd = q.shape
    G = H // cache.n_kv
    out, err = np.zeros((T, H, hd)), np.zeros((T, H, hd))
    seen_rows = np.zeros(T, bool)
    for r, end in enumerate(int(x) for x in kv_len):
        q0, q1 = int(q_start[r]), int(q_start[r + 1])
        if q1 <= q0:
            continue
        k, v = cache.rows(table[r], end)
        vs = np.array([cache.vs[p] for p in table[r, :blocks_of(end, cache.block)]], np.float64)
        step = end * 2.0 ** -34 * 128 * np.max(vs[np.isfinite(vs)], initial=0.0)
        n = q1 - q0
        p = np.arange(end - n, end)[:, None]
        j = np.arange(end)[None, :]
        seen = j <= p
        if window:
            seen &= j > p - window
        if prefix is not None:
            seen |= j < int(prefix[r])
        seen_rows[q0:q1] = True
        for h in range(H):
            qh = q[q0:q1, h].astype(np.float64)
            kh, vh = np.nan_to_num(k[h // G]), np.nan_to_num(v[h // G])
            s = kq_scale * qh @ kh.T
            e = (2 * hd * 2.0 ** -24 + 2.0 ** -22) * abs(kq_scale) * (np.abs(qh) @ np.abs(kh).T) + 2.0 ** -21 * np.abs(s)
            if cap:
                s = cap * np.tanh(s / cap)
                e += 2.0 ** -21 * cap
            if slopes is not None:
                bias = float(slopes[h]) * np.abs(p - j)
                s = s - bias
                e += 2.0 ** -23 * bias
            s = np.where(seen, s, -np.inf)
            m = s.max(1, keepdims=True, initial=-np.inf)
            some = np.isfinite(m)
            w = np.exp(s - np.where(some, m, 0.0))
            l = w.sum(1, keepdims=True)
            w = np.divide(w, l, out=np.zeros_like(w), where=l > 0)
            out[q0:q1, h] = w @ vh
            # keys whose weight is below 2^-30 of the sum add less than the rest of the bound
            worst = np.where(seen & (w > 2.0 ** -30), e, 0.0).max(1, initial=0.0)[:, None]
            worst = worst + 2.0 ** -23 * np.where(some, np.abs(m), 0.0)
            err[q0:q1, h] = (2 * worst + 2.0 ** -20 + (2 * end + 64) * 2.0 ** -24) * (w @ np.abs(vh)) + step
    return out, err, seen_rows


class OnDevice:
    """Arrays on the device by name, freed together."""

    def __init__(self, dev, **arrays):
        self.dev, self.bufs = dev, {}
        for name, a in arrays.items():
            self.put(name, a)

    def put(self, name, a):
        a = np.ascontiguousarray(a)
        self.bufs[name] = (self.dev.to_device(a), a.dtype, a.shape)
        return self.ptr(name)

    def ptr(self, name):
        return self.bufs[name][0].ptr

    def get(self, name):
        b, dtype, shape = self.bufs[name]
        return b.to_host(dtype, int(np.prod(shape))).reshape(shape)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for b, _, _ in self.bufs.values():
            b.free()


def put_cache(d, cache):
    d.put("k", cache.k), d.put("v", cache.v), d.put("ks", cache.ks), d.put("vs", cache.vs)
    return sa.KvCache(k=d.ptr("k"), v=d.ptr("v"), k_scale=d.ptr("ks"), v_scale=d.ptr("vs"), n_pages=cache.n_pages,
                      n_head_kv=cache.n_kv, head_dim=cache.hd, block=cache.block)


def put_batch(d, table, q_start, kv_len, n_tok, max_q=None, max_kv=None):
    d.put("table", table.astype(np.int32)), d.put("q_start", np.asarray(q_start, np.int32))
    d.put("kv_len", np.asarray(kv_len, np.int32))
    n = np.diff(q_start)
    return sa.KvBatch(q_start=d.ptr("q_start"), kv_len=d.ptr("kv_len"), table=d.ptr("table"), n_req=table.shape[0],
                      max_blocks=table.shape[1], n_tok=n_tok, max_q=int(n.max()) if max_q is None else max_q,
                      max_kv=int(np.max(kv_len)) if max_kv is None else max_kv)


def requests(rng, lengths, adds, block, n_kv, hd, spare_blocks=2, scale=1.0):
    """A cache that holds `lengths` + `adds` tokens of each request at random
    pages, (table, q_start, kv_len). Table entries past a request's blocks are
    junk, pages of nobody have NaN scales."""
    ends = [n + a for n, a in zip(lengths, adds)]
    held = [blocks_of(e, block) for e in ends]
    n_pages = sum(held) + 3
    order = rng.permutation(n_pages)
    cache = Cache(rng, n_pages, n_kv, hd, block)
    junk = np.array([-1, n_pages, 2 ** 31 - 1, -2 ** 31, int(order[-1])])
    table = rng.choice(junk, (len(ends), max(held) + spare_blocks)).astype(np.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    used = order[:at]
    cache.ks[used] = np.exp(rng.normal(0, 1, (at, n_kv))).astype(np.float32) * np.float32(0.02 * scale)
    cache.vs[used] = np.exp(rng.normal(0, 2, (at, n_kv))).astype(np.float32) * np.float32(0.02)
    q_start = np.concatenate([[0], np.cumsum(adds)]).astype(np.int32)
    return cache, table, q_start, np.array(ends, np.int32)
