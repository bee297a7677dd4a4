"""Attention over the paged 8-bit KV cache in 64 bits, with an error bound for
each row and head by itself, over the keys that the row sees (test
infrastructure; the cache and the device side are kv_oracle's).

For key j of a row, s_j its score and w_j its softmax weight:

d_j, what its exponent may be off by (absolute, natural units):
  2 hd 2^-24 sum |q k_j| (the f32 sum of 2 hd products), 2^-22 of the same (the
  split of q into two f16 halves) and 2^-38 max|q| sum |k_j| (a half that is
  subnormal: rows are scaled to [2^13, 2^14), half a step there is 2^-25), all
  times kq_scale; 2^-21 |s_j| for a handful of f32 roundings of the factors;
  where scores are capped no more than twice the cap of that (tanh is not
  steeper than 1 and within 1), and 2^-21 of the cap for the tanh, or of 4
  |s_j| if that is less (below 0.32 of the cap it is a series); 2^-23 of the bias; and 2^-24 (|s_j - s_max| + 8) for the
  rounding of the exponent that is taken (the running maximum is at most 4
  late and rounded up to the next integer, in log2 units).
r, what its weight may be off by besides, relative: 2^-20 for the exponential,
  its split into halves and the factors of joined sums, and 2^-24 for each of
  the 2 n + 64 additions of an output's chain.
u, absolute, before the quotient: a weight times its value scale is held in f16
  halves in units of 2^-9 of a power of two that is at most the largest of them
  in the row, so the lower half is off by at most half of 2^-24 there: 2^-34
  max_j w_j vs_j, and no less than 2^-134 (the power of two is kept above
  2^-100); the power of two is kept above 2^-104 of the value scales too, and
  weights below 2^-126 of the largest count as zero: 2^-126 max_j vs_j. Each
  times codes up to 128, for each key.

With e^d - 1 <= 2 d for d <= 1, the sums are off by
  sum_j w_j (2 d_j + r) |v_j| + 128 n u   and   sum_j w_j (2 d_j + r),
and their quotient by the first and the second times sum_j w_j |v_j|.
"""
import numpy as np


def attention(cache, table, q_start, kv_len, q, kq_scale, cap=0.0, slopes=None, prefix=None, window=0):
    """(out, error, size, seen): out and its error bound [token, head, dim],
    size = sum_j w_j |v_j| likewise, and which rows belong to a request."""
    T, H, hd = q.shape
    G = H // cache.n_kv
    out, err, size = np.zeros((3, T, H, hd))
    rows = np.zeros(T, bool)
    for r, end in enumerate(int(x) for x in kv_len):
        q0, q1 = int(q_start[r]), int(q_start[r + 1])
        if q1 <= q0:
            continue
        rows[q0:q1] = True
        k, v = cache.rows(table[r], end)
        at = np.arange(end)
        vs = cache.vs[table[r, at // cache.block]].astype(np.float64)  # [position, KV head]
        p = np.arange(end - (q1 - q0), end)[:, None]
        seen = at[None, :] <= p
        if window:
            seen &= at[None, :] > p - window
        if prefix is not None:
            seen |= at[None, :] < int(prefix[r])
        n = seen.sum(1, keepdims=True)
        for h in range(H):
            x = q[q0:q1, h].astype(np.float64)
            # keys that no row sees may stand for anything
            some = seen.any(0)
            kh, vh = (np.where(some[:, None], y[h // G], 0.0) for y in (k, v))
            scale = np.where(some, vs[:, h // G], 0.0)
            s = kq_scale * x @ kh.T
            d = ((2 * hd * 2.0 ** -24 + 2.0 ** -22) * (np.abs(x) @ np.abs(kh).T)
                 + 2.0 ** -38 * np.abs(x).max(1, keepdims=True) * np.abs(kh).sum(1)) * abs(kq_scale) + 2.0 ** -21 * np.abs(s)
            if cap:
                with np.errstate(over="ignore"):
                    d, s = np.minimum(d, 2 * cap) + 2.0 ** -21 * np.minimum(cap, 4 * np.abs(s)), cap * np.tanh(s / cap)
            if slopes is not None:
                bias = float(slopes[h]) * np.abs(p - at)
                s = s - bias
                d += 2.0 ** -23 * bias
            top = np.max(s, 1, keepdims=True, where=seen, initial=-np.inf)
            away = np.where(seen, s - np.where(n > 0, top, 0.0), -np.inf)
            w = np.exp(away)
            l = w.sum(1, keepdims=True)
            w = np.divide(w, l, out=np.zeros_like(w), where=l > 0)
            d = np.where(seen, d + 2.0 ** -24 * (np.where(seen, np.abs(away), 0.0) + 8), 0.0)
            assert d.max(initial=0.0, where=w > 0) <= 1.0
            wd = w * (2 * d + 2.0 ** -20 + (2 * n + 64) * 2.0 ** -24)
            most = np.where(seen, scale, 0.0).max(1, keepdims=True, initial=0.0)
            u = np.maximum(2.0 ** -34 * (w * scale).max(1, keepdims=True, initial=0.0), 2.0 ** -134) + 2.0 ** -126 * most
            out[q0:q1, h] = w @ vh
            size[q0:q1, h] = w @ np.abs(vh)
            err[q0:q1, h] = wd @ np.abs(vh) + 128 * n * u + wd.sum(1, keepdims=True) * size[q0:q1, h]
    return out, err, size, rows


def check(got, cache, table, q_start, kv_len, q, kq_scale, **o):
    """got [token, head, dim] against the definition, and the bound against a
    result of zeros: it has to refuse one for every row and head whose values
    do not cancel."""
    want, err, size, rows = attention(cache, table, q_start, kv_len, q, kq_scale, **o)
    alive = np.abs(want).max(2) > 0.05 * size.max(2)
    assert alive.any() and ((np.abs(want) > err).any(2) | ~alive).all(), "the bound would pass zeros"
    off = np.abs(got.astype(np.float64) - want)
    bad = (~(off <= err)).any(2) & rows[:, None]
    assert not bad.any(), f"rows and heads {np.argwhere(bad)[:6].tolist()}: off by up to {np.nanmax(off[rows] / (err[rows] + 1e-300)):.3g} bounds"
    return want
