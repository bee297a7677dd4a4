// Attention over the paged 8-bit KV cache (kvcache.h), for the ragged batch of
// a step: single tokens and prompt rows alike.
//
//   s_ij  = softcap(kq_scale <q_i, k_j>) - slope_h |p_i - j|
//   out_i = sum_j softmax_j(s_ij) v_j     over the visible j
//
// in one pass over the keys with a running maximum m and total l per row
// (in log2 units). The rows of a request and KV head are its tokens times
// the G query heads of that KV head: row = token * G + head, so that a key
// row, converted once, serves all of them.
//
// The matrix cores multiply f16 pairs into f32. Codes are whole numbers up
// to 127 and exact in f16. The other operand is f32 and is split into two
// f16 numbers, x = hi + lo with 22 bits: each product runs twice, and the
// results keep f32's accuracy (a single f16 would leave 2^-11, 70 times the
// f32 rounding of the sums). Query rows are scaled by a power of two to
// [2^13, 2^14) first and the probabilities, times their value scale, by
// 2^14, so that neither half falls among the subnormal numbers.
//
// Scores are computed transposed, S^T = K Q^T: a lane then holds the scores
// of one row against 16 consecutive tokens, which all lie in one page (pages
// are multiples of 16), have one key scale and one value scale, and are the
// operand of out^T = V^T P^T as they lie: no transposition, no exchange.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "agent.h"
#include "kvcache.h"

namespace sihip {

typedef _Float16 ap_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 ap_h2 __attribute__((ext_vector_type(2)));
typedef float ap_f4 __attribute__((ext_vector_type(4)));
typedef float ap_f16 __attribute__((ext_vector_type(16)));

struct AttnPArgs {
    CacheArgs C;
    BatchArgs R;
    const float *q, *slopes;
    const int32_t *prefix;
    float *out;
    int64_t ldq, ldo;
    int n_req, G, window;
    bool out_vec;    // rows of out and their heads are 16-byte aligned
    float sign;      // of kq_scale: queries are multiplied by it,
    float scale2;    // |kq_scale| * log2 e, so that factors of scores are not negative
    float cap, cap_in;  // softcap * log2 e (0: none), 2 |kq_scale| / softcap * log2 e
    int n_tiles, n_split;
    float *part;     // [item][split][rows][hd + 2]: out^T sums, m, l
    uint32_t *cnt;   // [item]
};

constexpr float kApNone = -3.4e38f;  // running maximum before any key
constexpr float kLog2e = 1.44269504088896340736f;

// four codes -> four halves: 0x6400 | (byte ^ 0x80) is 1024 + 128 + code
__device__ inline void ap_cvt4(uint32_t x, ap_h2 &a, ap_h2 &b) {
    x ^= 0x80808080u;
    const ap_h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    a = __builtin_bit_cast(ap_h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - off;
    b = __builtin_bit_cast(ap_h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - off;
}

__device__ inline ap_h8 ap_cvt8(uint32_t x, uint32_t y) {
    union {
        ap_h8 v;
        ap_h2 h[4];
    } u;
    ap_cvt4(x, u.h[0], u.h[1]);
    ap_cvt4(y, u.h[2], u.h[3]);
    return u.v;
}

// x = hi + lo in f16 (x up to 2^14 in magnitude). The empty statement keeps
// x a number in a register: a product rounded straight to f16 would be another
// one than the rounded product's, now and then, and lo is taken from the
// latter.
__device__ inline void ap_split8(float *x, ap_h8 &hi, ap_h8 &lo) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        asm("" : "+v"(x[j]));
        hi[j] = (_Float16)x[j];
        lo[j] = (_Float16)(x[j] - (float)hi[j]);
    }
}

// p w = hi + lo in f16 (p w up to 2^14). lo is taken from the product before
// it is rounded; the empty statement makes the hi of the difference the one
// that is multiplied.
__device__ inline void ap_split8w(const float *p, float w, ap_h8 &hi, ap_h8 &lo) {
#pragma unroll
    for (int j = 0; j < 8; j++) hi[j] = (_Float16)(p[j] * w);
    asm("" : "+v"(hi));
#pragma unroll
    for (int j = 0; j < 8; j++) lo[j] = (_Float16)fmaf(p[j], w, -(float)hi[j]);
}

// What a block of rows of one request sees: positions p_lo .. p_hi of its
// first and last row, the keys [0, keys), of which the first `prefix` are
// visible to every row. In 64-key chunks: chunks [0, np) hold the prefix,
// [c0, c1) the rest; chunk u of n is u < np ? u : u - np + c0.
struct Sight {
    int p_lo, p_hi, keys, prefix, np, c0, n;
};

__device__ inline Sight ap_sight(const AttnPArgs &A, int r, const Span &s, int t0, int t1) {
    Sight g;
    g.p_lo = s.p0 + t0;
    g.p_hi = s.p0 + t1;
    g.keys = min(s.end, A.R.max_kv);
    g.prefix = A.prefix ? max(0, min(A.prefix[r], g.keys)) : 0;
    const int end = min(max(g.p_hi + 1, g.prefix), g.keys);
    const int start = A.window ? max(0, g.p_lo - A.window + 1) : 0;
    g.np = A.window ? (g.prefix + 63) / 64 : 0;
    g.c0 = max(start / 64, g.np);
    g.n = g.np + max(0, (end + 63) / 64 - g.c0);
    return g;
}

__device__ inline int ap_chunk(const Sight &g, int u) { return u < g.np ? u : u - g.np + g.c0; }

// whether every row of the block sees all 64 keys of chunk c
__device__ inline bool ap_whole(const AttnPArgs &A, const Sight &g, int c) {
    const int j0 = c * 64, j1 = j0 + 63;
    if (j1 >= g.keys) return false;
    return j1 < g.prefix || (j1 <= g.p_lo && (!A.window || j0 > g.p_hi - A.window));
}

__device__ inline bool ap_visible(const AttnPArgs &A, const Sight &g, int p, int j) {
    return j < g.keys && (j < g.prefix || (j <= p && (!A.window || j > p - A.window)));
}

// bits 0 .. n - 1 of 16
__device__ inline uint32_t ap_below(int n) { return (1u << max(0, min(n, 16))) - 1u; }

// the keys j0 .. j0 + 15 that the row at position p does not see, as bits
__device__ inline uint32_t ap_hidden(const AttnPArgs &A, const Sight &g, int p, int j0) {
    uint32_t see = ap_below(min(p + 1, g.keys) - j0);
    if (A.window) see &= ~ap_below(p + 1 - A.window - j0);
    return 0xffffu & ~(see | ap_below(g.prefix - j0));
}

// -inf where bit e is set
__device__ inline float ap_hide(float x, uint32_t hidden, int e) {
    const uint32_t h = (uint32_t)((int32_t)(hidden << (31 - e)) >> 31);
    return __builtin_bit_cast(float, (h & 0xff800000u) | (~h & __builtin_bit_cast(uint32_t, x)));
}

// cap tanh(s / cap), s and cap in log2 units, x2 = 2 s / cap * log2 e. tanh x =
// 1 - 2 / (e^2x + 1) is off by 2^-23 of 1, which near zero is much of a small
// score: there (|x| < 0.32) the series up to x^11, off by 2^-24 of the score.
__device__ inline float ap_capped(const AttnPArgs &A, float s, float x2) {
    const float e = __builtin_amdgcn_exp2f(x2);
    const float far = A.cap * (1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f));
    const float x = x2 * (0.5f / kLog2e), z = x * x;
    float y = fmaf(z, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    y = fmaf(z, y, -17.0f / 315.0f);
    y = fmaf(z, y, 2.0f / 15.0f);
    y = fmaf(z, y, -1.0f / 3.0f);
    const float near = fmaf(s * z, y, s);
    return z < 0.1f ? near : far;
}

// The score of a raw product: `f` is the factor to log2 units, fc the one of
// the tanh's argument where scores are capped.
__device__ inline float ap_score(const AttnPArgs &A, float raw, float f, float fc, float slope, int p, int j) {
    float s = raw * f;
    if (A.cap != 0.0f) s = ap_capped(A, s, raw * fc);
    return fmaf(-slope, fabsf((float)(p - j)), s);
}

// Power of two (as an exponent) by which a query row is multiplied.
__device__ inline int ap_row_exponent(float amax) {
    if (!(amax > 0.0f) || !(amax < INFINITY)) return 0;
    return max(-126, min(126, 13 - ilogbf(amax)));
}

// sums over total, 0 where no key was seen
__device__ inline float ap_quotient(float o, float l) { return l > 0.0f || l != l ? o / l : 0.0f; }

// four values in a row; wide: p is 16-byte aligned
__device__ inline void ap_put4(float *p, float a, float b, float c, float d, bool wide) {
    if (wide) {
        *(float4 *)p = float4{a, b, c, d};
    } else {
        p[0] = a;
        p[1] = b;
        p[2] = c;
        p[3] = d;
    }
}

__device__ inline void ap_store(float *p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The end of a row block whose keys were split over workgroups, after each
// has stored its sums (agent-scope stores; agent.h says what their order rests
// on): the last to arrive adds them up in the order of the splits, so the
// result does not depend on the order of arrival, and leaves the counter zero.
template <int ROWS, int THREADS>
__device__ inline void ap_join(const AttnPArgs &A, const Span &s, int h, int tile, int64_t item, int rows, int n_split) {
    __shared__ uint32_t last;
    const int tid = threadIdx.x, hd = A.C.hd, stride = ROWS * (hd + 2);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (tid == 0)
        last = __hip_atomic_fetch_add(A.cnt + item, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)n_split - 1;
    __syncthreads();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (!last) return;
    const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
        A.part + item * A.n_split * stride, (short)0, n_split * stride * 4, 0x00020000);
    for (int i = tid; i < rows * hd; i += THREADS) {
        const int c = i / hd, d = i % hd;
        float mm = kApNone, ll = 0.0f, oo = 0.0f;
        for (int k = 0; k < n_split; k++) {
            const uint32_t at = (uint32_t)(k * stride + c * (hd + 2)) * 4;
            const float mk = load_agent_f32(pr, at + hd * 4), lk = load_agent_f32(pr, at + hd * 4 + 4);
            const float vk = load_agent_f32(pr, at + d * 4);
            const float m2 = fmaxf(mm, mk), ea = __builtin_amdgcn_exp2f(mm - m2), eb = __builtin_amdgcn_exp2f(mk - m2);
            ll = fmaf(ll, ea, lk * eb);
            oo = fmaf(oo, ea, vk * eb);
            mm = m2;
        }
        const int rw = tile * ROWS + c;
        A.out[(s.q0 + rw / A.G) * A.ldo + (int64_t)(h * A.G + rw % A.G) * hd + d] = ap_quotient(oo, ll);
    }
    if (tid == 0) __hip_atomic_store(A.cnt + item, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- few rows ----------------------------------------------------------------------
//
// One workgroup: 16 rows of one request and KV head, one split of its
// chunks; the waves take chunks in turn and join through LDS at the end.
// Nothing is staged: a lane loads 16 bytes of a key row (key tile t, row m
// of the matrix operand is token 16 (m / 4) + 4 t + m % 4) and 16 tokens of a
// value row, converts them in registers and feeds the matrix cores.

constexpr int kApWaves = 4, kApRows = 16;

// hd rounded up to 64 NK dims
template <int NK>
__global__ __launch_bounds__(kApWaves * 64) void attnp_rows_kernel(AttnPArgs A) {
    constexpr int ND = NK * 4;  // 16-dim tiles
    __shared__ float o_lds[kApWaves][16][NK * 64 + 1];
    __shared__ float m_lds[kApWaves][16], l_lds[kApWaves][16];
    const int r = blockIdx.z, h = blockIdx.y;
    const int tile = blockIdx.x / A.n_split, split = blockIdx.x % A.n_split;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int hd = A.C.hd, shift = A.C.shift, B = 1 << shift;
    const Span s = request_span(A.R, r);
    const int n_rows = min(s.n, A.R.max_q) * A.G;
    if (tile * 16 >= n_rows) return;
    const int t0 = tile * 16 / A.G, t1 = min((tile * 16 + 15) / A.G, min(s.n, A.R.max_q) - 1);
    const Sight S = ap_sight(A, r, s, t0, t1);
    const int n_split = max(1, min(A.n_split, (S.n + kApWaves - 1) / kApWaves));
    if (split >= n_split) return;
    const int u0 = (int)((int64_t)S.n * split / n_split), u1 = (int)((int64_t)S.n * (split + 1) / n_split);

    // this lane's row
    const int row = min(tile * 16 + col, n_rows - 1);
    const int tok = row / A.G, head = h * A.G + row % A.G;
    const int p = s.p0 + tok;
    const float slope = A.slopes ? A.slopes[head] * kLog2e : 0.0f;
    const float *qrow = A.q + (s.q0 + tok) * A.ldq + (int64_t)head * hd;
    ap_h8 qh[NK][2], ql[NK][2];
    float amax = 0.0f;
    {
        float x[NK][2][8];
#pragma unroll
        for (int c = 0; c < NK; c++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int d = 64 * c + 16 * g + 8 * e + j;
                    x[c][e][j] = d < hd ? qrow[d] : 0.0f;
                    amax = fmaxf(amax, fabsf(x[c][e][j]));
                }
        amax = fmaxf(amax, __shfl_xor(amax, 16));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        const int e2 = ap_row_exponent(amax);
#pragma unroll
        for (int c = 0; c < NK; c++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[c][e][j] = ldexpf(x[c][e][j] * A.sign, e2);
                ap_split8(x[c][e], qh[c][e], ql[c][e]);
            }
        amax = ldexpf(1.0f, -e2);
    }
    const float f_row = amax * A.scale2, fc_row = amax * A.cap_in;

    float m = kApNone, l = 0.0f, ref = 0.0f;  // ref: power of two of the value scales
    ap_f4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = ap_f4{0, 0, 0, 0};
    const int32_t *table = A.R.table + (int64_t)r * A.R.max_blocks;
    const int64_t page_bytes = (int64_t)hd << shift;

    for (int u = u0 + wave; u < u1; u += kApWaves) {
        const int c = ap_chunk(S, u);
        // the pages of the 16-token segments: of this lane's key rows
        // (segment col / 4) and of its values and scores (segment g)
        auto page_of = [&](int seg, bool &ok) {
            const int j = c * 64 + seg * 16, b = j >> shift;
            const int pg = j < S.keys && b < A.R.max_blocks ? table[b] : -1;
            ok = pg >= 0 && pg < A.C.n_pages;
            return (int64_t)(ok ? pg : 0) * A.C.n_kv + h;
        };
        bool okk, ok;
        const int64_t pk = page_of(col >> 2, okk), pv = page_of(g, ok);
        const int koff = (c * 64 + (col >> 2) * 16) & (B - 1), voff = (c * 64 + g * 16) & (B - 1);
        const int8_t *kp = A.C.k + pk * page_bytes + (int64_t)(koff + (col & 3)) * hd;
        const int8_t *vp = A.C.v + pv * page_bytes + voff;
        uint4 kr[4][NK], vr[ND];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < NK; e++) {
                const int d = 64 * e + 16 * g;
                kr[t][e] = *(const uint4 *)(kp + 4 * t * hd + (d < hd ? d : 0));
            }
        const float ksc = A.C.ks[pv], vsc = A.C.vs[pv];
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const int dim = 16 * d + col;
            vr[d] = *(const uint4 *)(vp + ((int64_t)(dim < hd ? dim : 0) << shift));
        }
        ap_f4 sc[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            sc[t] = ap_f4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < NK; e++) {
                const ap_h8 a = ap_cvt8(kr[t][e].x, kr[t][e].y), b = ap_cvt8(kr[t][e].z, kr[t][e].w);
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[e][0], sc[t], 0, 0, 0);
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, qh[e][1], sc[t], 0, 0, 0);
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[e][0], sc[t], 0, 0, 0);
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, ql[e][1], sc[t], 0, 0, 0);
            }
        }
        // scores, in log2 units; tokens of this lane: j0 + 4 t + i
        const int j0 = c * 64 + g * 16;
        const float f = f_row * ksc, fc = fc_row * ksc;
        const bool mask = !ap_whole(A, S, c) || __any(!ok);
        float mx = kApNone;
        bool any_seen = false;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = j0 + 4 * t + i;
                float v = ap_score(A, sc[t][i], f, fc, slope, p, j);
                if (mask) {
                    const bool see = ok && ap_visible(A, S, p, j);
                    any_seen |= see;
                    v = see ? v : -INFINITY;
                }
                sc[t][i] = v;
                mx = fmaxf(mx, v);
            }
        const bool seen = ok && (!mask || any_seen);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        // the value scales' power of two: the largest so far. A segment that
        // this row does not see counts nothing, whatever its page holds.
        const float vs = seen ? vsc : 0.0f;
        float top = vs >= 0x1p-100f && vs < INFINITY ? ldexpf(1.0f, ilogbf(vs)) : 0x1p-100f;
        for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        const float ref2 = fmaxf(ref, top), m2 = fmaxf(m, mx);
        const float am = __builtin_amdgcn_exp2f(m - m2);
        const float ao = am * (ref / ref2);
        m = m2;
        ref = ref2;
        const float w = vs * (0x1p13f / ref);
        float sum = 0.0f;
        ap_h8 ph[2], pl[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float pr = __builtin_amdgcn_exp2f(sc[2 * e + (j >> 2)][j & 3] - m);
                sum += pr;
                x[j] = pr * w;
            }
            ap_split8(x, ph[e], pl[e]);
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        l = fmaf(l, am, sum);
#pragma unroll
        for (int d = 0; d < ND; d++) {
            if (16 * d >= hd) continue;
            const ap_h8 a = ap_cvt8(vr[d].x, vr[d].y), b = ap_cvt8(vr[d].z, vr[d].w);
            o[d] *= ao;
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[0], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, ph[1], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[0], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, pl[1], o[d], 0, 0, 0);
        }
    }

    // join the waves: all lanes of a column hold the same m and l
    const float back = ref * 0x1p-13f;
    if (g == 0) {
        m_lds[wave][col] = m;
        l_lds[wave][col] = l;
    }
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) o_lds[wave][col][16 * d + 4 * g + i] = o[d][i] * back;
    __syncthreads();
    const int rows = min(16, n_rows - tile * 16);
    const int64_t item = ((int64_t)r * A.C.n_kv + h) * A.n_tiles + tile;
    float *part = A.part + (item * A.n_split + split) * 16 * (hd + 2);
    for (int i = tid; i < rows * hd; i += kApWaves * 64) {
        const int c = i / hd, d = i % hd;
        float mm = kApNone;
#pragma unroll
        for (int w = 0; w < kApWaves; w++) mm = fmaxf(mm, m_lds[w][c]);
        float ll = 0.0f, oo = 0.0f;
#pragma unroll
        for (int w = 0; w < kApWaves; w++) {
            const float e = __builtin_amdgcn_exp2f(m_lds[w][c] - mm);
            ll = fmaf(l_lds[w][c], e, ll);
            oo = fmaf(o_lds[w][c][d], e, oo);
        }
        if (n_split == 1) {
            const int rw = tile * 16 + c;
            A.out[(s.q0 + rw / A.G) * A.ldo + (int64_t)(h * A.G + rw % A.G) * hd + d] = ap_quotient(oo, ll);
        } else {
            ap_store(part + c * (hd + 2) + d, oo);
            if (d == 0) {
                ap_store(part + c * (hd + 2) + hd, mm);
                ap_store(part + c * (hd + 2) + hd + 1, ll);
            }
        }
    }
    if (n_split == 1) return;

    ap_join<kApRows, kApWaves * 64>(A, s, h, tile, item, rows, n_split);
}

// ---- many rows ---------------------------------------------------------------------
//
// One workgroup: 128 rows of one request and KV head, 32 for each of its four
// waves, one split of its 64-key chunks. A chunk's codes are loaded as they
// lie, two chunks ahead, converted to f16 once for all waves and put into
// LDS, two chunks in turn with one barrier each: converting in every wave
// would cost as many vector instructions as the softmax. The 16-byte granules
// of a row are permuted by an exclusive or, so that 16 lanes that read the same
// column of 16 rows reach all 64 banks: by four bits of the row where a row
// is a multiple of 256 bytes, by three where it is an odd multiple of 128 and
// neighbouring rows lie in the two halves.
//
// A wave's 32x32 tile of S^T has its key rows in the order that gives lane
// (row c, half e) the scores of keys 32 u + 16 e + i in register i: row m of
// the operand is key 16 (m / 4 % 2) + 4 (m / 8) + m % 4.

// A row's maximum follows the scores when they pass it by 2^4, so that most
// chunks leave the sums alone: weights reach 2^4 and are held times 2^9.
constexpr float kApLate = 4.0f, kApUnit = 0x1p9f;

// the power of two below x (x is 0 or more), at least 2^-100
__device__ inline float ap_power(float x) {
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, fmaxf(x, 0x1p-100f)) & 0x7f800000u);
}

// the larger of lane i's and lane i + 32's
__device__ inline float ap_max_halves(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// hd rounded up to 16 NS dims
template <int NS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, NS <= 8 ? 2 : 1) void attnp_tiles_kernel(AttnPArgs A) {
    constexpr int kApTileRows = 32 * WAVES, kApTileThreads = 64 * WAVES;
    constexpr int ND = (NS + 1) / 2;             // 32-dim tiles of the output
    constexpr int KC = (2 * NS + 7) / 8 * 8;     // granules of a key row in LDS
    constexpr int NU = (64 * NS + kApTileThreads - 1) / kApTileThreads;  // 16-byte loads of a chunk, each
    __shared__ uint4 k_lds[2][64][KC];
    __shared__ uint4 v_lds[2][ND * 32][8];
    __shared__ float s_lds[2][8];
    const int h = blockIdx.x % A.C.n_kv, tile = A.n_tiles - 1 - blockIdx.x / A.C.n_kv, split = blockIdx.y, r = blockIdx.z;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int hd = A.C.hd, shift = A.C.shift, B = 1 << shift;
    const Span s = request_span(A.R, r);
    const int n_tok = min(s.n, A.R.max_q), n_rows = n_tok * A.G;
    if (tile * kApTileRows >= n_rows) return;
    const Sight S = ap_sight(A, r, s, tile * kApTileRows / A.G, min((tile * kApTileRows + kApTileRows - 1) / A.G, n_tok - 1));
    const int n_split = max(1, min(A.n_split, S.n));
    if (split >= n_split) return;
    const int u0 = (int)((int64_t)S.n * split / n_split), u1 = (int)((int64_t)S.n * (split + 1) / n_split);

    // the wave's rows and this lane's
    const int row0 = tile * kApTileRows + wave * 32;
    const bool idle = row0 >= n_rows;
    const int row = min(row0 + col, n_rows - 1), tok = row / A.G, head = h * A.G + row % A.G, p = s.p0 + tok;
    Sight W = S;
    W.p_lo = s.p0 + min(row0, n_rows - 1) / A.G;
    W.p_hi = s.p0 + min(row0 + 31, n_rows - 1) / A.G;
    const float slope = A.slopes ? A.slopes[head] * kLog2e : 0.0f;
    ap_h8 qh[NS], ql[NS];
    float f_row;
    {
        const float *qrow = A.q + (s.q0 + tok) * A.ldq + (int64_t)head * hd + 8 * half;
        float amax = 0.0f;
#pragma unroll
        for (int c = 0; c < NS; c++)
            if (16 * c < hd)
#pragma unroll
                for (int j = 0; j < 8; j++) amax = fmaxf(amax, fabsf(qrow[16 * c + j]));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        const int e2 = ap_row_exponent(amax);
#pragma unroll
        for (int c = 0; c < NS; c++) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = 16 * c < hd ? ldexpf(qrow[16 * c + j] * A.sign, e2) : 0.0f;
            ap_split8(x, qh[c], ql[c]);
        }
        f_row = ldexpf(1.0f, -e2);
    }
    const float fc_row = f_row * A.cap_in;
    f_row *= A.scale2;

    // loads without branches: what is not there is read from elsewhere in the
    // table or the page and replaced
    const int32_t *table = A.R.table + (int64_t)r * A.R.max_blocks;
    const int last_block = max(S.keys - 1, 0) >> shift, n_pages = (int)A.C.n_pages;
    auto page_of = [&](int j) {
        const int pg = table[min(j >> shift, last_block)];
        return j < S.keys && pg >= 0 && pg < n_pages ? pg : -1;
    };
    // this thread's parts of a chunk: 16 dims of a key, 16 keys of a dim. A
    // chunk starts at a multiple of 64, so a part's place in its page is the
    // thread's own and, in pages of more than 64, the chunk's.
    constexpr bool kWhole = 64 * NS % kApTileThreads == 0;
    uint4 kr[NU], vr[NU];
    int kpg[NU], vpg;
    float scale;  // of threads 0 .. 7: a key or value scale of segment tid % 4, -1 where it has no page
    auto unit = [&](int i) { return kWhole ? tid + kApTileThreads * i : min(tid + kApTileThreads * i, 64 * NS - 1); };
    const uint32_t head_bytes = (uint32_t)hd << shift, page_bytes = head_bytes * (uint32_t)A.C.n_kv;
    const int8_t *kb[NU], *vb[NU];
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int key = unit(i) / NS, d16 = unit(i) % NS, dim = unit(i) >> 2;
        kb[i] = A.C.k + h * (int64_t)head_bytes + (key & (B - 1)) * hd + (d16 * 16 < hd ? d16 * 16 : 0);
        vb[i] = A.C.v + h * (int64_t)head_bytes + ((dim < hd ? dim : 0) << shift) + ((16 * (tid & 3)) & (B - 1));
    }
    auto load_pages = [&](int u) {
        const int j0 = ap_chunk(S, u) * 64;
#pragma unroll
        for (int i = 0; i < NU; i++) kpg[i] = page_of(j0 + unit(i) / NS);
        vpg = page_of(j0 + 16 * (tid & 3));
    };
    auto load_chunk = [&](int u) {
        const int at = ap_chunk(S, u) * 64 & (B - 1);
        const uint64_t vp = (uint64_t)(uint32_t)max(vpg, 0) * page_bytes + at;
#pragma unroll
        for (int i = 0; i < NU; i++) {
            kr[i] = *(const uint4 *)(kb[i] + ((uint64_t)(uint32_t)max(kpg[i], 0) * page_bytes + at * hd));
            vr[i] = *(const uint4 *)(vb[i] + vp);
        }
        if (tid < 8) scale = vpg >= 0 ? (tid < 4 ? A.C.ks : A.C.vs)[(int64_t)vpg * A.C.n_kv + h] : -1.0f;
    };
    auto put_chunk = [&](int buf) {
        const uint4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int key = unit(i) / NS, d16 = unit(i) % NS, dim = unit(i) >> 2;
            // dims past hd meet zeros of q: they must be numbers
            const uint4 a = d16 * 16 < hd ? kr[i] : zero;
            const int kx = (key & 3) | ((key >> 2) & 4) | ((key << 1) & 8), x = KC % 16 ? kx >> 1 : kx;
            const int c = 2 * (tid & 3), y = (dim >> 1) & 7;
            k_lds[buf][key][(2 * d16) ^ x] = __builtin_bit_cast(uint4, ap_cvt8(a.x, a.y));
            k_lds[buf][key][(2 * d16 + 1) ^ x] = __builtin_bit_cast(uint4, ap_cvt8(a.z, a.w));
            v_lds[buf][dim][c ^ y] = __builtin_bit_cast(uint4, ap_cvt8(vr[i].x, vr[i].y));
            v_lds[buf][dim][(c + 1) ^ y] = __builtin_bit_cast(uint4, ap_cvt8(vr[i].z, vr[i].w));
        }
        if (tid < 8) s_lds[buf][tid] = scale;
    };

    ap_f16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    float m = kApNone, l = 0.0f, ref = 0.0f, over = 0.0f;
    if (u0 < u1) {
        load_pages(u0);
        load_chunk(u0);
        load_pages(min(u0 + 1, u1 - 1));
        put_chunk(0);
        load_chunk(min(u0 + 1, u1 - 1));
        load_pages(min(u0 + 2, u1 - 1));
    }
    for (int u = u0; u < u1; u++) {
        const int buf = (u - u0) & 1;
        __syncthreads();
        if (u + 1 < u1) {
            put_chunk(buf ^ 1);
            load_chunk(min(u + 2, u1 - 1));
            load_pages(min(u + 3, u1 - 1));
        }
        const int j0 = ap_chunk(S, u) * 64;
        // nothing here for this wave's rows
        if (idle || (j0 >= S.prefix && (j0 > W.p_hi || (A.window && j0 + 63 <= W.p_lo - A.window)))) continue;

        const bool whole = ap_whole(A, W, j0 >> 6);
        const int key = 16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3);
        const int x = KC % 16 ? (col >> 1) & 7 : col & 15, y = (col >> 1) & 7;
#pragma unroll 1
        for (int i = 0; i < 2; i++) {
            const uint4 *kl = k_lds[buf][32 * i + key];
            ap_f16 sc;
#pragma unroll
            for (int e = 0; e < 16; e++) sc[e] = 0.0f;
#pragma unroll
            for (int c = 0; c < NS; c++) {
                const ap_h8 a = __builtin_bit_cast(ap_h8, kl[(2 * c + half) ^ x]);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[c], sc, 0, 0, 0);
            }
            // scores in log2 units are sc * f; the factor is kept above zero, so
            // that it leaves -inf as it is, and is a number where no key is seen
            const float ksc = s_lds[buf][2 * i + half];
            float vsc = s_lds[buf][4 + 2 * i + half], f = fmaxf(f_row * ksc, 0x1p-120f);
            if (A.cap != 0.0f) {
                const float fc = fc_row * ksc;
#pragma unroll
                for (int e = 0; e < 16; e++) sc[e] = ap_capped(A, sc[e] * f, sc[e] * fc);
                f = 1.0f;
            }
            const int j1 = j0 + 32 * i + 16 * half;
            if (A.slopes) {
                const float far = (float)(j1 - p), base = slope * far;
                if (j0 + 63 <= W.p_lo) {  // no key behind a row's own
#pragma unroll
                    for (int e = 0; e < 16; e++) sc[e] = fmaf(sc[e], f, fmaf(slope, (float)e, base));
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) sc[e] = fmaf(sc[e], f, -slope * fabsf(far + (float)e));
                }
                f = 1.0f;
            }
            if (!whole || __any(vsc < 0.0f)) {
                const uint32_t hidden = vsc < 0.0f ? 0xffffu : ap_hidden(A, S, p, j1);
#pragma unroll
                for (int e = 0; e < 16; e++) sc[e] = ap_hide(sc[e], hidden, e);
                vsc = hidden != 0xffffu ? vsc : 0.0f;
            }
            float mx = sc[0];
#pragma unroll
            for (int e = 1; e < 16; e++) mx = fmaxf(mx, sc[e]);
            mx = ap_max_halves(mx * f);
            const float top = ap_max_halves(ap_power(vsc));
            if (__any(mx > m + kApLate || top > ref)) {
                const float m2 = fmaxf(m, mx), r2 = fmaxf(ref, top), am = __builtin_amdgcn_exp2f(m - m2), ao = am * (ref / r2);
                l *= am;
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= ao;
                m = m2;
                ref = r2;
                over = kApUnit / ref;
            }
            const float w = vsc * over;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                ap_h8 ph, pl;
                float pr[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    pr[j] = __builtin_amdgcn_exp2f(fmaf(sc[8 * e + j], f, -m));
                    l += pr[j];
                }
                ap_split8w(pr, w, ph, pl);
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    const ap_h8 a = __builtin_bit_cast(ap_h8, v_lds[buf][32 * d + col][(4 * i + 2 * half + e) ^ y]);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph, o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl, o[d], 0, 0, 0);
                }
            }
        }
    }
    l += __shfl_xor(l, 32);

    const int64_t item = ((int64_t)r * A.C.n_kv + h) * A.n_tiles + tile;
    const int rows = min(kApTileRows, n_rows - tile * kApTileRows);
    const float back = ref * (1.0f / kApUnit);
    if (row0 + col < n_rows) {
        // four dims in a row a register group: 32 d + 8 a + 4 half ..
        if (n_split == 1) {
            float *to = A.out + (s.q0 + tok) * A.ldo + (int64_t)head * hd + 4 * half;
            const float z = l > 0.0f || l != l ? back / l : 0.0f;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    if (32 * d + 8 * a < hd) ap_put4(to + 32 * d + 8 * a, o[d][4 * a] * z, o[d][4 * a + 1] * z,
                                o[d][4 * a + 2] * z, o[d][4 * a + 3] * z, A.out_vec);
        } else {
            float *to = A.part + ((item * A.n_split + split) * kApTileRows + wave * 32 + col) * (hd + 2);
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    if (32 * d + 8 * a < hd)
#pragma unroll
                        for (int b = 0; b < 4; b++) ap_store(to + 32 * d + 8 * a + 4 * half + b, o[d][4 * a + b] * back);
            if (half == 0) {
                ap_store(to + hd, m);
                ap_store(to + hd + 1, l);
            }
        }
    }
    if (n_split > 1) ap_join<kApTileRows, kApTileThreads>(A, s, h, tile, item, rows, n_split);
}

}  // namespace sihip
