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
// [2^13, 2^14) first; weights times their value scale by one that puts the
// largest such product of the row so far into [2^9, 2^13) (Running): a page of
// large values that the row hardly looks at takes no bits from the others. What
// the lower halves lose as subnormal numbers is below 2^-34 of that product a
// key, and 2^-38 of a query row's largest value. Results differ from 64 bits
// by 2 to 7 10^-7 of their norm.
//
// Scores are computed transposed, S^T = K Q^T: a lane then holds the scores
// of one row against 16 consecutive tokens, which all lie in one page (pages
// are multiples of 16), have one key scale and one value scale, and are the
// operand of out^T = V^T P^T as they lie: no transposition, no exchange.
#pragma once

#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

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
    bool q_vec, out_vec;  // rows of q or out and their heads are 16-byte aligned
    float sign;      // of kq_scale: queries are multiplied by it,
    float scale2;    // |kq_scale| * log2 e, so that factors of scores are not negative
    float cap, cap_in;  // softcap * log2 e (0: none), 2 |kq_scale| / softcap * log2 e
    int n_tiles;     // most row blocks of a request
    int ranks;       // most row blocks' worth of keys before a request's new ones
    int n_split, per_split;  // most splits of a row block's keys, least chunks of one
    int whole;       // chunks that are not split
    int slots;       // placed 16-row blocks: workgroups that share the chunks of all
    int chunk;       // log2 of the keys of a chunk
    int placed;      // 1: the grid is a list made on the device (ap_place, ap_deal)
    int least, most; // rows of the requests that are in it
    float *part;     // [piece][hd / 4 + 1][rows] of four: sums by dims, then m, l
    uint32_t *cnt;   // 16-row blocks: pieces that have arrived, zero between launches
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

// eight values of a query row; wide: rows of q and their heads are 16-byte aligned
__device__ inline void ap_load8(const float *q, bool wide, float *x) {
    if (wide) {
        const float4 a = ((const float4 *)q)[0], b = ((const float4 *)q)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = q[j];
    }
}

// What a block of rows of one request sees: positions p_lo .. p_hi of its
// first and last row, the keys [0, keys), of which the first `prefix` are
// visible to every row. In chunks: [0, np) hold the prefix, [c0, c1) the rest;
// chunk u of n is u < np ? u : u - np + c0.
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
    // (keys come up to 2^31 - 16: rounded up to whole chunks without a sign)
    auto chunks = [&](int keys) { return (int)(((uint32_t)keys + (1u << A.chunk) - 1) >> A.chunk); };
    g.np = A.window ? chunks(g.prefix) : 0;
    g.c0 = max(start >> A.chunk, g.np);
    g.n = g.np + max(0, chunks(end) - g.c0);
    return g;
}

__device__ inline int ap_chunk(const Sight &g, int u) { return u < g.np ? u : u - g.np + g.c0; }

// whether every row of the block sees the n keys from j0 on
__device__ inline bool ap_whole(const AttnPArgs &A, const Sight &g, int j0, int n) {
    const int j1 = j0 + (n - 1);  // (j0 + n can be 2^31)
    if (j1 >= g.keys) return false;
    return j1 < g.prefix || (j1 <= g.p_lo && (!A.window || j0 > g.p_hi - A.window));
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

// Splits of a row block with n chunks, in pieces of `per`.
__device__ inline int ap_splits(const AttnPArgs &A, int n, int per) {
    return n <= max(per, A.whole) ? 1 : min(A.n_split, (n + per - 1) / per);
}

// Sums, maxima and totals of a piece (a row block's split)
__device__ inline float4 *ap_part(const AttnPArgs &A, int64_t piece, int rows) {
    return (float4 *)A.part + piece * (A.C.hd / 4 + 1) * rows;
}

// Adds up to 16 pieces' totals (ml: maximum, total) and sums to those of the
// pieces before them.
__device__ inline void ap_add16(int n, const float4 *ml, const float4 *v, float &m, float &l, float4 &o) {
    float m2 = m;
#pragma unroll
    for (int k = 0; k < 16; k++) m2 = fmaxf(m2, ml[k].x);
    const float a = __builtin_amdgcn_exp2f(m - m2);
    l *= a;
    o = float4{o.x * a, o.y * a, o.z * a, o.w * a};
    m = m2;
#pragma unroll
    for (int k = 0; k < 16; k++) {
        const float e = k < n ? __builtin_amdgcn_exp2f(ml[k].x - m) : 0.0f;
        l = fmaf(ml[k].y, e, l);
        o = float4{fmaf(v[k].x, e, o.x), fmaf(v[k].y, e, o.y), fmaf(v[k].z, e, o.z), fmaf(v[k].w, e, o.w)};
    }
}

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

// the largest of lanes i, i + 16, i + 32 and i + 48
__device__ inline float ap_max_quarters(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, ap_max_halves(x));
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// The state of a row's softmax in a wave, in log2 units: weights are 2^(s - m),
// l is their sum, and the sums of weights times values are held in units of
// ref / 2^9. m follows the scores when they pass it by 4, and ref the products of
// weight and value scale when they pass it 16 times, so that most chunks leave
// the sums alone; what is multiplied stays below 2^14. m is a whole number and
// ref a power of two: both move without a rounding. ref goes down with m, so
// that it never is above the largest product of the row's keys so far, but
// for two floors: 2^-100, and 2^-104 of the value scales (the quotient of a
// scale and ref is to be a number; weights below 2^-126 are zero anyway).
constexpr float kApLate = 4.0f, kApUnit = 0x1p9f, kApLeast = 0x1p-100f;

struct Running {
    float m = kApNone, l = 0.0f, ref = 0.0f, over = 0.0f;  // over = kApUnit / ref

    // largest weight of a lane's keys (raw: their largest score is raw * f) times their value scale
    __device__ float most(float raw, float f, float vs) const {
        return vs * fmaxf(__builtin_amdgcn_exp2f(fmaf(raw, f, -m)), kApLeast);
    }
    // whether a lane's largest score, or that product, asks for a move of the row's
    __device__ bool late(float mx, float most) const { return mx > m + kApLate || most > 16.0f * ref; }
    // to a new maximum; returns the power of two that it takes from the weights so far
    __device__ float raise(float mx) {
        const float m2 = fmaxf(m, ceilf(mx)), am = ldexpf(1.0f, (int)fmaxf(m - m2, -256.0f));
        m = m2;
        l *= am;
        return am;
    }
    // the reference, for `most` under the new maximum; returns the factor of the sums so far
    __device__ float refer(float am, float most) {
        const float kept = ref * am;
        ref = fmaxf(kept, ap_power(most));
        over = kApUnit / ref;
        return kept / ref;
    }
};

// ---- few rows ----------------------------------------------------------------------
//
// One workgroup: 16 rows of one request and KV head, one split of its
// chunks; its waves take chunks in turn and join through LDS at the end.
// Nothing is staged: a lane loads 16 bytes of a key row and 4 TT tokens of a
// value row, converts them in registers and feeds the matrix cores. A chunk is
// TT tiles of 16 keys: row m of key tile t is token 4 TT (m / 4) + 4 t + m % 4,
// so that a lane's scores are of 4 TT tokens in a row. The next chunk's keys
// are loaded once this one's are converted, its values after this one's:
// each has half an iteration to arrive, and two waves of a SIMD keep the memory
// busy. (Wide heads take half the keys a chunk, so that two waves fit.)
//
// Single tokens are bound by memory, or by the chain of dependent loads when
// short (32 heads of 128 on 8): 600 keys 10.8 us, of which a launch with nothing
// to do takes 3.5; 131072 keys 55 us, 268 MB at 4.9 TB/s; 64 requests of up to
// 8192 keys, 408 MB, 91 us, 4.5 TB/s (a read of as much that does nothing else
// 5.4 to 5.9, a copy 4.8). Prompts of up to 1500 rows by the vector
// instructions between the products: 512 rows 24 us.

constexpr int kApRows = 16;
constexpr int kPlaceRegs = 4;  // requests a lane keeps in ap_deal and ap_place

// The pieces of a ragged batch. The host knows bounds on the lengths only, so
// the device deals: all chunks of all row blocks over the slots give the length
// of a piece, a row block has as many as it needs, and the grid, slots plus row
// blocks, holds them all. Every wave does the same sums over the requests, 64 at
// a time. (Grids of the longest request's splits for everybody started
// workgroups without work, 4 us each.)
struct Deal {
    int per;                 // chunks of a piece
    Span s[kPlaceRegs];      // of request lane + 64 k: its tokens,
    int n[kPlaceRegs];       // chunks,
    int last[kPlaceRegs];    // and the pieces up to and with it

    __device__ int splits(const AttnPArgs &A, int n) const { return n <= max(per, A.whole) ? 1 : (n + per - 1) / per; }
};

// x of this lane and all before it
template <class T>
__device__ inline T ap_scan(T x) {
    static_assert(sizeof(T) == 4, "one register");
    auto from = [&](auto ctrl, int rows) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, false) & rows);
    };
    const int lane = threadIdx.x & 63, in_row = lane & 15;
    // shifts by 1, 2, 4 and 8 within rows of 16, then lanes 15 and 31 to the rows behind them
    x += from(std::integral_constant<int, 0x111>(), in_row >= 1 ? -1 : 0);
    x += from(std::integral_constant<int, 0x112>(), in_row >= 2 ? -1 : 0);
    x += from(std::integral_constant<int, 0x114>(), in_row >= 4 ? -1 : 0);
    x += from(std::integral_constant<int, 0x118>(), in_row >= 8 ? -1 : 0);
    x += from(std::integral_constant<int, 0x142>(), lane & 16 ? -1 : 0);
    x += from(std::integral_constant<int, 0x143>(), lane & 32 ? -1 : 0);
    return x;
}

__device__ inline Deal ap_deal(const AttnPArgs &A) {
    const int lane = threadIdx.x & 63;
    Deal D;
    int tiles[kPlaceRegs];
    float all = 0.0f;
#pragma unroll
    for (int k = 0; k < kPlaceRegs; k++) {
        const int r = lane + 64 * k;
        D.n[k] = tiles[k] = 0;
        D.s[k] = Span{0, 0, 0, 0};
        if (64 * k >= A.n_req) continue;  // (of the whole wave)
        if (r < A.n_req) {
            D.s[k] = request_span(A.R, r);
            const int n = min(D.s[k].n, A.R.max_q);
            if (n > 0 && n * A.G <= A.most) {
                tiles[k] = (n * A.G + kApRows - 1) / kApRows;
                D.n[k] = ap_sight(A, r, D.s[k], 0, n - 1).n;
            }
        }
        all += (float)tiles[k] * (float)A.C.n_kv * (float)D.n[k];
    }
    // rounded up by more than the sum can be off: a piece too long by that is
    // harmless, one too short would make more pieces than the grid has
    all = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ap_scan(all)), 63));
    D.per = max(A.per_split, (int)fminf(ceilf(all * 1.0001f / (float)A.slots), 0x1p30f));
    int before = 0;
#pragma unroll
    for (int k = 0; k < kPlaceRegs; k++) {
        D.last[k] = before;
        if (64 * k >= A.n_req) continue;
        D.last[k] += ap_scan(tiles[k] * A.C.n_kv * D.splits(A, D.n[k]));
        before = __builtin_amdgcn_readlane(D.last[k], 63);
    }
    return D;
}

// pieces before request r's, its chunks and its tokens
__device__ inline int ap_dealt(const Deal &D, int r, int &n, Span &s) {
    int before = 0;
#pragma unroll
    for (int k = 0; k < kPlaceRegs; k++) {
        if (r >= 64 * k && r < 64 * k + 64) {
            const int l = r - 64 * k;
            n = __builtin_amdgcn_readlane(D.n[k], l);
            s.q0 = __builtin_amdgcn_readlane((int)D.s[k].q0, l);  // (a row of at most 2^31)
            s.n = __builtin_amdgcn_readlane(D.s[k].n, l);
            s.p0 = __builtin_amdgcn_readlane(D.s[k].p0, l);
            s.end = __builtin_amdgcn_readlane(D.s[k].end, l);
            if (l > 0) before = __builtin_amdgcn_readlane(D.last[k], l - 1);
        } else if (r >= 64 * k + 64) {
            before = __builtin_amdgcn_readlane(D.last[k], 63);
        }
    }
    return before;
}

// the request that piece i belongs to, or -1
__device__ inline int ap_dealt_to(const Deal &D, int i) {
    int r = -1;
#pragma unroll
    for (int k = kPlaceRegs - 1; k >= 0; k--) {
        const uint64_t past = __ballot(D.last[k] > i);
        if (past) r = 64 * k + __ffsll((unsigned long long)past) - 1;
    }
    return r;
}

// four values at agent scope (agent.h)
__device__ inline void ap_store4(__amdgpu_buffer_rsrc_t r, uint32_t at, float4 v) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), r, (int)(at * 16), 0, 16);
}
__device__ inline float4 ap_fetch4(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    return __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(at * 16), 0, 16));
}
__device__ inline __amdgpu_buffer_rsrc_t ap_pieces(const AttnPArgs &A, int64_t piece, int n) {
    return __builtin_amdgcn_make_buffer_rsrc(ap_part(A, piece, kApRows), (short)0, n * (A.C.hd / 4 + 1) * kApRows * 16, 0x00020000);
}

// The end of a 16-row block whose keys were split over n pieces, after each
// workgroup has stored its own at agent scope (agent.h says what the order
// rests on): the last to arrive adds them up in the order of the splits, so
// that the result does not depend on the order of arrival, and leaves the counter
// zero. (A second launch took 10 to 20 us: most of its workgroups had nothing to
// join, and each had to find that out.)
template <int THREADS>
__device__ inline void ap_join_rows(const AttnPArgs &A, const Span &s, int h, int tile, int rows, int64_t first, int n) {
    __shared__ uint32_t last;
    const int tid = threadIdx.x, hd = A.C.hd;
    uint32_t *cnt = A.cnt + first;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (tid == 0) last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)n - 1;
    __syncthreads();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (!last) return;
    const __amdgpu_buffer_rsrc_t part = ap_pieces(A, first, n);
    const uint32_t step = (hd / 4 + 1) * kApRows;
    for (int i = tid; i < rows * (hd / 4); i += THREADS) {
        const int c = i % rows, d4 = i / rows;
        float m = kApNone, l = 0.0f;
        float4 o = {0, 0, 0, 0};
        for (int k0 = 0; k0 < n; k0 += 16) {
            float4 ml[16], v[16];
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const uint32_t at = min(k0 + k, n - 1) * step + c;
                ml[k] = ap_fetch4(part, at + hd / 4 * kApRows);
                v[k] = ap_fetch4(part, at + d4 * kApRows);
            }
            ap_add16(n - k0, ml, v, m, l, o);
        }
        const int rw = tile * kApRows + c;
        ap_put4(A.out + (s.q0 + rw / A.G) * A.ldo + (int64_t)(h * A.G + rw % A.G) * hd + 4 * d4, ap_quotient(o.x, l),
                ap_quotient(o.y, l), ap_quotient(o.z, l), ap_quotient(o.w, l), A.out_vec);
    }
    if (tid == 0) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// hd rounded up to 64 NK dims
template <int NK, int TT, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void attnp_rows_kernel(AttnPArgs A) {
    constexpr int ND = NK * 4;  // 16-dim tiles
    constexpr int CH = 16 * TT, SEG = 4 * TT;
    constexpr uint32_t kAll = (1u << SEG) - 1;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int hd = A.C.hd, shift = A.C.shift, B = 1 << shift;
    int r = blockIdx.z, h = blockIdx.y, tile, split, per = A.per_split;
    int64_t piece;
    Span s;
    if (A.placed) {
        const Deal D = ap_deal(A);
        const int i = blockIdx.x;
        r = ap_dealt_to(D, i);
        if (r < 0) return;
        int n;
        const int before = ap_dealt(D, r, n, s), parts = D.splits(A, n);
        split = (i - before) % parts;
        h = (i - before) / parts % A.C.n_kv;
        tile = (i - before) / parts / A.C.n_kv;
        per = D.per;
        piece = i;
        // (spans that overlap are more than the grid was made for: what a block
        // cannot join in it, it does not begin)
        if (i < split || i - split + parts > (int)gridDim.x) return;
    } else {
        s = request_span(A.R, r);
        // workgroups go to the eight XCDs in turn, and of a ragged batch only the
        // low splits have work: turned by request and head they reach all XCDs
        tile = blockIdx.x / A.n_split;
        split = (blockIdx.x % A.n_split + h + r) % A.n_split;
        piece = (((int64_t)r * A.n_tiles + tile) * A.C.n_kv + h) * A.n_split + split;
    }
    const int32_t *table = A.R.table + (int64_t)r * A.R.max_blocks;
    const int n_tok = min(s.n, A.R.max_q), n_rows = n_tok * A.G;
    if (tile * 16 >= n_rows) return;
    const int t0 = tile * 16 / A.G, t1 = min((tile * 16 + 15) / A.G, n_tok - 1);
    const Sight S = ap_sight(A, r, s, t0, t1);
    const int n_split = ap_splits(A, S.n, per);
    if (split >= n_split) return;
    const int u0 = (int)((int64_t)S.n * split / n_split), u1 = (int)((int64_t)S.n * (split + 1) / n_split);

    // pages of this lane's key rows, and of its values and scores
    const int last_block = max(S.keys - 1, 0) >> shift, n_pages = (int)A.C.n_pages;
    auto page_of = [&](int u, int seg) {
        const int j = ap_chunk(S, u) * CH + seg * SEG, pg = table[min(j >> shift, last_block)];
        return j < S.keys && pg >= 0 && pg < n_pages ? pg : -1;
    };
    int u = u0 + wave, pk = 0, pv = 0;
    if (u < u1) {
        pk = page_of(u, col >> 2);
        pv = page_of(u, g);
    }

    // this lane's row
    const int row = min(tile * 16 + col, n_rows - 1);
    const int tok = row / A.G, head = h * A.G + row % A.G;
    const int p = s.p0 + tok;
    const float slope = A.slopes ? A.slopes[head] * kLog2e : 0.0f;
    const float *qrow = A.q + (s.q0 + tok) * A.ldq + (int64_t)head * hd;
    float x[NK][2][8];
#pragma unroll
    for (int c = 0; c < NK; c++)
#pragma unroll
        for (int e = 0; e < 2; e++) ap_load8(qrow + (64 * c + 16 * g < hd ? 64 * c + 16 * g : 0) + 8 * e, A.q_vec, x[c][e]);

    // a chunk starts at a multiple of its length: a lane's place in a page is
    // its own and, in longer pages, the chunk's
    const uint32_t head_bytes = (uint32_t)hd << shift, page_bytes = head_bytes * (uint32_t)A.C.n_kv;
    const int8_t *kb = A.C.k + h * (int64_t)head_bytes + (((col >> 2) * SEG & (B - 1)) + (col & 3)) * hd;
    const int8_t *vb = A.C.v + h * (int64_t)head_bytes + (col << shift) + (g * SEG & (B - 1));
    int dim[NK];  // this lane's dims of a key row; those past hd meet zeros of q
#pragma unroll
    for (int e = 0; e < NK; e++) dim[e] = 64 * e + 16 * g < hd ? 64 * e + 16 * g : 0;
    uint4 kr[TT][NK];
    uint32_t vr[ND][TT];
    float ksc = 0.0f, vsc = 0.0f;
    auto load_keys = [&](int u) {
        const int8_t *kp = kb + ((uint64_t)(uint32_t)max(pk, 0) * page_bytes + (ap_chunk(S, u) * CH & (B - 1)) * hd);
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int e = 0; e < NK; e++) kr[t][e] = *(const uint4 *)(kp + (4 * t * hd + dim[e]));
        const int64_t at = (int64_t)max(pv, 0) * A.C.n_kv + h;
        ksc = A.C.ks[at];
        vsc = pv < 0 ? -1.0f : A.C.vs[at];  // -1: no page
    };
    auto load_values = [&](int u, int page) {
        const int8_t *vp = vb + ((uint64_t)(uint32_t)max(page, 0) * page_bytes + (ap_chunk(S, u) * CH & (B - 1)));
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const int8_t *at = vp + (min(16 * d, hd - 16) << shift);
            if constexpr (TT == 4) {
                const uint4 v = *(const uint4 *)at;
                vr[d][0] = v.x, vr[d][1] = v.y, vr[d][2] = v.z, vr[d][3] = v.w;
            } else {
                const uint2 v = *(const uint2 *)at;
                vr[d][0] = v.x, vr[d][1] = v.y;
            }
        }
    };
    if (u < u1) {
        load_keys(u);
        load_values(u, pv);
        const int next = min(u + WAVES, u1 - 1);
        pk = page_of(next, col >> 2);
        pv = page_of(next, g);
    }

    // the query, while the first keys are on their way
    ap_h8 qh[NK][2], ql[NK][2];
    float f_row, fc_row;
    {
        float amax = 0.0f;
#pragma unroll
        for (int c = 0; c < NK; c++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[c][e][j] = 64 * c + 16 * g < hd ? x[c][e][j] * A.sign : 0.0f;
                    amax = fmaxf(amax, fabsf(x[c][e][j]));
                }
        const int e2 = ap_row_exponent(ap_max_quarters(amax));
#pragma unroll
        for (int c = 0; c < NK; c++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[c][e][j] = ldexpf(x[c][e][j], e2);
                ap_split8(x[c][e], qh[c][e], ql[c][e]);
            }
        f_row = ldexpf(1.0f, -e2);
        fc_row = fminf(f_row * A.cap_in, FLT_MAX);
        f_row *= A.scale2;
    }
    Running R;
    ap_f4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = ap_f4{0, 0, 0, 0};
    for (; u < u1; u += WAVES) {
        const int next = min(u + WAVES, u1 - 1), c = ap_chunk(S, u);
        ap_f4 sc[TT];
#pragma unroll
        for (int t = 0; t < TT; t++) sc[t] = ap_f4{0, 0, 0, 0};
        // (two tiles at a time: a product waits for the one before it of its sum)
#pragma unroll
        for (int e = 0; e < NK; e++)
#pragma unroll
            for (int t = 0; t < TT; t += 2) {
                ap_h8 a[2][2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    a[i][0] = ap_cvt8(kr[t + i][e].x, kr[t + i][e].y);
                    a[i][1] = ap_cvt8(kr[t + i][e].z, kr[t + i][e].w);
                }
#pragma unroll
                for (int y = 0; y < 2; y++) {
#pragma unroll
                    for (int i = 0; i < 2; i++) sc[t + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i][y], qh[e][y], sc[t + i], 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 2; i++) sc[t + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i][y], ql[e][y], sc[t + i], 0, 0, 0);
                }
            }
        // scores in log2 units are sc * f; the factor is kept above zero, so
        // that it leaves -inf as it is, and is a number where no key is seen
        const int j0 = c * CH + g * SEG;  // key of register (t, i): j0 + 4 t + i
        float f = fmaxf(f_row * ksc, 0x1p-120f), vs = vsc;
        const float fc = fminf(fc_row * ksc, FLT_MAX);  // a number: zero times it is zero
        const int pv_next = pv;
        load_keys(next);
        if (A.cap != 0.0f) {
#pragma unroll
            for (int i = 0; i < SEG; i++) sc[i >> 2][i & 3] = ap_capped(A, sc[i >> 2][i & 3] * f, sc[i >> 2][i & 3] * fc);
            f = 1.0f;
        }
        if (A.slopes) {
            const float far = (float)(j0 - p);
#pragma unroll
            for (int i = 0; i < SEG; i++) sc[i >> 2][i & 3] = fmaf(sc[i >> 2][i & 3], f, -slope * fabsf(far + (float)i));
            f = 1.0f;
        }
        if (!ap_whole(A, S, c * CH, CH) || __any(vs < 0.0f)) {
            const uint32_t hidden = vs < 0.0f ? kAll : ap_hidden(A, S, p, j0) & kAll;
#pragma unroll
            for (int i = 0; i < SEG; i++) sc[i >> 2][i & 3] = ap_hide(sc[i >> 2][i & 3], hidden, i);
            vs = hidden != kAll ? vs : 0.0f;
        }
        float mx = sc[0][0];
#pragma unroll
        for (int i = 1; i < SEG; i++) mx = fmaxf(mx, sc[i >> 2][i & 3]);
        if (__any(R.late(mx * f, R.most(mx, f, vs)))) {
            const float am = R.raise(ap_max_quarters(mx * f)), ao = R.refer(am, ap_max_quarters(R.most(mx, f, vs)));
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= ao;
        }
        const float w = vs * R.over;
        ap_h8 ph[TT / 2], pl[TT / 2];
#pragma unroll
        for (int e = 0; e < TT / 2; e++) {
            float pr[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                pr[j] = __builtin_amdgcn_exp2f(fmaf(sc[2 * e + (j >> 2)][j & 3], f, -R.m));
                R.l += pr[j];
            }
            ap_split8w(pr, w, ph[e], pl[e]);
        }
#pragma unroll
        for (int d = 0; d < ND; d += 2)
#pragma unroll
            for (int e = 0; e < TT / 2; e++) {
                const ap_h8 a = ap_cvt8(vr[d][2 * e], vr[d][2 * e + 1]), b = ap_cvt8(vr[d + 1][2 * e], vr[d + 1][2 * e + 1]);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[e], o[d], 0, 0, 0);
                o[d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, ph[e], o[d + 1], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[e], o[d], 0, 0, 0);
                o[d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, pl[e], o[d + 1], 0, 0, 0);
            }
        load_values(next, pv_next);
        pk = page_of(min(next + WAVES, u1 - 1), col >> 2);
        pv = page_of(min(next + WAVES, u1 - 1), g);
    }

    // all lanes of a column hold the same m and parts of l
    float m = R.m, l = R.l;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const float back = R.ref * (1.0f / kApUnit);
    const int rows = min(16, n_rows - tile * 16);
    const __amdgpu_buffer_rsrc_t part = ap_pieces(A, piece, 1);
    if constexpr (WAVES == 1) {
        if (n_split == 1) {
            if (col >= rows) return;
            const float z = l > 0.0f || l != l ? back / l : 0.0f;
            float *to = A.out + (s.q0 + tok) * A.ldo + (int64_t)head * hd + 4 * g;
#pragma unroll
            for (int d = 0; d < ND; d++)
                if (16 * d < hd) ap_put4(to + 16 * d, o[d][0] * z, o[d][1] * z, o[d][2] * z, o[d][3] * z, A.out_vec);
        } else if (col < rows) {
#pragma unroll
            for (int d = 0; d < ND; d++)
                if (16 * d < hd)
                    ap_store4(part, (4 * d + g) * 16 + col, float4{o[d][0] * back, o[d][1] * back, o[d][2] * back, o[d][3] * back});
            if (g == 0) ap_store4(part, 4 * hd + col, float4{m, l, 0, 0});
        }
    } else {
        __shared__ float4 o_lds[WAVES][ND * 4][17];
        __shared__ float m_lds[WAVES][16], l_lds[WAVES][16];
        if (g == 0) {
            m_lds[wave][col] = m;
            l_lds[wave][col] = l;
        }
#pragma unroll
        for (int d = 0; d < ND; d++)
            o_lds[wave][4 * d + g][col] = float4{o[d][0] * back, o[d][1] * back, o[d][2] * back, o[d][3] * back};
        __syncthreads();
        for (int i = tid; i < 4 * hd; i += WAVES * 64) {
            // whole rows to out, the sums of a dim for all rows to the splits
            const int c = n_split == 1 ? i / (hd / 4) : i % 16, d4 = n_split == 1 ? i % (hd / 4) : i / 16;
            if (c >= rows) continue;
            float mm = kApNone, ll = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) mm = fmaxf(mm, m_lds[w][c]);
            float4 oo = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float e = __builtin_amdgcn_exp2f(m_lds[w][c] - mm);
                const float4 v = o_lds[w][d4][c];
                ll = fmaf(l_lds[w][c], e, ll);
                oo = float4{fmaf(v.x, e, oo.x), fmaf(v.y, e, oo.y), fmaf(v.z, e, oo.z), fmaf(v.w, e, oo.w)};
            }
            if (n_split == 1) {
                const int rw = tile * 16 + c;
                ap_put4(A.out + (s.q0 + rw / A.G) * A.ldo + (int64_t)(h * A.G + rw % A.G) * hd + 4 * d4,
                        ap_quotient(oo.x, ll), ap_quotient(oo.y, ll), ap_quotient(oo.z, ll), ap_quotient(oo.w, ll), A.out_vec);
            } else {
                ap_store4(part, i, oo);
                if (d4 == 0) ap_store4(part, 4 * hd + c, float4{mm, ll, 0, 0});
            }
        }
    }
    if (n_split > 1) ap_join_rows<WAVES * 64>(A, s, h, tile, rows, piece - split, n_split);
}

// ---- many rows ---------------------------------------------------------------------
//
// One workgroup: 32 rows of one request and KV head for each of its waves, 128 or
// 256, and one split of its 64-key chunks. A chunk's codes are loaded as they
// lie, two chunks ahead, converted to f16 once for all waves and put into
// LDS, two chunks in turn: converting in every wave would cost as many vector
// instructions as the softmax. The 16-byte granules
// of a row are permuted by an exclusive or, so that 16 lanes that read the same
// column of 16 rows reach all 64 banks: by four bits of the row where a row
// is a multiple of 256 bytes, by three where it is an odd multiple of 128 and
// neighbouring rows lie in the two halves.
//
// Each half of a chunk is two steps between barriers: vector work (weights from
// scores, codes to f16) and matrix work (weights times values, the next half's
// scores). Of eight waves four are a step behind the others, which leaves each
// SIMD one wave of either kind at any time: kTurns.
//
// Bound by the latency of the vector step: a wave that is alone in it on its
// SIMD issues an instruction every 6 to 7 cycles, about 1850 a half, where the
// matrix step takes 1024. Neither pipe is full: of 3 prompts of up to 4096 vector
// instructions take half of the launch's cycles, products 0.37. 32 heads of 128
// on 8: 4096 rows 290 us, 16384 rows 3.8 ms, at 1150 TFLOP/s of f16 products (575
// of the formula's: each runs twice); 4096 capped 420 us, with slopes 332. Heads
// of 64: 4096 rows 180 us.
//
// A wave's 32x32 tile of S^T has its key rows in the order that gives lane
// (row c, half e) the scores of keys 32 u + 16 e + i in register i: row m of
// the operand is key 16 (m / 4 % 2) + 4 (m / 8) + m % 4.

// Large row blocks lie in the grid by their rank, the position of their first
// row in blocks, high ones first, whatever the request: those see the most keys,
// and a launch that starts them last would end with them alone (3 prompts of up
// to 4096 tokens behind up to 1000 keys, 40 heads: by rank 701 us, by their number
// in their request 770; 8 of 2048 behind up to 8000, 32 heads: 1210, 1409). Block
// i of that order: with F(t) = the blocks of rank t and above, its rank t has
// F(t + 1) <= i < F(t), and it is the i - F(t + 1)th of the requests that have
// one of that rank. Up to 64 kPlaceRegs requests.
__device__ inline bool ap_place(const AttnPArgs &A, int rows, int64_t i, int &r, int &tile) {
    const int lane = threadIdx.x & 63;
    if (A.n_req == 1) {
        r = 0;
        const int n = min(request_span(A.R, 0).n, A.R.max_q) * A.G;
        tile = (n + rows - 1) / rows - 1 - (int)i;
        return n >= A.least && tile >= 0;
    }
    int blocks[kPlaceRegs], first[kPlaceRegs];
#pragma unroll
    for (int k = 0; k < kPlaceRegs; k++) {
        const int q = lane + 64 * k;
        const Span s = q < A.n_req ? request_span(A.R, q) : Span{0, 0, 0, 0};
        const int n = min(s.n, A.R.max_q) * A.G;
        blocks[k] = n < A.least ? 0 : (n + rows - 1) / rows;
        first[k] = (int)min((int64_t)min(s.p0, A.R.max_kv) * A.G / rows, (int64_t)A.ranks);
    }
    int lo = 0, span = A.ranks + A.n_tiles;  // past the highest rank
    uint32_t f = 0;  // F(lo): at most 2^31, as the grid bounds the blocks of a request
    const uint32_t n = (uint32_t)i;
    if (A.n_req <= 32) {
        // the lanes try 64 ranks at once
        for (;;) {
            const int step = (span + 63) / 64, t = lo + lane * step;
            f = 0;
            for (int q = 0; q < A.n_req; q++) {
                const int b = __builtin_amdgcn_readlane(blocks[0], q);
                f += min(b, max(0, __builtin_amdgcn_readlane(first[0], q) + b - t));
            }
            const int c = __popcll(__ballot(f > n));
            if (c == 0) return false;  // (of the first round only: past the last block)
            lo += (c - 1) * step;
            f = (uint32_t)__builtin_amdgcn_readlane((int)f, c - 1);
            if (step == 1) break;
            span = step;
        }
    } else {
        // each lane has its requests, and the ranks are bisected (200 prompts of
        // up to 512: 697 us, 888 with the loop above; 64 of up to 1024 behind up to
        // 8000: 2185, 2230)
        auto from = [&](int t) {
            uint32_t x = 0;
#pragma unroll
            for (int k = 0; k < kPlaceRegs; k++) x += min(blocks[k], max(0, first[k] + blocks[k] - t));
            return (uint32_t)__builtin_amdgcn_readlane((int)ap_scan(x), 63);
        };
        f = from(0);
        if (f <= n) return false;
        while (span > 1) {
            const int half = span / 2;
            const uint32_t g = from(lo + half);
            if (g > n) {
                lo += half;
                f = g;
                span -= half;
            } else {
                span = half;
            }
        }
    }
    int more = 0;
#pragma unroll
    for (int k = 0; k < kPlaceRegs; k++) more += __popcll(__ballot(first[k] <= lo && lo - first[k] < blocks[k]));
    int rank = (int)(n - (f - more));
#pragma unroll
    for (int k = 0; k < kPlaceRegs; k++) {
        uint64_t has = __ballot(first[k] <= lo && lo - first[k] < blocks[k]);
        const int m = __popcll(has);
        if (rank >= 0 && rank < m) {
            for (; rank; rank--) has &= has - 1;
            const int l = __ffsll((unsigned long long)has) - 1;
            r = 64 * k + l;
            tile = lo - __builtin_amdgcn_readlane(first[k], l);
        }
        rank -= m;
    }
    r = __builtin_amdgcn_readfirstlane(r);
    tile = __builtin_amdgcn_readfirstlane(tile);
    return true;
}

// Waves of a large row block, heads of up to hd dims: up to 64 three workgroups
// of four fit a CU and fill each other's gaps (4096 rows of 32 heads: 170 us, two
// groups that take turns 213); wider ones take turns (256 rows behind 7000 keys
// 77 us, workgroups of four 84).
constexpr int ap_tile_waves(int hd) { return hd <= 64 ? 4 : 8; }

// hd rounded up to 16 NS dims
template <int NS, int WAVES = ap_tile_waves(16 * NS)>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 ? 3 : 2) void attnp_tiles_kernel(AttnPArgs A) {
    constexpr int kApTileRows = 32 * WAVES, kApTileThreads = 64 * WAVES;
    constexpr bool kTurns = WAVES == 8;
    constexpr int ND = (NS + 1) / 2;             // 32-dim tiles of the output
    constexpr int KC = (2 * NS + 7) / 8 * 8;     // granules of a key row in LDS
    constexpr int NU = (64 * NS + kApTileThreads - 1) / kApTileThreads;  // 16-byte loads of a chunk, each
    __shared__ uint4 k_lds[2][64][KC];
    __shared__ uint4 v_lds[2][ND * 32][8];
    __shared__ float s_lds[2][8];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int hd = A.C.hd, shift = A.C.shift, B = 1 << shift;
    const int h = blockIdx.x % A.C.n_kv, split = blockIdx.y;
    const int64_t place = blockIdx.x / A.C.n_kv;
    int r = blockIdx.z, tile = (int)(A.n_tiles - 1 - place);
    if (A.placed && !ap_place(A, kApTileRows, place, r, tile)) return;
    const int64_t item = (A.placed ? place : (int64_t)r * A.n_tiles + tile) * A.C.n_kv + h;
    const Span s = request_span(A.R, r);
    const int n_tok = min(s.n, A.R.max_q), n_rows = n_tok * A.G;
    if (tile * kApTileRows >= n_rows) return;
    const Sight S = ap_sight(A, r, s, tile * kApTileRows / A.G, min((tile * kApTileRows + kApTileRows - 1) / A.G, n_tok - 1));
    const int n_split = ap_splits(A, S.n, A.per_split);
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
    const float *qrow = A.q + (s.q0 + tok) * A.ldq + (int64_t)head * hd + 8 * half;

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
    auto load_keys = [&](int u) {
        const int at = ap_chunk(S, u) * 64 & (B - 1);
#pragma unroll
        for (int i = 0; i < NU; i++) kr[i] = *(const uint4 *)(kb[i] + ((uint64_t)(uint32_t)max(kpg[i], 0) * page_bytes + at * hd));
        if (tid < 8) scale = vpg >= 0 ? (tid < 4 ? A.C.ks : A.C.vs)[(int64_t)vpg * A.C.n_kv + h] : -1.0f;
    };
    auto load_values = [&](int u) {
        const uint64_t at = (uint64_t)(uint32_t)max(vpg, 0) * page_bytes + (ap_chunk(S, u) * 64 & (B - 1));
#pragma unroll
        for (int i = 0; i < NU; i++) vr[i] = *(const uint4 *)(vb[i] + at);
    };
    auto put_keys = [&](int buf) {
        const uint4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int key = unit(i) / NS, d16 = unit(i) % NS;
            // dims past hd meet zeros of q: they must be numbers
            const uint4 a = d16 * 16 < hd ? kr[i] : zero;
            const int kx = (key & 3) | ((key >> 2) & 4) | ((key << 1) & 8), x = KC % 16 ? kx >> 1 : kx;
            k_lds[buf][key][(2 * d16) ^ x] = __builtin_bit_cast(uint4, ap_cvt8(a.x, a.y));
            k_lds[buf][key][(2 * d16 + 1) ^ x] = __builtin_bit_cast(uint4, ap_cvt8(a.z, a.w));
        }
        if (tid < 8) s_lds[buf][tid] = scale;
    };
    auto put_values = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int dim = unit(i) >> 2, c = 2 * (tid & 3), y = (dim >> 1) & 7;
            v_lds[buf][dim][c ^ y] = __builtin_bit_cast(uint4, ap_cvt8(vr[i].x, vr[i].y));
            v_lds[buf][dim][(c + 1) ^ y] = __builtin_bit_cast(uint4, ap_cvt8(vr[i].z, vr[i].w));
        }
    };

    Running R;
    if (u0 < u1) {
        load_pages(u0);
        load_keys(u0);
        load_values(u0);
        load_pages(min(u0 + 1, u1 - 1));
    }
    // the query, while the first chunk is on its way
    ap_h8 qh[NS], ql[NS];
    float f_row, fc_row;
    {
        float x[NS][8], amax = 0.0f;
#pragma unroll
        for (int c = 0; c < NS; c++) ap_load8(qrow + (16 * c < hd ? 16 * c : 0), A.q_vec, x[c]);
#pragma unroll
        for (int c = 0; c < NS; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[c][j] = 16 * c < hd ? x[c][j] * A.sign : 0.0f;
                amax = fmaxf(amax, fabsf(x[c][j]));
            }
        const int e2 = ap_row_exponent(ap_max_halves(amax));
#pragma unroll
        for (int c = 0; c < NS; c++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[c][j] = ldexpf(x[c][j], e2);
            ap_split8(x[c], qh[c], ql[c]);
        }
        f_row = ldexpf(1.0f, -e2);
        fc_row = fminf(f_row * A.cap_in, FLT_MAX);
        f_row *= A.scale2;
    }
    ap_f16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    // nothing in a chunk for this wave's rows
    auto blind = [&](int u) {
        const int j0 = ap_chunk(S, u) * 64;
        return idle || (j0 >= S.prefix && (j0 > W.p_hi || (A.window && j0 + 63 <= W.p_lo - A.window)));
    };
    const int key = 16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3);
    const int x = KC % 16 ? (col >> 1) & 7 : col & 15, y = (col >> 1) & 7;
    ap_f16 sc;
    auto scores = [&](int buf, int i) {
        const uint4 *kl = k_lds[buf][32 * i + key];
#pragma unroll
        for (int e = 0; e < 16; e++) sc[e] = 0.0f;
#pragma unroll
        for (int c = 0; c < NS; c++) {
            const ap_h8 a = __builtin_bit_cast(ap_h8, kl[(2 * c + half) ^ x]);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], sc, 0, 0, 0);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[c], sc, 0, 0, 0);
        }
    };
    if (u0 < u1) {
        put_keys(0);
        put_values(0);
        load_keys(min(u0 + 1, u1 - 1));
        load_values(min(u0 + 1, u1 - 1));
        load_pages(min(u0 + 2, u1 - 1));
        __syncthreads();
        if (!blind(u0)) scores(0, 0);
        if (kTurns && wave >= 4) __syncthreads();
    }
    for (int u = u0; u < u1; u++) {
        const int buf = (u - u0) & 1, j0 = ap_chunk(S, u) * 64;
        const bool skip = blind(u), whole = ap_whole(A, W, j0, 64);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            // weights of the half's 32 keys, and a part of the next chunk
            ap_h8 ph[2], pl[2];
            if (!skip) {
                // scores in log2 units are sc * f; the factor is kept above zero,
                // so that it leaves -inf as it is, and is a number where no key is seen
                const float ksc = s_lds[buf][2 * i + half];
                float vsc = s_lds[buf][4 + 2 * i + half], f = fmaxf(f_row * ksc, 0x1p-120f);
                if (A.cap != 0.0f) {
                    const float fc = fminf(fc_row * ksc, FLT_MAX);
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
                if (__any(R.late(mx * f, R.most(mx, f, vsc)))) {
                    const float am = R.raise(ap_max_halves(mx * f)), ao = R.refer(am, ap_max_halves(R.most(mx, f, vsc)));
#pragma unroll
                    for (int d = 0; d < ND; d++) o[d] *= ao;
                }
                const float w = vsc * R.over;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float pr[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        pr[j] = __builtin_amdgcn_exp2f(fmaf(sc[8 * e + j], f, -R.m));
                        R.l += pr[j];
                    }
                    ap_split8w(pr, w, ph[e], pl[e]);
                }
            }
            if (i == 0) {
                if (u + 1 < u1) put_keys(buf ^ 1);
                load_keys(min(u + 2, u1 - 1));
            } else {
                if (u + 1 < u1) put_values(buf ^ 1);
                load_values(min(u + 2, u1 - 1));
                load_pages(min(u + 3, u1 - 1));
            }
            __syncthreads();
            // their products with the values, and the next half's scores
            if (!skip) {
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        const ap_h8 a = __builtin_bit_cast(ap_h8, v_lds[buf][32 * d + col][(4 * i + 2 * half + e) ^ y]);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[e], o[d], 0, 0, 0);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[e], o[d], 0, 0, 0);
                    }
                if (i == 0) scores(buf, 1);
            }
            if (i == 1 && u + 1 < u1 && !blind(u + 1)) scores(buf ^ 1, 0);
            __syncthreads();
        }
    }
    if (kTurns && u0 < u1 && wave < 4) __syncthreads();
    float m = R.m, l = R.l;
    l += __shfl_xor(l, 32);

    const float back = R.ref * (1.0f / kApUnit);
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
            float4 *to = ap_part(A, item * A.n_split + split, kApTileRows) + wave * 32 + col;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    if (32 * d + 8 * a < hd)
                        to[(8 * d + 2 * a + half) * kApTileRows] = float4{o[d][4 * a] * back, o[d][4 * a + 1] * back,
                                                                          o[d][4 * a + 2] * back, o[d][4 * a + 3] * back};
            if (half == 0) to[hd / 4 * kApTileRows] = float4{m, l, 0, 0};
        }
    }
}

// ---- row blocks whose keys were split -----------------------------------------------
//
// A second launch adds up a large row block's splits, in their order: a thread has
// four dims of a row. (One workgroup, the last of a block to arrive, would
// have to read all of it: 66 KB a split for 128 rows of 128 dims.)

constexpr int kApJoinThreads = 256;

template <int ROWS>
__global__ __launch_bounds__(kApJoinThreads) void attnp_join_kernel(AttnPArgs A) {
    const int h = blockIdx.x % A.C.n_kv, hd = A.C.hd;
    const int64_t place = blockIdx.x / A.C.n_kv;
    int r = blockIdx.z, tile = (int)place;
    if (A.placed && !ap_place(A, ROWS, place, r, tile)) return;
    const int64_t piece = ((A.placed ? place : (int64_t)r * A.n_tiles + tile) * A.C.n_kv + h) * A.n_split;
    const Span s = request_span(A.R, r);
    const int n_tok = min(s.n, A.R.max_q), n_rows = n_tok * A.G;
    const int c = threadIdx.x % ROWS, d4 = blockIdx.y * (kApJoinThreads / ROWS) + threadIdx.x / ROWS, row = tile * ROWS + c;
    if (tile * ROWS >= n_rows) return;
    const int t0 = tile * ROWS / A.G, t1 = min((tile * ROWS + ROWS - 1) / A.G, n_tok - 1);
    const int n_split = ap_splits(A, ap_sight(A, r, s, t0, t1).n, A.per_split);
    if (n_split == 1 || row >= n_rows || 4 * d4 >= hd) return;
    const float4 *part = ap_part(A, piece, ROWS) + c;
    const int64_t step = (int64_t)(hd / 4 + 1) * ROWS;
    // sixteen splits at once, all their loads in flight
    float m = kApNone, l = 0.0f;
    float4 o = {0, 0, 0, 0};
    for (int k0 = 0; k0 < n_split; k0 += 16) {
        float4 ml[16], v[16];
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const int64_t at = min(k0 + k, n_split - 1) * step;
            ml[k] = part[at + hd / 4 * ROWS];
            v[k] = part[at + d4 * ROWS];
        }
        ap_add16(n_split - k0, ml, v, m, l, o);
    }
    ap_put4(A.out + (s.q0 + row / A.G) * A.ldo + (int64_t)(h * A.G + row % A.G) * hd + 4 * d4, ap_quotient(o.x, l),
            ap_quotient(o.y, l), ap_quotient(o.z, l), ap_quotient(o.w, l), A.out_vec);
}

}  // namespace sihip
