// The paged 4-bit KV cache: the write of new rows (kv4_append_kernel) and the
// read-back of rows (kv4_read_kernel). Its attention is in attnp4.h.
//
// A value is code * sub * scale. Codes -8 .. 7, eight to a word (below): keys
// [page][head][token][dim], values [page][head][dim][token]; subs, signed bytes, one for
// each token and 32 dims, [page][head][group][token]; scales, bfloat16, one for each token
// and head, [page][head][token]. Two levels, because code * sub is then a whole number
// of at most 8 * 127 = 1016, which f16 holds: the matrix cores multiply the cache without
// a rounding, and the f32 side is one factor a token, as in the 8-bit cache. A row is quantized
// once, by itself: nothing that comes later changes it.
//
// Of a row's group the step is -1/8 of its value of largest magnitude (so that this
// one is code -8 and the 16 codes reach from it to 7/8 of its opposite); the scale is
// the row's largest step / 127, rounded up to bfloat16; the sub is the step over the
// scale, rounded away from zero, so that no value lies beyond code -8. A scale of 8
// bits of mantissa costs nothing: codes are rounded with the scale that is stored.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kvcache.h"
#include "rope.h"

namespace sihip {

struct Cache4Args {
    uint8_t *k, *v;
    int8_t *ksub, *vsub;
    uint16_t *ks, *vs;
    int64_t n_pages;
    int n_kv, hd, shift;
};

// Words: element e of eight is the nibble e / 2 + 4 (e % 2), plus 8. Elements 2 i
// and 2 i + 1 then lie 16 bits apart, the halves of a pair of f16 numbers.

// the codes (plus 8) of elements 4 odd .. 4 odd + 3, a byte each, as nibbles of their word
__device__ inline uint32_t kv4_half_word(uint32_t c, int odd) {
    const uint32_t w = (c & 15) | (c >> 16 & 15) << 4 | (c >> 8 & 15) << 16 | (c >> 24) << 20;
    return w << (8 * odd);
}

// the nibbles of the elements that lie in [lo, hi) of a word that begins at element 0
__device__ inline uint32_t kv4_mask(int lo, int hi) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) m |= e >= lo && e < hi ? 15u << (4 * ((e >> 1) + 4 * (e & 1))) : 0u;
    return m;
}

// the word's elements in order, element e at nibble e
__device__ inline uint32_t kv4_in_order(uint32_t w) {
    auto spread = [](uint32_t x) {
        x = (x | x << 8) & 0x00ff00ffu;
        return (x | x << 4) & 0x0f0f0f0fu;
    };
    return spread(w & 0xffffu) | spread(w >> 16) << 4;
}

__device__ inline float kv4_scale(uint16_t bits) { return __builtin_bit_cast(float, (uint32_t)bits << 16); }

// ---- append ------------------------------------------------------------------------

struct Append4Args {
    Cache4Args C;
    BatchArgs R;
    RopeArgs P;     // P.table NULL: keys as they are
    RopeQueries Q;  // Q.q NULL: none
    const float *k, *v;
    int64_t ldk, ldv;
    bool wide;  // rows of k and v and their heads are 16-byte aligned
};

constexpr int k4Threads = 256;
constexpr int k4Chunk = 64;  // tokens of a page at a time
constexpr float k4Most = 0x1p126f;  // larger magnitudes count as this one for the steps

// x / step rounded to an integer, ties to even, exactly (quantize_exact says
// how; step = |sub| * scale has 15 bits), at most 7 and at least -8. NaN and a step of zero: 0.
__device__ inline int kv4_code(float x, float step, float inv) {
    if (x != x || step == 0.0f) return 0;
    float q = rintf(x * inv);
    const float up = fmaf(-(q + 0.5f), step, x), down = fmaf(-(q - 0.5f), step, x);
    const bool odd = ((int)q & 1) != 0;
    if (up > 0.0f || (up == 0.0f && odd)) q += 1.0f;
    else if (down < 0.0f || (down == 0.0f && odd)) q -= 1.0f;
    return (int)fminf(fmaxf(q, -8.0f), 7.0f);
}

// x of another lane of the row of 16
template <int CTRL>
__device__ inline float kv4_from(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

// the largest of eight lanes in a row (lanes 8 i .. 8 i + 7)
__device__ inline float kv4_max8(float x) {
    x = fmaxf(x, kv4_from<0xb1>(x));      // lane ^ 1
    x = fmaxf(x, kv4_from<0x4e>(x));      // lane ^ 2
    return fmaxf(x, kv4_from<0x141>(x));  // 7 - lane of eight
}

struct Kv4Step {
    float sub, scale;  // sub is a whole number
};

// The sub and the scale of this lane's group of 32: eight lanes have it, four values each, and hd / 4
// lanes from `row0` on have the row.
__device__ inline Kv4Step kv4_step(const float *v, int hd, int row0) {
    float most = kv4_max8(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))));
    float low = fminf(fminf(v[0], v[1]), fminf(v[2], v[3]));
    if (__any(!(most < INFINITY) || !(low > -INFINITY))) {  // (numbers alone count)
        float a = 0.0f;
        low = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float f = fabsf(v[e]) < INFINITY ? v[e] : 0.0f;
            a = fmaxf(a, fabsf(f));
            low = fminf(low, f);
        }
        most = kv4_max8(a);
    }
    most = fminf(most, k4Most);
    // the largest is negative in one of the eight lanes: code -8 is on that side
    const bool plus = (__ballot(low <= -most) >> (threadIdx.x & 56) & 255) != 0;
    const float size = 0.125f * most;  // |step|
    float row = size;
    if (hd == 128 || hd == 256 || hd == 64) {
        row = fmaxf(row, kv4_from<0x128>(row));  // lane ^ 8
        const uint32_t b = __builtin_bit_cast(uint32_t, row);
        if (hd >= 128) {
            const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
            row = fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
        }
        if (hd == 256) {
            const uint32_t w = __builtin_bit_cast(uint32_t, row);
            const auto r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
            row = fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
        }
    } else {
        for (int i = 0; i < hd / 32; i++) row = fmaxf(row, __shfl(size, row0 + 8 * i));
    }
    // row / 127, rounded to the nearest (the remainder of the product with the rounded reciprocal is
    // exact, and corrects it), then up to bfloat16
    const float rough = row * (1.0f / 127.0f), exact = fmaf(fmaf(-127.0f, rough, row), 1.0f / 127.0f, rough);
    const uint32_t up = (__builtin_bit_cast(uint32_t, exact) + 0xffffu) & 0xffff0000u;
    const float scale = row < 0.125f * kTinyAmax ? 0.0f : __builtin_bit_cast(float, up);
    // |sub|: size / scale up to a whole number; the rough quotient is off by less than one, the
    // products that show it are exact
    float n = 1.0f;
    if (scale > 0.0f) {
        n = ceilf(size * __builtin_amdgcn_rcpf(scale));
        if ((n - 1.0f) * scale >= size) n -= 1.0f;
        else if (n * scale < size) n += 1.0f;
        n = fminf(fmaxf(n, 1.0f), 127.0f);
    }
    return {plus ? n : -n, scale};
}

// The codes, plus 8, of four values, a byte each. The sum with 1.5 2^23 + 8 leaves the rounded quotient in the
// low bits; what is within 10^-4 of a border between two codes (or no number) is rounded exactly.
__device__ inline uint32_t kv4_codes(const float *v, const Kv4Step &q) {
    constexpr float kMagic = 12582920.0f;
    const float step = fabsf(q.sub) * q.scale, side = q.sub < 0.0f ? -1.0f : 1.0f;
    const float inv = step > 0.0f ? side * __builtin_amdgcn_rcpf(step) : 0.0f;
    bool clear = true;
    uint32_t c = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float r = fmaf(v[e], inv, kMagic);
        clear &= fabsf(fmaf(v[e], inv, kMagic - r)) <= 0.4999f;
        c |= (__builtin_bit_cast(uint32_t, fminf(fmaxf(r, kMagic - 8.0f), kMagic + 7.0f)) & 15u) << (8 * e);
    }
    if (clear) return c;
    const float near = step > 0.0f ? 1.0f / step : 0.0f;
    c = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) c |= (uint32_t)(kv4_code(side * v[e], step, near) + 8) << (8 * e);
    return c;
}

// A workgroup: one page of new tokens and one KV head, keys (z = 0), values (1) or, rotated,
// the queries of that KV head (2). hd / 4 lanes have a row, four values each, and its
// groups of 32 are eight lanes in a row: the step is found by them, the scale among the
// groups' first lanes. Keys go from there to the page; values through LDS, 64 tokens at a time,
// from where a thread takes four dims of eight tokens, turns them round and writes a
// word a dim. Words that hold other tokens as well keep those.
//
// Bound by memory: 5 prompt chunks of up to 2047 tokens, 40 heads of 128 on 8, rotated, 288 MB in 58.4 us (4.9 TB/s; the
// queries are four fifths of it), 26.8 without queries, where four rows a wave at a time are quantized in about 100 instructions each: divisions
// and rounding proofs only next to a border. One token each for 64 requests 6.2 us, of which an empty launch takes 3.5.
__global__ __launch_bounds__(k4Threads) void kv4_append_kernel(Append4Args A) {
    __shared__ uint32_t turn[k4Chunk * (256 / 4 + 1)];
    const int n_kv = A.C.n_kv, hd = A.C.hd, shift = A.C.shift, B = 1 << shift;
    const int h = blockIdx.x % n_kv, r = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const PageSpan g = page_span(A.R, r, blockIdx.x / n_kv, shift);
    const int lo = g.lo, hi = g.hi;
    if (lo >= hi) return;
    if (blockIdx.z == 2) {
        const int first = (int)(g.base - g.p0);
        rope_queries<k4Threads>(A.P, A.Q, hd, h, g.q0, g.p0, first + lo, first + hi);
        return;
    }
    const bool is_v = blockIdx.z != 0, rotate = !is_v && A.P.table;
    const int64_t page = A.R.table[(int64_t)r * A.R.max_blocks + g.block];
    if (page < 0 || page >= A.C.n_pages) return;
    const int64_t ld = is_v ? A.ldv : A.ldk, ph = page * n_kv + h;
    // row of the page's token 0 (may lie before the first row)
    const float *x = (is_v ? A.v : A.k) + (g.q0 + g.base - g.p0) * ld + (int64_t)h * hd;
    uint32_t *codes = (uint32_t *)((is_v ? A.C.v : A.C.k) + ph * ((int64_t)(hd / 2) << shift));
    int8_t *subs = (is_v ? A.C.vsub : A.C.ksub) + ph * ((int64_t)(hd / 32) << shift);
    uint16_t *scales = (is_v ? A.C.vs : A.C.ks) + (ph << shift);

    const int lanes = hd / 4, per_wave = 64 / lanes, of = lane / lanes, li = lane % lanes, row0 = of * lanes;
    const int per_pass = per_wave * (k4Threads / 64);
    const int pitch = lanes + 1;
    constexpr int kAhead = 4;
    for (int c0 = lo & -k4Chunk; c0 < hi; c0 += k4Chunk) {
        const int t_lo = max(lo, c0), t_hi = min(hi, c0 + k4Chunk);
        for (int p0 = t_lo; p0 < t_hi; p0 += kAhead * per_pass) {
            float4 val[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; a++) {
                const int t = p0 + a * per_pass + wave * per_wave + of;
                val[a] = float4{0, 0, 0, 0};
                if (of >= per_wave || t >= t_hi) continue;
                const float *row = x + (int64_t)t * ld;
                if (rotate) val[a] = rope_load4(A.P, row, A.P.table + (g.base + t) * (2 * A.P.pairs), 4 * li, A.wide);
                else if (A.wide) val[a] = *(const float4 *)(row + 4 * li);
                else val[a] = float4{row[4 * li], row[4 * li + 1], row[4 * li + 2], row[4 * li + 3]};
            }
#pragma unroll
            for (int a = 0; a < kAhead; a++) {
                if (p0 + a * per_pass >= t_hi) break;
                const int t = p0 + a * per_pass + wave * per_wave + of;
                const float v[4] = {val[a].x, val[a].y, val[a].z, val[a].w};
                const Kv4Step q = kv4_step(v, hd, row0);
                const uint32_t c = kv4_codes(v, q);
                const bool here = of < per_wave && t < t_hi;
                if (is_v) {
                    if (here) turn[(t - c0) * pitch + li] = c;
                } else {
                    uint32_t w = kv4_half_word(c, li & 1);
                    w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xb1, 0xf, 0xf, true);
                    if (here && !(li & 1)) codes[t * (hd / 8) + li / 2] = w;
                }
                if (here && li % 8 == 0) subs[((li / 8) << shift) + t] = (int8_t)q.sub;
                if (here && li == 0) scales[t] = (uint16_t)(__builtin_bit_cast(uint32_t, q.scale) >> 16);
            }
        }
        if (!is_v) continue;
        __syncthreads();
        // words of eight tokens that hold new ones
        const int w0 = (t_lo - c0) / 8, n_words = (t_hi - c0 + 7) / 8 - w0;
        for (int u = tid; u < n_words * lanes; u += k4Threads) {
            const int w = w0 + u % n_words, d4 = u / n_words;
            uint32_t c[8];
#pragma unroll
            for (int e = 0; e < 8; e++) c[e] = turn[(8 * w + e) * pitch + d4] & 0x0f0f0f0fu;  // (of tokens that are not new: anything)
            // bytes of a dim: elements 0 and 2, 4 and 6, 1 and 3, 5 and 7
            const uint32_t a0 = c[0] | c[2] << 4, a1 = c[4] | c[6] << 4, a2 = c[1] | c[3] << 4, a3 = c[5] | c[7] << 4;
            const uint32_t mask = kv4_mask(t_lo - c0 - 8 * w, t_hi - c0 - 8 * w);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t *to = codes + (4 * d4 + e) * (B / 8) + c0 / 8 + w;
                const uint32_t b0 = a0 >> (8 * e) & 255, b1 = a1 >> (8 * e) & 255, b2 = a2 >> (8 * e) & 255, b3 = a3 >> (8 * e) & 255;
                const uint32_t got = b0 | b1 << 8 | b2 << 16 | b3 << 24;
                *to = mask == 0xffffffffu ? got : (*to & ~mask) | (got & mask);
            }
        }
        __syncthreads();
    }
}

// ---- read ---------------------------------------------------------------------------

struct Read4Args {
    Cache4Args C;
    const int64_t *slots;
    float *k, *v;
    int64_t n, ldk, ldv;
    bool wide;  // rows of k and v and their heads are 16-byte aligned
};

// One workgroup: ROWS slots of one KV head, keys (z = 0): eight dims of a slot a
// thread; or values: two dims of 16 slots a thread, so that the lanes of a wave write
// rows. 16 slots that go on from one another lie in one or two segments of 16
// tokens of the transposed pages: two loads a dim. Any others are read a word at a time.
//
// Bound by memory: 8192 tokens of 8 heads of 128 in 17 us (3.2 TB/s), those that 64 single tokens share a page with 9.6, of
// which an empty launch takes 3.5 and three loads that wait for one another most of the rest.
template <int ROWS>
__global__ __launch_bounds__(kReadThreads) void kv4_read_kernel(Read4Args A) {
    __shared__ int64_t at[ROWS];  // first code of the page and head, or -1
    __shared__ int off[ROWS];     // place in the page
    __shared__ float step[8][ROWS];
    __shared__ int run[ROWS / 16];  // whether the 16 slots go on from one another
    const int h = blockIdx.y, hd = A.C.hd, shift = A.C.shift, tid = threadIdx.x;
    const bool is_v = blockIdx.z != 0;
    const int64_t i0 = (int64_t)blockIdx.x * ROWS;
    if (tid < ROWS) {
        const int64_t slot = i0 + tid < A.n ? A.slots[i0 + tid] : -1, page = slot >> shift;
        const bool ok = slot >= 0 && page < A.C.n_pages;
        const int64_t ph = page * A.C.n_kv + h;
        const int o = (int)(slot & ((1 << shift) - 1));
        at[tid] = ok ? ph * ((int64_t)(hd / 2) << shift) : -1;
        off[tid] = o;
        const int8_t *subs = (is_v ? A.C.vsub : A.C.ksub) + (ok ? (ph * (hd / 32) << shift) + o : 0);
        const float scale = ok ? kv4_scale((is_v ? A.C.vs : A.C.ks)[(ph << shift) + o]) : 0.0f;
        for (int g = 0; g < hd / 32; g++) step[g][tid] = scale * subs[g << shift];
        const int64_t s0 = __shfl(slot, tid & 48);
        const int left = 16 - (int)(s0 & 15), k = tid & 15;
        const int64_t s1 = __shfl(slot, (tid & 48) + (left & 15));
        const bool on = ok && (k < left ? slot == s0 + k : (s1 & 15) == 0 && slot == s1 + k - left);
        const uint64_t all = __ballot(on);
        if (k == 0) run[tid >> 4] = (all >> (tid & 48) & 0xffffu) == 0xffffu;
    }
    __syncthreads();
    if (!is_v) {
        const int per_row = hd / 8;
#pragma unroll 4
        for (int u = tid; u < ROWS * per_row; u += kReadThreads) {
            const int i = u / per_row, w = u % per_row;
            if (at[i] < 0) continue;
            const uint32_t c = kv4_in_order(*(const uint32_t *)(A.C.k + at[i] + off[i] * (hd / 2) + 4 * w));
            const float s = step[w / 4][i];
            float *to = A.k + (i0 + i) * A.ldk + (int64_t)h * hd + 8 * w;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = ((int)(c >> (4 * e) & 15) - 8) * s;
            if (A.wide) {
                *(float4 *)to = float4{y[0], y[1], y[2], y[3]};
                *(float4 *)(to + 4) = float4{y[4], y[5], y[6], y[7]};
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) to[e] = y[e];
            }
        }
        return;
    }
    const int row_bytes = 1 << shift >> 1;  // of a dim
    for (int u = tid; u < ROWS / 16 * (hd / 2); u += kReadThreads) {
        const int first = u / (hd / 2) * 16, d = u % (hd / 2) * 2, grp = d / 32;
        float *to = A.v + (i0 + first) * A.ldv + (int64_t)h * hd + d;
        uint32_t c[2][2];  // 16 codes of two dims, in order
        if (run[first >> 4]) {
            const int from = off[first] & 15, left = 16 - from, next = first + (left & 15);
            const uint8_t *a = A.C.v + at[first] + (off[first] & ~15) / 2 + d * row_bytes;
            const uint8_t *b = A.C.v + at[next] + (off[next] & ~15) / 2 + d * row_bytes;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint2 x = *(const uint2 *)(a + e * row_bytes), y = *(const uint2 *)(b + e * row_bytes);
                uint32_t w[4] = {kv4_in_order(x.x), kv4_in_order(x.y), kv4_in_order(y.x), kv4_in_order(y.y)};
                if (from & 8) w[0] = w[1], w[1] = w[2], w[2] = w[3];
                c[e][0] = __builtin_amdgcn_alignbit(w[1], w[0], 4 * (from & 7));
                c[e][1] = __builtin_amdgcn_alignbit(w[2], w[1], 4 * (from & 7));
            }
        } else {
            uint32_t w[2][16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                // (a slot that is none reads the first page, and writes nothing)
                const int64_t from = at[first + i] < 0 ? 0 : at[first + i] + (off[first + i] & ~7) / 2;
                const uint8_t *a = A.C.v + from + d * row_bytes;
                w[0][i] = *(const uint32_t *)a;
                w[1][i] = *(const uint32_t *)(a + row_bytes);
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                c[e][0] = c[e][1] = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int o = off[first + i] & 7;
                    c[e][i / 8] |= (w[e][i] >> (4 * ((o >> 1) + 4 * (o & 1))) & 15) << (4 * (i % 8));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            if (at[first + i] < 0) continue;
            const float s = step[grp][first + i];
            const float a = ((int)(c[0][i / 8] >> (4 * (i % 8)) & 15) - 8) * s, b = ((int)(c[1][i / 8] >> (4 * (i % 8)) & 15) - 8) * s;
            if (A.wide) {
                *(float2 *)(to + i * A.ldv) = float2{a, b};
            } else {
                to[i * A.ldv] = a;
                to[i * A.ldv + 1] = b;
            }
        }
    }
}

}  // namespace sihip
