// The rotation of queries and keys by their positions, on the way into a paged
// cache. Pair i of a head at position p, (a, b), becomes
//   (a cos - b sin, a sin + b cos)
// with cosine and sine from a table of f32. Both products of f32 numbers are exact in
// f64; their sum is rounded there and once more to f32. A code of the cache next to the
// border between two steps depends on the last bit of its value, and this value is
// the same whatever the order or contraction of the operations: it is that of the formula in
// 64 bits. The f64 operations, six a pair, cost no time beside the memory traffic.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kvcache.h"

namespace sihip {

struct RopeArgs {
    const float *table;  // [position][pairs][2], NULL: no rotation
    int pairs;           // of a head; dims from 2 pairs on stay as they are
    bool neighbours;     // pair i: dims 2 i, 2 i + 1; else i, i + pairs
    bool fours;          // the table is 16-byte aligned and pairs a multiple of 4
};

// The queries of a step, rotated into rows of their own (or in place).
struct RopeQueries {
    const float *q;
    float *out;
    int64_t ldq, ldo;
    int G;      // query heads of a KV head
    bool wide;  // rows of q and out and their heads are 16-byte aligned
    bool past;  // out is more than the L2s hold: written past them
};

__device__ inline float2 rope_pair(float a, float b, float c, float s) {
    const double x = a, y = b, u = c, v = s;
    return float2{(float)(x * u - y * v), (float)(x * v + y * u)};
}

// Dims d .. d + 3 (d a multiple of 4) of a head's row x, rotated; cs: the table's row
// of its position. wide: x is 16-byte aligned.
__device__ inline float4 rope_load4(const RopeArgs &P, const float *x, const float *cs, int d, bool wide) {
    const int turned = 2 * P.pairs;
    float v[4];
    if (wide) {
        const float4 f = *(const float4 *)(x + d);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = x[d + e];
    }
    if (d >= turned) return float4{v[0], v[1], v[2], v[3]};
    if (P.neighbours && P.fours) {
        const float4 t = *(const float4 *)(cs + d);
        const float2 a = rope_pair(v[0], v[1], t.x, t.y), b = rope_pair(v[2], v[3], t.z, t.w);
        return float4{a.x, a.y, b.x, b.y};
    }
    if (P.neighbours) {
        const float2 a = rope_pair(v[0], v[1], cs[d], cs[d + 1]);
        if (d + 2 >= turned) return float4{a.x, a.y, v[2], v[3]};
        const float2 b = rope_pair(v[2], v[3], cs[d + 2], cs[d + 3]);
        return float4{a.x, a.y, b.x, b.y};
    }
    if (wide && P.fours) {  // all four in the same half
        const bool low = d < P.pairs;
        const int i = low ? d : d - P.pairs;
        const float4 o = *(const float4 *)(x + (low ? d + P.pairs : i));
        const float4 t0 = *(const float4 *)(cs + 2 * i), t1 = *(const float4 *)(cs + 2 * i + 4);
        const float w[4] = {o.x, o.y, o.z, o.w}, c[4] = {t0.x, t0.z, t1.x, t1.z}, s[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 r = rope_pair(low ? v[e] : w[e], low ? w[e] : v[e], c[e], s[e]);
            v[e] = low ? r.x : r.y;
        }
        return float4{v[0], v[1], v[2], v[3]};
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int j = d + e;
        if (j >= turned) continue;
        const bool low = j < P.pairs;
        const int i = low ? j : j - P.pairs;
        const float o = x[low ? j + P.pairs : i];
        const float2 r = rope_pair(low ? v[e] : o, low ? o : v[e], cs[2 * i], cs[2 * i + 1]);
        v[e] = low ? r.x : r.y;
    }
    return float4{v[0], v[1], v[2], v[3]};
}

typedef float rope_f4 __attribute__((ext_vector_type(4)));
template <bool PAST>
__device__ inline void rope_store4(float *to, float4 v) {
    if constexpr (PAST) __builtin_nontemporal_store(rope_f4{v.x, v.y, v.z, v.w}, (rope_f4 *)to);
    else *(float4 *)to = v;
}

// The rows q0 + t0 .. q0 + t1 - 1 of a request whose row 0 is at position p0, of the
// query heads of KV head h, by a workgroup of THREADS: a thread takes four pairs (or
// eight dims that are not rotated) at a time, reads both of each pair and writes
// both, so that out may be q. What the L2s cannot hold is written past them: queries of 111 MB, with the append of their
// keys and values and its read-back, 73 us and 89 the other way, 78 MB 60 / 65, 65 MB 47 / 50; 49 MB 79 / 78, 34 MB
// 24 / 25 alone over 8 bits and 23 / 22 over 4.
template <int THREADS, bool PAST>
__device__ inline void rope_queries_to(const RopeArgs &P, const RopeQueries &Q, int hd, int h, int64_t q0, int p0, int t0, int t1) {
    const int turns = (P.pairs + 3) / 4, rest = (hd - 2 * P.pairs + 7) / 8, per_head = turns + rest;
    const int n = (t1 - t0) * Q.G * per_head;
    const bool fours = Q.wide && P.fours;
    for (int u = threadIdx.x; u < n; u += THREADS) {
        const int it = u % per_head, head = h * Q.G + u / per_head % Q.G, t = t0 + u / per_head / Q.G;
        const float *x = Q.q + (q0 + t) * Q.ldq + (int64_t)head * hd;
        float *to = Q.out + (q0 + t) * Q.ldo + (int64_t)head * hd;
        if (it >= turns) {
            const int d0 = 2 * P.pairs + 8 * (it - turns);
            if (fours) {  // (2 pairs is a multiple of 8, so d0 is; hd of 16)
                const float4 a = *(const float4 *)(x + d0), b = *(const float4 *)(x + d0 + 4);
                rope_store4<PAST>(to + d0, a);
                rope_store4<PAST>(to + d0 + 4, b);
            } else {
                for (int d = d0; d < min(d0 + 8, hd); d++) to[d] = x[d];
            }
            continue;
        }
        const float *cs = P.table + (int64_t)(p0 + t) * (2 * P.pairs) + 8 * it;
        if (fours) {
            // (neighbours past the L2s: two times two pairs, so that a wave's lanes write whole lines at a time)
            const bool four = P.neighbours && !PAST;
            const int at = four ? 8 * it : 4 * it, next = four ? at + 4 : at + P.pairs;
            const float *c0 = cs, *c1 = cs + 4;
            if constexpr (PAST)
                if (P.neighbours) c0 = cs - at, c1 = c0 + P.pairs;
            const float4 t0 = *(const float4 *)c0, t1 = *(const float4 *)c1;
            const float4 a = *(const float4 *)(x + at), b = *(const float4 *)(x + next);
            if (P.neighbours) {
                const float2 r0 = rope_pair(a.x, a.y, t0.x, t0.y), r1 = rope_pair(a.z, a.w, t0.z, t0.w);
                const float2 r2 = rope_pair(b.x, b.y, t1.x, t1.y), r3 = rope_pair(b.z, b.w, t1.z, t1.w);
                rope_store4<PAST>(to + at, float4{r0.x, r0.y, r1.x, r1.y});
                rope_store4<PAST>(to + next, float4{r2.x, r2.y, r3.x, r3.y});
            } else {
                const float2 r0 = rope_pair(a.x, b.x, t0.x, t0.y), r1 = rope_pair(a.y, b.y, t0.z, t0.w);
                const float2 r2 = rope_pair(a.z, b.z, t1.x, t1.y), r3 = rope_pair(a.w, b.w, t1.z, t1.w);
                rope_store4<PAST>(to + at, float4{r0.x, r1.x, r2.x, r3.x});
                rope_store4<PAST>(to + next, float4{r0.y, r1.y, r2.y, r3.y});
            }
            continue;
        }
        for (int i = 4 * it; i < min(4 * it + 4, P.pairs); i++) {
            const int a = P.neighbours ? 2 * i : i, b = P.neighbours ? 2 * i + 1 : i + P.pairs;
            const float2 r = rope_pair(x[a], x[b], cs[2 * (i - 4 * it)], cs[2 * (i - 4 * it) + 1]);
            to[a] = r.x;
            to[b] = r.y;
        }
    }
}

template <int THREADS>
__device__ inline void rope_queries(const RopeArgs &P, const RopeQueries &Q, int hd, int h, int64_t q0, int p0, int t0, int t1) {
    if (Q.past) rope_queries_to<THREADS, true>(P, Q, hd, h, q0, p0, t0, t1);
    else rope_queries_to<THREADS, false>(P, Q, hd, h, q0, p0, t0, t1);
}

}  // namespace sihip
