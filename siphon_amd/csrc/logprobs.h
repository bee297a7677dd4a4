// Log probabilities of given tokens, entropy and the most likely tokens of rows of
// logits, in one pass over them (declaration in include/sihip.h).
//
//   m = max x, l = sum e^(x - m), t = sum e^(x - m) (x - m)
//   log p_i = x_i - m - log l,  H = log l - t / l
//
// Both terms of H are not negative, so nothing cancels. Each thread has a running m of
// its own; exponentials are f32 and added in f64: where one token has nearly all of the
// probability, log l is what the others add to 1.
//
// The most likely: of a logit and its index a key is made, a 63-bit number that grows with the
// logit and, of equal ones, falls with the index, so that no two are equal. The pass itself keeps the
// largest of each thread's 16 logits at a time, no more. Every kLpRounds of them a wave ranks a few of
// its lanes' largest; the n_topth of these is a threshold, as n_top keys reach it: what is below is not
// among the most likely. The few runs of 16 that reach it are read again, four lanes a run (a single round's are
// still in registers), and the keys that reach it go to a list in LDS. In the end, or when it is full, a
// list is cut to its n_top largest, found by counting for each key how many are larger.
//
// A row of many logits is split over workgroups. A wave of each leaves its n_top largest in order, and the first
// wave of the last workgroup to arrive takes from the lists' fronts what may be among the row's.
//
// Bound by memory where there are rows enough: 500 rows of 151936 (304 MB) 50-53 us (5.8-6.0 TB/s, a part of them from the
// Infinity Cache), with the 20 most likely 67-72 (4.2-4.5), with 64 105; few rows by instructions in turn: one row of 151936 with 5
// tokens takes 9.5 us, 3.5 of which an empty launch takes, 1 the pass, 2 the choices of the splits, 1.5 sums and
// their way to the last workgroup, 1.5 its choice. (A choice of single keys as they came, with comparisons of integers:
// 11.9, 64 rows of 32003 with 20 tokens 17 and not 13.8.)
#pragma once

#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "agent.h"

namespace sihip {

struct LogprobArgs {
    const float *x;
    int64_t ld, n;  // n logits a row
    const int32_t *token;
    float *logprob, *entropy, *top_logprob;
    int32_t *top_id;
    int64_t n_token;
    int n_top, n_split;
    int64_t per_split;  // granules of 16 bytes of a split
    uint8_t *part;      // of each row: [split] maximum and sums, [split][wave][n_top] keys
    uint32_t *cnt;      // of each row: splits that have arrived, zero between launches
};

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr int kLpMostSplits = 64;  // of a row, where tokens are chosen
constexpr int kLpMostTop = 64;  // keys that a wave can choose with a lane each
constexpr int kLpList = 384;
constexpr int kLpGroup = 4;     // 16-byte loads of a thread at a time
constexpr int kLpRounds = 8;    // of them between choices

// bytes of a row's part
__host__ __device__ inline int64_t lp_part_bytes(int n_top, int n_split) { return (int64_t)n_split * (32 + kLpWaves * n_top * 8); }

// x of another lane: 1 .. 32 lanes away, once all lanes between have the same
template <int D>
__device__ inline uint32_t lp_other(uint32_t x) {
    if constexpr (D >= 16) {  // (one of the two is this lane's: the sum of both, less it)
        const auto r = D == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false) : __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return (uint32_t)r[0] ^ (uint32_t)r[1] ^ x;
    } else {
        constexpr int ctrl = D == 1 ? 0xb1 : D == 2 ? 0x4e : D == 4 ? 0x141 : 0x140;
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, true);
    }
}
template <int D>
__device__ inline uint64_t lp_other(uint64_t x) {
    return (uint64_t)lp_other<D>((uint32_t)(x >> 32)) << 32 | lp_other<D>((uint32_t)x);
}
template <int D>
__device__ inline double lp_other(double x) { return __builtin_bit_cast(double, lp_other<D>(__builtin_bit_cast(uint64_t, x))); }
template <int D>
__device__ inline float lp_other(float x) { return __builtin_bit_cast(float, lp_other<D>(__builtin_bit_cast(uint32_t, x))); }

struct LpSums {
    float m;
    double l, t;

    // of no logits
    static __device__ LpSums none() { return {-FLT_MAX, 0.0, 0.0}; }

    // to a maximum that is not smaller
    __device__ void raise(float to) {
        const double d = (double)m - (double)to, f = (double)__builtin_amdgcn_exp2f((float)d * 1.44269504088896340736f);
        t = f > 0.0 ? f * (t + d * l) : 0.0 * l;  // (keeps a NaN)
        l *= f;
        m = to;
    }
    template <int D, int N>
    __device__ void largest(float &to) const {
        to = fmaxf(to, lp_other<D>(to));
        if constexpr (2 * D < N) largest<2 * D, N>(to);
    }
    template <int D, int N>
    __device__ void sum() {
        l += lp_other<D>(l);
        t += lp_other<D>(t);
        if constexpr (2 * D < N) sum<2 * D, N>();
    }
    // of N lanes in a row, the same bits in each of them
    template <int N>
    __device__ void join() {
        float to = m;
        largest<1, N>(to);
        raise(to);
        sum<1, N>();
    }
};

// a number that grows with x; NaN counts as -inf, -0 as 0
__device__ inline uint32_t lp_order(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x == x ? x + 0.0f : -INFINITY);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kLpNone = 0x007fffffu;  // of -inf
// (63 bits, of which the first 11 are never all set: as f64 numbers keys are finite and in the same order, and
// those are compared faster)
__device__ inline uint64_t lp_pair(uint32_t order, uint32_t index) { return (uint64_t)order << 31 | (0x7fffffffu - index); }
__device__ inline bool lp_above(uint64_t a, uint64_t b) { return __builtin_bit_cast(double, a) > __builtin_bit_cast(double, b); }
__device__ inline uint64_t lp_key(float x, uint32_t index) { return lp_pair(lp_order(x), index); }
__device__ inline float lp_value(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 31);
    return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ inline int32_t lp_index(uint64_t key) { return 0x7fffffff - (int32_t)(key & 0x7fffffff); }

typedef uint32_t lp_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t lp_u2 __attribute__((ext_vector_type(2)));

// how many of n keys in LDS are larger (n is padded to a multiple of eight with zeros, by lp_pad)
__device__ inline int lp_larger(const uint64_t *keys, int n, uint64_t key) {
    int k = 0;
#pragma unroll 1
    for (int i = 0; i < n; i += 8) {
        ulonglong2 o[4];
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = *(const ulonglong2 *)(keys + i + 2 * e);
#pragma unroll
        for (int e = 0; e < 4; e++) k += lp_above(o[e].x, key) + lp_above(o[e].y, key);
    }
    return k;
}
__device__ inline void lp_pad(uint64_t *keys, int n) {
    const int lane = threadIdx.x & 63;
    if (lane < (-n & 7)) keys[n + lane] = 0;
}

// A wave's choice of the n_top largest of the keys it is shown.
struct LpChoice {
    uint64_t *list;  // of the wave, in LDS: kLpList keys and 128 more
    int n_top, count = 0;
    uint64_t least = 1;  // keys below it are not among the largest (0 is no key)

    // a wave's LDS accesses are in order; the compiler is told not to move them
    static __device__ void fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

    // cuts the list to its n_top largest, in order
    __device__ void cut() {
        const int lane = threadIdx.x & 63;
        uint64_t *to = list + kLpList;
        lp_pad(list, count);
        fence();
#pragma unroll 1
        for (int at = lane; at < count; at += 64) {
            const uint64_t key = list[at];
            const int rank = lp_larger(list, count, key);
            if (rank < n_top) to[rank] = key;
        }
        fence();
        count = min(count, n_top);
        if (lane < count) list[lane] = to[lane];
        fence();
        if (count == n_top) least = max(least, list[n_top - 1]);
    }
    // raises the threshold by two keys of each lane (or 0), each reached by one of its own: to the logit of the
    // n_topth largest, or, if many reach that, as of equal logits, to that key. How many keys are ranked goes by
    // how many are wanted: the 5th of 16 is reached by 6 keys on average (16 log 16 / 11), the 20th of 64 by
    // 24, the 64th of 128 by 89 (of 64 by 300).
    __device__ void limit(uint64_t a, uint64_t b) {
        const int lane = threadIdx.x & 63, shift = n_top <= 8 ? 2 : 0;
        const bool two = n_top > 32;
        if (!two) a = max(a, b), b = 0;
        if (shift) {
            a = max(a, lp_other<1>(a));
            a = max(a, lp_other<2>(a));
        }
        const bool first = !(lane & ((1 << shift) - 1));
        if (__popcll(__ballot(first && a >= least)) + __popcll(__ballot(b >= least)) < n_top) return;
        const int n = two ? 128 : 64 >> shift;
        uint64_t *all = list + kLpList;
        uint32_t *order = (uint32_t *)all;
        const uint32_t a_high = (uint32_t)(a >> 32), b_high = (uint32_t)(b >> 32);
        if (first) order[lane >> shift] = a_high;
        if (two) order[64 + lane] = b_high;
        fence();
        int over_a = 0, over_b = two ? 0 : n_top;  // how many are larger
#pragma unroll 4
        for (int i = 0; i < n; i += 4) {
            const lp_u4 o = *(const lp_u4 *)(order + i);
#pragma unroll
            for (int e = 0; e < 4; e++) over_a += o[e] > a_high;
            if (two)
#pragma unroll
                for (int e = 0; e < 4; e++) over_b += o[e] > b_high;
        }
        fence();
        const bool many = __popcll(__ballot(first && over_a < n_top)) + __popcll(__ballot(over_b < n_top)) > n_top + 8;
        if (many) {
            if (first) all[lane >> shift] = a;
            if (two) all[64 + lane] = b;
            fence();
            over_a = lp_larger(all, n, a);
            if (two) over_b = lp_larger(all, n, b);
            fence();
        }
        int rank = n_top - 1;
        uint64_t in_a, in_b;
        while (in_a = __ballot(over_a == rank), in_b = __ballot(over_b == rank), !(in_a | in_b) && rank > 0) rank--;
        const int from = __ffsll((unsigned long long)(in_a ? in_a : in_b)) - 1;
        const uint64_t key = in_a ? a : b;
        const uint64_t k = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), from) << 32 |
                           (many ? (uint32_t)__builtin_amdgcn_readlane((int)key, from) : 0u);
        least = k > least ? k : least;
    }
    // a key a lane, where it reaches the threshold
    __device__ void add(uint64_t key) {
        const uint64_t here = __ballot(key >= least);
        if (key >= least) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(here >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)here, 0))] = key;
        count += __popcll(here);
    }
    // four keys a lane, 0 for none; whether any was taken
    __device__ bool take(const uint64_t (&key)[4]) {
        static_assert(kLpMostTop + 256 <= kLpList && kLpList % 8 == 0, "");
        int more = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) more += __popcll(__ballot(key[e] >= least));
        if (!more) return false;
        if (count + more > kLpList) cut();
#pragma unroll
        for (int e = 0; e < 4; e++) add(key[e]);
        fence();
        return true;
    }
};

// One workgroup: a split of a row, per_split granules of 16 bytes (the first and the last of a row
// may be parts: rows begin at any f32). The last of a row's workgroups to arrive joins the
// splits in their order.
template <bool TOP>
__global__ __launch_bounds__(kLpThreads) void logprobs_kernel(LogprobArgs A) {
    __shared__ __attribute__((aligned(16))) uint64_t lists[TOP ? kLpWaves : 1][TOP ? kLpList + 128 : 1];
    __shared__ uint32_t largest[TOP ? kLpWaves : 1][TOP ? kLpRounds : 1][64];  // of a thread's 16 logits; then runs to read again
    __shared__ int counts[kLpWaves];
    __shared__ LpSums sums[kLpWaves];
    __shared__ uint32_t last;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t row = blockIdx.x / A.n_split;
    const int split = blockIdx.x % A.n_split;
    const float *x = A.x + row * A.ld;
    // places of logits: from the start of the row's first granule, of which `skew` elements lie before the row
    const uint32_t skew = (uint32_t)((uintptr_t)x >> 2 & 3), end = (uint32_t)A.n + skew;
    const uint32_t p0 = (uint32_t)min((int64_t)split * A.per_split * 4, (int64_t)end), p1 = (uint32_t)min((int64_t)(split + 1) * A.per_split * 4, (int64_t)end);

    LpSums S = LpSums::none();
    LpChoice C;
    C.list = lists[TOP ? wave : 0];
    C.n_top = A.n_top;
    constexpr uint32_t kRound = kLpThreads * kLpGroup * 4, kStep = kLpThreads * 4;
    auto load4 = [&](uint32_t p, float *v) {
        if (p >= skew && p + 4 <= p1) {
            const float4 f = *(const float4 *)(x + (p - skew));
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = p + e >= skew && p + e < p1 ? x[p + e - skew] : -INFINITY;
        }
    };
    auto key_at = [&](float v, uint32_t p) { return p >= skew && p < p1 ? lp_key(v, p - skew) : 0; };
    for (uint32_t first = p0; first < p1; first += kLpRounds * kRound) {
        const int rounds = (int)min((p1 - first + kRound - 1) / kRound, (uint32_t)kLpRounds);
        float v[4 * kLpGroup];
        for (int r = 0; r < rounds; r++) {
#pragma unroll
            for (int k = 0; k < kLpGroup; k++) load4(first + r * kRound + k * kStep + 4 * tid, v + 4 * k);
            float most = v[0];
#pragma unroll
            for (int e = 1; e < 4 * kLpGroup; e++) most = fmaxf(most, v[e]);
            if (most > S.m) S.raise(most);
            float t = 0.0f;
#pragma unroll
            for (int e = 0; e < 4 * kLpGroup; e++) {
                const float d = v[e] - S.m, p = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
                S.l += (double)p;
                t = fmaf(p, fmaxf(d, -1e4f), t);  // (where p is zero d may be infinite)
            }
            S.t += (double)t;
            if constexpr (TOP) largest[wave][r][lane] = lp_order(most);
        }
        if constexpr (!TOP) continue;
        // runs of 16, by the bounds of their largest key: its place is between the run's first and last
        // (where it is -inf all are, and the first has the largest key)
        LpChoice::fence();
        const uint32_t mine = first + 4 * tid;
        uint64_t low[2] = {0, 0};
        auto bound = [&](uint32_t o, uint32_t p, uint32_t to) { return p >= p1 ? 0 : lp_pair(o, o > kLpNone ? min(p + to, 0x7fffffffu) : p > skew ? p - skew : 0); };
        if (rounds == 1) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float most = v[8 * k];
#pragma unroll
                for (int e = 1; e < 8; e++) most = fmaxf(most, v[8 * k + e]);
                low[k] = bound(lp_order(most), mine + 2 * k * kStep, kStep + 3);
            }
        } else {
            for (int r = 0; r < rounds; r++) {
                const uint64_t k = bound(largest[wave][r][lane], mine + r * kRound, 3 * kStep + 3);
                if (r & 1) low[1] = max(low[1], k);
                else low[0] = max(low[0], k);
            }
        }
        C.limit(low[0], low[1]);
        if (rounds == 1 && (uint32_t)(C.least >> 31) > kLpNone) {  // they are still here
            const float border = lp_value(C.least);
            int more = 0;
#pragma unroll
            for (int e = 0; e < 4 * kLpGroup; e++) more += __popcll(__ballot(v[e] >= border));
            if (C.count + more <= kLpList) {
#pragma unroll
                for (int e = 0; e < 4 * kLpGroup; e++)
                    if (__any(v[e] >= border)) C.add(v[e] >= border ? lp_key(v[e], mine + e / 4 * kStep + e % 4 - skew) : 0);
                LpChoice::fence();
                continue;
            }
        }
        uint32_t reach = 0;
        for (int r = 0; r < rounds; r++) {
            const uint32_t p = mine + r * kRound;
            if (p < p1 && lp_pair(largest[wave][r][lane], p > skew ? p - skew : 0) >= C.least) reach |= 1u << r;
        }
        LpChoice::fence();
        uint16_t *runs = (uint16_t *)largest[wave];
        int n = 0;
        for (int r = 0; r < rounds; r++) {
            const uint64_t all = __ballot(reach >> r & 1);
            if (reach >> r & 1) runs[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0))] = r << 6 | lane;
            n += __popcll(all);
        }
        LpChoice::fence();
        for (int j = lane >> 2; __any(j < n); j += 16) {
            const int run = j < n ? runs[j] : 0;
            const uint32_t p = j < n ? first + (run >> 6) * kRound + (lane & 3) * kStep + 4 * (wave * 64 + (run & 63)) : p1;
            float v[4];
            load4(p, v);
            const uint64_t key[4] = {key_at(v[0], p), key_at(v[1], p + 1), key_at(v[2], p + 2), key_at(v[3], p + 3)};
            C.take(key);
        }
        LpChoice::fence();
    }
    // the wave's sums and choice; of several splits, those of all of them
    if constexpr (TOP)
        if (A.n_split > 1 || C.count > A.n_top) C.cut();
    if (A.n_split > 1) {
        const int64_t bytes = lp_part_bytes(A.n_top, A.n_split);
        const __amdgpu_buffer_rsrc_t part = __builtin_amdgcn_make_buffer_rsrc(A.part + row * bytes, (short)0, (int)bytes, 0x00020000);
        if constexpr (TOP)
            if (lane < A.n_top) {
                const uint64_t key = lane < C.count ? C.list[lane] : 0;
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(lp_u2, key), part,
                                                      A.n_split * 32 + ((split * kLpWaves + wave) * A.n_top + lane) * 8, 0, 16);
            }
        S.join<64>();
        if (lane == 0) sums[wave] = S;
        __syncthreads();
        S = sums[lane & (kLpWaves - 1)];
        S.join<kLpWaves>();
        if (tid == 0) {
            const double two[2] = {S.l, S.t};
            const lp_u4 first = {__builtin_bit_cast(uint32_t, S.m), 0, 0, 0};
            __builtin_amdgcn_raw_buffer_store_b128(first, part, split * 32, 0, 16);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(lp_u4, two), part, split * 32 + 16, 0, 16);
        }
        // (the order that agent.h describes)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __syncthreads();
        if (tid == 0) last = __hip_atomic_fetch_add(A.cnt + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)A.n_split - 1;
        __syncthreads();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        if (!last) return;
        if (tid == 0) __hip_atomic_store(A.cnt + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        S = LpSums::none();
        if (tid < A.n_split) {  // (at most kLpThreads)
            const lp_u4 a = __builtin_amdgcn_raw_buffer_load_b128(part, tid * 32, 0, 16);
            const lp_u4 b = __builtin_amdgcn_raw_buffer_load_b128(part, tid * 32 + 16, 0, 16);
            S.m = __builtin_bit_cast(float, a.x);
            S.l = __builtin_bit_cast(double, (uint64_t)b.y << 32 | b.x);
            S.t = __builtin_bit_cast(double, (uint64_t)b.w << 32 | b.z);
        }
        if constexpr (TOP) {
            C.count = 0;
            C.least = 1;
            // Lists in order: a list a lane, two or four, or, of few, a list to `lanes` lanes, four keys a lane
            // at a time from the lists' largest on, until none is among the largest.
            const int n = A.n_split * kLpWaves, ranks = n <= 64 ? 4 : n <= 128 ? 2 : 1;
            static_assert(kLpMostSplits * kLpWaves <= 256, "");
            int lanes = 1;
            while (2 * lanes * n <= 64) lanes *= 2;
            for (int r = lane % lanes; wave == 0; r += ranks * lanes) {
                uint64_t key[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int list = lane / lanes + e / ranks * 64, rank = r + e % ranks * lanes;
                    key[e] = 0;
                    if (list < n && rank < A.n_top)
                        key[e] = __builtin_bit_cast(uint64_t, __builtin_amdgcn_raw_buffer_load_b64(part, A.n_split * 32 + (list * A.n_top + rank) * 8, 0, 16));
                }
                if (r < lanes) C.limit(max(key[0], key[2]), max(key[1], key[3]));
                if (!C.take(key)) break;
            }
        }
    } else if constexpr (TOP) {
        if (lane == 0) counts[wave] = C.count;
        __syncthreads();
        if (wave == 0) {
            uint64_t key[4];
#pragma unroll
            for (int w = 0; w < kLpWaves; w++) key[w] = lane < counts[w] ? lists[w][lane] : 0;
            C.count = 0;
            LpChoice::fence();
            C.limit(max(key[0], key[1]), max(key[2], key[3]));
            C.take(key);
        }
    }
    S.join<64>();
    __syncthreads();
    if (lane == 0) sums[wave] = S;
    __syncthreads();
    S = sums[lane & (kLpWaves - 1)];
    S.join<kLpWaves>();
    // S.l is zero where no logit is above -inf: then there is no token to choose
    const bool none = S.l == 0.0;
    const double log_l = none ? 0.0 : log(S.l);
    auto logprob = [&](float v) { return none ? -INFINITY : (float)(((double)v - (double)S.m) - log_l); };
    if (A.logprob)
        for (int64_t i = tid; i < A.n_token; i += kLpThreads) {
            const int32_t id = A.token[row * A.n_token + i];
            if (id >= 0 && id < A.n) A.logprob[row * A.n_token + i] = logprob(x[id]);
        }
    if (A.entropy && tid == 0) A.entropy[row] = none ? 0.0f : (float)(log_l - S.t / S.l);
    if constexpr (TOP)
        if (wave == 0) {
            C.cut();
            if (lane < A.n_top) {
                const uint64_t key = C.list[lane];
                A.top_id[row * A.n_top + lane] = lp_index(key);
                A.top_logprob[row * A.n_top + lane] = logprob(lp_value(key));
            }
        }
}

}  // namespace sihip
