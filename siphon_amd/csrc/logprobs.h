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
// The most likely: of a logit and its index a key is made, a 64-bit number that grows with the
// logit and, of equal ones, falls with the index, so that no two are equal. The pass itself keeps the
// largest of each thread's 16 logits at a time, no more. Every kLpRounds of them a wave finds the n_topth largest of
// its lanes' largest (each lane has one that reaches it, so n_top keys do): what is below is not among the most
// likely. The few runs of 16 that reach it are read again, four lanes a run, and the keys that reach it
// go to a list in LDS. A list that is full is cut to its n_top largest, found by counting for each key how
// many are larger, and the threshold goes up to the last of them.
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
    uint8_t *part;      // [row][split]: maximum, sums, keys
    uint32_t *cnt;      // of each row: splits that have arrived, zero between launches
};

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr int kLpMostTop = 64;  // keys that a wave can choose with a lane each
constexpr int kLpList = 192;
constexpr int kLpGroup = 4;     // 16-byte loads of a thread at a time
constexpr int kLpRounds = 8;    // of them between choices

// bytes of a split's part
__host__ __device__ inline int64_t lp_part_bytes(int n_top) { return 32 + (int64_t)(n_top + 1) / 2 * 16; }

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
    __device__ void add(LpSums o) {
        const float to = fmaxf(m, o.m);
        raise(to);
        o.raise(to);
        l += o.l;
        t += o.t;
    }
};

// NaN counts as -inf, -0 as 0
__device__ inline uint64_t lp_key(float x, uint32_t index) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x == x ? x + 0.0f : -INFINITY);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xffffffffu - index);
}
__device__ inline float lp_value(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ inline int32_t lp_index(uint64_t key) { return (int32_t)(0xffffffffu - (uint32_t)key); }

// how many of n keys in LDS are larger (n is padded to even with zeros)
__device__ inline int lp_larger(const uint64_t *keys, int n, uint64_t key) {
    int k = 0;
#pragma unroll 8
    for (int i = 0; i < n; i += 2) {
        const ulonglong2 o = *(const ulonglong2 *)(keys + i);
        k += (o.x > key) + (o.y > key);
    }
    return k;
}

// A wave's choice of the n_top largest of the keys it is shown.
struct LpChoice {
    uint64_t *list;  // of the wave, in LDS: kLpList and 64 more
    int n_top, count = 0;
    uint64_t least = 1;  // keys below it are not among the largest (0 is no key)

    // a wave's LDS accesses are in order; the compiler is told not to move them
    static __device__ void fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

    // cuts the list to its n_top largest, in order
    __device__ void cut() {
        const int lane = threadIdx.x & 63;
        uint64_t own[kLpList / 64];
        int rank[kLpList / 64];
        if (lane == 0) list[count] = 0;
        fence();
#pragma unroll
        for (int i = 0; i < kLpList / 64; i++) {
            const int at = lane + 64 * i;
            own[i] = at < count ? list[at] : 0;
            rank[i] = own[i] ? lp_larger(list, count, own[i]) : n_top;
        }
        fence();
#pragma unroll
        for (int i = 0; i < kLpList / 64; i++)
            if (rank[i] < n_top) list[rank[i]] = own[i];
        fence();
        if (count >= n_top) {
            count = n_top;
            const uint64_t last = list[n_top - 1];
            least = last > least ? last : least;
        }
    }
    // raises the threshold to the n_topth largest of a key of each lane, that is reached by one of its keys
    __device__ void limit(uint64_t key) {
        const int lane = threadIdx.x & 63;
        if (__popcll(__ballot(key >= least)) < n_top) return;
        uint64_t *all = list + kLpList;
        all[lane] = key;
        fence();
        const int rank = lp_larger(all, 64, key);
        const uint64_t last = __ballot(key && rank == n_top - 1);
        if (last) {
            const int from = __ffsll((unsigned long long)last) - 1;
            const uint64_t k = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), from) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((int)key, from);
            least = k > least ? k : least;
        }
        fence();
    }
    // a key a lane, 0 for none
    __device__ void take(uint64_t key) {
        uint64_t takes = __ballot(key >= least);
        if (!takes) return;
        if (count + __popcll(takes) > kLpList - 1) {
            cut();
            takes = __ballot(key >= least);
        }
        if (key >= least) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(takes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)takes, 0))] = key;
        count += __popcll(takes);
        fence();
    }
};

typedef uint32_t lp_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t lp_u2 __attribute__((ext_vector_type(2)));

// One workgroup: a split of a row, per_split granules of 16 bytes (the first and the last of a row
// may be parts: rows begin at any f32). The last of a row's workgroups to arrive joins the
// splits in their order.
template <bool TOP>
__global__ __launch_bounds__(kLpThreads) void logprobs_kernel(LogprobArgs A) {
    __shared__ __attribute__((aligned(16))) uint64_t lists[TOP ? kLpWaves : 1][TOP ? kLpList + 64 : 1];
    __shared__ float largest[TOP ? kLpWaves : 1][TOP ? kLpRounds : 1][64];  // of a thread's 16 logits; then runs to read again
    __shared__ uint64_t chosen[kLpMostTop];
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
            if constexpr (TOP) largest[wave][r][lane] = most;
        }
        if constexpr (!TOP) continue;
        if (rounds == 1) {  // they are still here
            uint64_t key[4 * kLpGroup], low = 0;
#pragma unroll
            for (int e = 0; e < 4 * kLpGroup; e++) {
                key[e] = key_at(v[e], first + e / 4 * kStep + 4 * tid + e % 4);
                low = key[e] > low ? key[e] : low;
            }
            C.limit(low);
#pragma unroll
            for (int e = 0; e < 4 * kLpGroup; e++) C.take(key[e]);
            continue;
        }
        // runs of 16, by the bounds of their largest key: its place is between the run's first and last
        LpChoice::fence();
        const uint32_t mine = first + 4 * tid;
        uint64_t low = 0;
        for (int r = 0; r < rounds; r++) {
            const uint32_t p = mine + r * kRound;
            const uint64_t k = p < p1 ? lp_key(largest[wave][r][lane], p + 3 * kStep + 3) : 0;
            low = k > low ? k : low;
        }
        C.limit(low);
        uint32_t reach = 0;
        for (int r = 0; r < rounds; r++) {
            const uint32_t p = mine + r * kRound;
            if (p < p1 && lp_key(largest[wave][r][lane], p > skew ? p - skew : 0) >= C.least) reach |= 1u << r;
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
#pragma unroll
            for (int e = 0; e < 4; e++) C.take(key_at(v[e], p + e));
        }
        LpChoice::fence();
    }
    // the workgroup's sums and choice
    auto join = [&]() {
        for (int d = 1; d < 64; d <<= 1) {
            LpSums o;
            o.m = __shfl_xor(S.m, d);
            o.l = __shfl_xor(S.l, d);
            o.t = __shfl_xor(S.t, d);
            S.add(o);
        }
        if (lane == 0) sums[wave] = S;
        if constexpr (TOP) {
            if (C.count > 64) C.cut();
            if (lane == 0) {
                counts[wave] = C.count;
                C.list[C.count] = 0;
            }
            if (tid < A.n_top) chosen[tid] = 0;
        }
        __syncthreads();
        S = sums[0];
#pragma unroll
        for (int w = 1; w < kLpWaves; w++) S.add(sums[w]);
        if constexpr (TOP) {
            if (lane < C.count) {
                const uint64_t key = C.list[lane];
                int rank = 0;
#pragma unroll
                for (int w = 0; w < kLpWaves; w++) rank += lp_larger(lists[w], counts[w], key);
                if (rank < A.n_top) chosen[rank] = key;
            }
        }
        __syncthreads();
    };
    join();
    if (A.n_split > 1) {
        const int64_t bytes = lp_part_bytes(A.n_top);
        const __amdgpu_buffer_rsrc_t part = __builtin_amdgcn_make_buffer_rsrc(A.part + row * A.n_split * bytes, (short)0,
                                                                              (int)(A.n_split * bytes), 0x00020000);
        const uint32_t to = split * (uint32_t)bytes;
        if (tid == 0) {
            const double two[2] = {S.l, S.t};
            const lp_u4 first = {__builtin_bit_cast(uint32_t, S.m), 0, 0, 0};
            __builtin_amdgcn_raw_buffer_store_b128(first, part, (int)to, 0, 16);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(lp_u4, two), part, (int)to + 16, 0, 16);
        }
        if constexpr (TOP)
            if (tid < A.n_top) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(lp_u2, chosen[tid]), part, (int)to + 32 + 8 * tid, 0, 16);
        // (the order that agent.h describes)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __syncthreads();
        if (tid == 0) last = __hip_atomic_fetch_add(A.cnt + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)A.n_split - 1;
        __syncthreads();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        if (!last) return;
        S = LpSums::none();
        C.count = 0;
        C.least = 1;
        for (int k = tid; k < A.n_split; k += kLpThreads) {
            LpSums o;
            const lp_u4 a = __builtin_amdgcn_raw_buffer_load_b128(part, (int)(k * bytes), 0, 16);
            const lp_u4 b = __builtin_amdgcn_raw_buffer_load_b128(part, (int)(k * bytes) + 16, 0, 16);
            o.m = __builtin_bit_cast(float, a.x);
            o.l = __builtin_bit_cast(double, (uint64_t)b.y << 32 | b.x);
            o.t = __builtin_bit_cast(double, (uint64_t)b.w << 32 | b.z);
            S.add(o);
        }
        if constexpr (TOP) {
            for (int k0 = 0; k0 < A.n_split * A.n_top; k0 += 4 * kLpThreads) {
                uint64_t key[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = k0 + e * kLpThreads + tid;
                    key[e] = 0;
                    if (i < A.n_split * A.n_top) {
                        const lp_u2 w = __builtin_amdgcn_raw_buffer_load_b64(part, (int)(i / A.n_top * bytes + 32 + i % A.n_top * 8), 0, 16);
                        key[e] = (uint64_t)w.y << 32 | w.x;
                    }
                }
                uint64_t low = key[0];
#pragma unroll
                for (int e = 1; e < 4; e++) low = key[e] > low ? key[e] : low;
                C.limit(low);
#pragma unroll
                for (int e = 0; e < 4; e++) C.take(key[e]);
            }
        }
        __syncthreads();
        join();
        if (tid == 0) __hip_atomic_store(A.cnt + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
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
        if (tid < A.n_top) {
            const uint64_t key = chosen[tid];
            A.top_id[row * A.n_top + tid] = lp_index(key);
            A.top_logprob[row * A.n_top + tid] = logprob(lp_value(key));
        }
}

}  // namespace sihip
