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
// logit and, of equal ones, falls with the index, so that no two are equal. A wave keeps a
// threshold that n_top of the keys it has seen reach, and puts the keys that reach it
// into a list in LDS. The first threshold is the n_topth largest of the lanes' largest keys
// (each lane has one that reaches it, so n_top keys do); a list that is full is cut to its n_top
// largest, found by counting for each key how many are larger, and the threshold goes up to
// the last of them. Most of the time no logit of a wave reaches the threshold, which costs a
// comparison a lane.
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
#pragma unroll 4
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
    // E keys a lane, 0 for none
    template <int E>
    __device__ void show(const uint64_t (&key)[E]) {
        const int lane = threadIdx.x & 63;
        uint64_t best = key[0];
#pragma unroll
        for (int e = 1; e < E; e++) best = key[e] > best ? key[e] : best;
        if (__popcll(__ballot(best >= least)) >= n_top) {
            uint64_t *all = list + kLpList;
            all[lane] = best;
            fence();
            const int rank = lp_larger(all, 64, best);
            const uint64_t last = __ballot(best && rank == n_top - 1);
            if (last) {
                const int from = __ffsll((unsigned long long)last) - 1;
                const uint64_t k = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(best >> 32), from) << 32 |
                                   (uint32_t)__builtin_amdgcn_readlane((int)best, from);
                least = k > least ? k : least;
            }
            fence();
        }
#pragma unroll
        for (int e = 0; e < E; e++) {
            uint64_t takes = __ballot(key[e] >= least);
            if (!takes) continue;
            if (count + __popcll(takes) > kLpList - 1) {
                cut();
                takes = __ballot(key[e] >= least);
            }
            if (key[e] >= least) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(takes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)takes, 0))] = key[e];
            count += __popcll(takes);
        }
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
    __shared__ __attribute__((aligned(16))) uint64_t chosen[TOP ? kLpWaves * kLpMostTop + 2 : 2];
    __shared__ LpSums sums[kLpWaves];
    __shared__ uint32_t last;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t row = blockIdx.x / A.n_split;
    const int split = blockIdx.x % A.n_split;
    const float *x = A.x + row * A.ld;
    const int skew = (int)((uintptr_t)x >> 2 & 3);  // elements of the first granule before the row
    const int64_t granules = (A.n + skew + 3) / 4;
    const int64_t g0 = split * A.per_split, g1 = min(g0 + A.per_split, granules);

    LpSums S = LpSums::none();
    LpChoice C;
    C.list = lists[TOP ? wave : 0];
    C.n_top = A.n_top;
    for (int64_t g = g0; g < g1; g += kLpThreads * kLpGroup) {
        float v[4 * kLpGroup];
#pragma unroll
        for (int k = 0; k < kLpGroup; k++) {
            const int64_t at = g + k * kLpThreads + tid, i = 4 * at - skew;
            if (at < g1 && i >= 0 && i + 4 <= A.n) {
                const float4 f = *(const float4 *)(x + i);
                v[4 * k] = f.x, v[4 * k + 1] = f.y, v[4 * k + 2] = f.z, v[4 * k + 3] = f.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) v[4 * k + e] = at < g1 && i + e >= 0 && i + e < A.n ? x[i + e] : -INFINITY;
            }
        }
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
        if constexpr (TOP) {
            if (__any(lp_key(most, 0) >= C.least)) {
                uint64_t key[4 * kLpGroup];
#pragma unroll
                for (int e = 0; e < 4 * kLpGroup; e++) {
                    const int64_t at = g + e / 4 * kLpThreads + tid, i = 4 * at - skew + e % 4;
                    key[e] = at < g1 && i >= 0 && i < A.n ? lp_key(v[e], (uint32_t)i) : 0;
                }
                C.show(key);
            }
        }
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
            C.cut();
            chosen[wave * A.n_top + min(lane, A.n_top - 1)] = 0;
            LpChoice::fence();
            if (lane < min(C.count, A.n_top)) chosen[wave * A.n_top + lane] = C.list[lane];
            if (tid < 2) chosen[kLpWaves * A.n_top + tid] = 0;
        }
        __syncthreads();
        S = sums[0];
#pragma unroll
        for (int w = 1; w < kLpWaves; w++) S.add(sums[w]);
        uint64_t key = 0;
        int rank = kLpMostTop;
        if constexpr (TOP) {
            if (tid < kLpWaves * A.n_top) {
                key = chosen[tid];
                if (key) rank = lp_larger(chosen, kLpWaves * A.n_top, key);
            }
            __syncthreads();
            if (tid < A.n_top) chosen[tid] = 0;
            __syncthreads();
            if (rank < A.n_top) chosen[rank] = key;
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
                C.show(key);
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
