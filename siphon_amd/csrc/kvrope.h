// The write of new rows into the paged 8-bit cache with the rotation on the
// way (rope.h): kv_append_kernel (kvcache.h) on rotated keys, and in the same
// launch the step's queries.
#pragma once

#include "kvcache.h"
#include "rope.h"

namespace sihip {

struct RopeKeys {
    static constexpr bool kAsTheyAre = false;
    RopeArgs P;
    bool wide;  // rows of k and their heads are 16-byte aligned

    // 16 dims, from `inner` on, of the key row x at position p
    __device__ void load(const float *x, int p, int inner, float *val) const {
        const float *cs = P.table + (int64_t)p * (2 * P.pairs);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float4 y = rope_load4(P, x, cs, inner + 4 * e, wide);
            val[4 * e] = y.x, val[4 * e + 1] = y.y, val[4 * e + 2] = y.z, val[4 * e + 3] = y.w;
        }
    }
};

struct AppendRopeArgs {
    AppendArgs A;
    RopeArgs P;
    RopeQueries Q;  // Q.q NULL: none
};

// A workgroup: one page of new tokens and one KV head, keys (z = 0), values (1) or the
// queries of that KV head (2).
template <int U, int THREADS>
__global__ __launch_bounds__(THREADS) void kv_append_rope_kernel(AppendRopeArgs R) {
    const AppendArgs &A = R.A;
    if (blockIdx.z < 2) {
        kv_append_page<U, THREADS>(A, RopeKeys{R.P, A.k_wide});
        return;
    }
    const PageSpan g = page_span(A.R, blockIdx.y, blockIdx.x / A.C.n_kv, A.C.shift);
    if (g.lo < g.hi)
        rope_queries<THREADS>(R.P, R.Q, A.C.hd, blockIdx.x % A.C.n_kv, g.q0, g.p0, (int)(g.base - g.p0) + g.lo,
                              (int)(g.base - g.p0) + g.hi);
}

}  // namespace sihip
