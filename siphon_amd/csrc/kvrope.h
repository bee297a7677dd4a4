// The write of new rows into the paged 8-bit cache with the rotation on the
// way (rope.h): kv_append_kernel (kvcache.h) on rotated keys, and in the same
// launch the step's queries.
//
// Bound by memory: 5 prompt chunks of up to 2047 tokens, 40 heads of 128 on 8, 293 MB in 59 us (4.9 TB/s; the queries are
// four fifths of it, 27 us without them); one token each for 64 requests 7 us, of which an empty launch takes
// 3.5. Queries are a layer of workgroups of their own, a page's tokens and a KV head each, because keys and values
// need the whole page's maximum first, and they nothing.
#pragma once

#include "kvcache.h"
#include "rope.h"

namespace sihip {

struct KeyRope {
    RopeArgs P;
    RopeQueries Q;  // Q.q NULL: none

    // 16 dims, from `inner` on, of the key row x at position p; wide: rows and heads are 16-byte aligned
    __device__ void key(const float *x, int p, int inner, bool wide, float *val) const {
        const float *cs = P.table + (int64_t)p * (2 * P.pairs);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float4 y = rope_load4(P, x, cs, inner + 4 * e, wide);
            val[4 * e] = y.x, val[4 * e + 1] = y.y, val[4 * e + 2] = y.z, val[4 * e + 3] = y.w;
        }
    }

    // the queries of KV head h at a page's new tokens
    template <int THREADS>
    __device__ void queries(const PageSpan &g, int hd, int h) const {
        const int first = (int)(g.base - g.p0);
        rope_queries<THREADS>(P, Q, hd, h, g.q0, g.p0, first + g.lo, first + g.hi);
    }
};

}  // namespace sihip
