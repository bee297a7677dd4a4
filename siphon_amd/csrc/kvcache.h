// The paged 8-bit KV cache: a step's bookkeeping (kv_plan_kernel), the write
// of new rows (kv_append_kernel) and the read-back of rows (kv_read_kernel).
//
// A page holds B tokens of every KV head. Codes are signed bytes, keys
// [page][head][token][dim], values [page][head][dim][token], and each page
// and head has one f32 scale for its keys and one for its values; a code
// times its scale is the value it stands for.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace sihip {

// ---- the plan of a step --------------------------------------------------------

constexpr int kPlanThreads = 1024;
constexpr int64_t kMaxRequests = 4096;  // three prefix arrays of them fit 48 KiB of LDS

struct PlanArgs {
    const int32_t *len, *add, *n_free;
    int32_t *free_pages, *table, *q_start, *kv_len, *pos, *n_free_out, *status;
    int64_t *slot;
    int64_t n_tok;
    int n_req, n_pages, max_blocks, shift;  // block = 1 << shift
};

// what the requests of a span add up to
struct PlanSum {
    int64_t tok, need, back;  // new tokens, pages taken, pages given back
};

__device__ inline PlanSum operator+(const PlanSum &a, const PlanSum &b) {
    return {a.tok + b.tok, a.need + b.need, a.back + b.back};
}

// One request's part, and what is wrong with it (SIHIP_KV_* bits).
__device__ inline PlanSum plan_request(const PlanArgs &A, int r, int &bad, int &len) {
    const int64_t n = A.len[r], add = A.add[r];
    const int64_t B = (int64_t)1 << A.shift;
    len = (int)n;
    if (n < 0 || add < -1) {
        bad |= 1;
        return {0, 0, 0};
    }
    const int64_t before = (n + B - 1) >> A.shift, after = (n + max(add, (int64_t)0) + B - 1) >> A.shift;
    if (after > A.max_blocks) {
        bad |= 2;
        return {0, 0, 0};
    }
    if (add < 0) return {0, 0, before};
    return {add, after - before, 0};
}

// Every workgroup adds up all requests itself (a few thousand words that
// stay in the L2), so that no workgroup waits for another; the tokens are
// spread over the grid and find their request by bisection in LDS. Nothing
// that a workgroup reads is written in the same launch: list entries at and
// past n_free and table entries of new blocks are only written.
__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(PlanArgs A) {
    extern __shared__ int32_t plan_lds[];
    __shared__ PlanSum wave_sum[kPlanThreads / 64];
    __shared__ int wave_bad[kPlanThreads / 64];
    int32_t *tok0 = plan_lds, *need0 = tok0 + A.n_req, *back0 = need0 + A.n_req;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int n_free = *A.n_free;

    // exclusive prefix sums: a span of requests per thread
    const int per = (A.n_req + kPlanThreads - 1) / kPlanThreads;
    const int r0 = min(tid * per, A.n_req), r1 = min(r0 + per, A.n_req);
    int bad = 0, unused;
    PlanSum own = {0, 0, 0};
    for (int r = r0; r < r1; r++) own = own + plan_request(A, r, bad, unused);
    PlanSum run = own;
    for (int d = 1; d < 64; d <<= 1) {
        const PlanSum o = {__shfl_up(run.tok, d), __shfl_up(run.need, d), __shfl_up(run.back, d)};
        if (lane >= d) run = run + o;
    }
    if (lane == 63) wave_sum[wave] = run;
    const bool any_bad1 = __any(bad & 1), any_bad2 = __any(bad & 2);
    if (lane == 0) wave_bad[wave] = (any_bad1 ? 1 : 0) | (any_bad2 ? 2 : 0);
    __syncthreads();
    PlanSum before = {0, 0, 0}, all = {0, 0, 0};
    int status = 0;
    for (int w = 0; w < kPlanThreads / 64; w++) {
        if (w == wave) before = all;
        all = all + wave_sum[w];
        status |= wave_bad[w];
    }
    if (all.tok > A.n_tok) status |= 4;
    if (n_free < 0 || n_free > A.n_pages || n_free + all.back > A.n_pages) status |= 16;
    else if (n_free + all.back < all.need) status |= 8;
    PlanSum at = before + run;  // inclusive; walk the span from its start
    at = {at.tok - own.tok, at.need - own.need, at.back - own.back};
    for (int r = r0; r < r1; r++) {
        const bool first = blockIdx.x == 0;
        int len;
        int b = 0;
        const PlanSum s = plan_request(A, r, b, len);
        if (status) {
            if (first) {
                A.q_start[r] = 0;
                A.kv_len[r] = len;
            }
            continue;
        }
        tok0[r] = (int)at.tok;
        need0[r] = (int)at.need;
        back0[r] = (int)at.back;
        if (first) {
            A.q_start[r] = (int)at.tok;
            A.kv_len[r] = A.add[r] < 0 ? 0 : len + (int)s.tok;
        }
        at = at + s;
    }
    const int n_out = status ? n_free : (int)(n_free + all.back - all.need);
    if (blockIdx.x == 0 && tid == 0) {
        A.q_start[A.n_req] = status ? 0 : (int)all.tok;
        *A.n_free_out = n_out;
        *A.status = status;
    }
    __syncthreads();

    // the last request whose prefix is at most i (of equal ones the last:
    // those before it hold nothing)
    auto find = [&](const int32_t *prefix, int i) {
        int lo = 0, hi = A.n_req;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] <= i) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    // entry i of the free list with the pages given back behind it
    auto list = [&](int i) {
        if (i < n_free) return A.free_pages[i];
        const int r = find(back0, i - n_free);
        return A.table[(int64_t)r * A.max_blocks + (i - n_free - back0[r])];
    };
    const int64_t step = (int64_t)gridDim.x * kPlanThreads;
    const int64_t first = (int64_t)blockIdx.x * kPlanThreads + tid;
    if (!status)
        for (int64_t i = n_free + first; i < n_out; i += step) A.free_pages[i] = list((int)i);
    const int top = (int)(n_free + all.back) - 1;
    for (int64_t t = first; t < A.n_tok; t += step) {
        if (status || t >= all.tok) {
            A.slot[t] = -1;
            A.pos[t] = -1;
            continue;
        }
        const int r = find(tok0, (int)t);
        const int len = A.len[r], pos = len + (int)(t - tok0[r]);
        const int old = (int)(((int64_t)len + (1 << A.shift) - 1) >> A.shift), b = pos >> A.shift;
        const int64_t entry = (int64_t)r * A.max_blocks + b;
        const int off = pos & ((1 << A.shift) - 1);
        const int page = b < old ? A.table[entry] : list(top - (need0[r] + b - old));
        // a new block's first token is always among the new ones
        if (b >= old && off == 0) A.table[entry] = page;
        A.slot[t] = page >= 0 && page < A.n_pages ? ((int64_t)page << A.shift) + off : -1;
        A.pos[t] = pos;
    }
}

// ---- the cache and a step's requests, as the kernels see them ---------------------

struct CacheArgs {
    int8_t *k, *v;
    float *ks, *vs;
    int64_t n_pages;
    int n_kv, hd, shift;
};

struct BatchArgs {
    const int32_t *q_start, *kv_len, *table;
    int64_t n_tok;
    int max_blocks, max_q, max_kv;
};

// The new tokens of request r as rows q0 .. q0 + n - 1, at positions p0 ..;
// n = 0 where the device's numbers do not describe any.
struct Span {
    int64_t q0;
    int n, p0, end;
};

__device__ inline Span request_span(const BatchArgs &A, int r) {
    const int64_t q0 = A.q_start[r], q1 = A.q_start[r + 1], end = A.kv_len[r];
    Span s = {q0, 0, 0, (int)end};
    if (q0 < 0 || q1 <= q0 || q1 > A.n_tok || q1 - q0 > end) return s;
    s.n = (int)(q1 - q0);
    s.p0 = (int)(end - s.n);
    return s;
}

// ---- append ------------------------------------------------------------------------

constexpr int kAppendThreads = 256;

struct AppendArgs {
    CacheArgs C;
    BatchArgs R;
    const float *k, *v;
    int64_t ldk, ldv;
    int blocks;  // most blocks of a request that get new tokens
};

// Magnitudes below this count as zero, so that a scale's reciprocal and the
// remainders below stay in the range of f32.
constexpr float kTinyAmax = 0x1p-100f;

// x / scale rounded to an integer, ties to even, exactly: the product with
// the rounded reciprocal is off by at most one step, and one FMA gives the
// sign of the remainder at the border between two steps without error.
__device__ inline int quantize_exact(float x, float scale, float inv) {
    if (!(fabsf(x) < INFINITY)) return x != x || scale == 0.0f ? 0 : x > 0.0f ? 127 : -127;
    if (scale == 0.0f) return 0;
    float q = rintf(x * inv);
    const float up = fmaf(-(q + 0.5f), scale, x), down = fmaf(-(q - 0.5f), scale, x);
    const bool odd = ((int)q & 1) != 0;
    if (up > 0.0f || (up == 0.0f && odd)) q += 1.0f;
    else if (down < 0.0f || (down == 0.0f && odd)) q -= 1.0f;
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// code * was / now rounded to an integer, ties to even, exactly: the product
// of a code and an f32 has 31 bits, so f64 holds it and the remainders.
__device__ inline int requantize_exact(int code, float was, float now, double inv) {
    const double a = (double)code * (double)was;
    double q = rint(a * inv);
    const double up = fma(-(q + 0.5), (double)now, a), down = fma(-(q - 0.5), (double)now, a);
    const bool odd = ((int)q & 1) != 0;
    if (up > 0.0 || (up == 0.0 && odd)) q += 1.0;
    else if (down < 0.0 || (down == 0.0 && odd)) q -= 1.0;
    return (int)q;
}

// One workgroup: one page, one KV head, keys (z = 0) or values (z = 1). The
// scale of a page grows with its tokens: the largest magnitude of the new
// rows over 127, or what it was where that is more; codes of tokens that
// were there are rounded again when it grows. A page whose first token is new
// starts from nothing. Bytes behind the last token are left as they are.
__global__ __launch_bounds__(kAppendThreads) void kv_append_kernel(AppendArgs A) {
    __shared__ float wave_max[kAppendThreads / 64];
    const int h = blockIdx.x % A.C.n_kv, j = blockIdx.x / A.C.n_kv, r = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const int tid = threadIdx.x, B = 1 << A.C.shift, hd = A.C.hd;
    const Span s = request_span(A.R, r);
    const int b = (s.p0 >> A.C.shift) + j;
    const int64_t base = (int64_t)b << A.C.shift;
    if (s.n == 0 || base >= s.end || b >= A.R.max_blocks) return;
    const int64_t page = A.R.table[(int64_t)r * A.R.max_blocks + b];
    if (page < 0 || page >= A.C.n_pages) return;
    const int lo = (int)max((int64_t)s.p0 - base, (int64_t)0), hi = (int)min((int64_t)s.end - base, (int64_t)B);
    const int64_t ld = is_v ? A.ldv : A.ldk;
    // row of the page's token 0 (may lie before the first row)
    const float *x = (is_v ? A.v : A.k) + (s.q0 + base - s.p0) * ld + (int64_t)h * hd;
    float *sp = (is_v ? A.C.vs : A.C.ks) + page * A.C.n_kv + h;
    int8_t *codes = (is_v ? A.C.v : A.C.k) + (page * A.C.n_kv + h) * ((int64_t)hd << A.C.shift);
    const float was = lo > 0 ? *sp : 0.0f;

    float top = 0.0f;
    for (int i = tid; i < (hi - lo) * hd; i += kAppendThreads) {
        const float a = fabsf(x[(int64_t)(lo + i / hd) * ld + i % hd]);
        if (a < INFINITY) top = fmaxf(top, a);
    }
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if ((tid & 63) == 0) wave_max[tid >> 6] = top;
    __syncthreads();
    for (int w = 0; w < kAppendThreads / 64; w++) top = fmaxf(top, wave_max[w]);
    const float now = fmaxf(was, top < kTinyAmax ? 0.0f : top / 127.0f);
    const bool grew = now > was;
    const float inv = now > 0.0f ? 1.0f / now : 0.0f;
    const double inv64 = now > 0.0f ? 1.0 / (double)now : 0.0;

    // 16 bytes a thread: dims of one token (keys), tokens of one dim (values)
    for (int u = tid; u < (hd << A.C.shift) / 16; u += kAppendThreads) {
        const int outer = is_v ? u % hd : u / (hd / 16);
        const int inner = (is_v ? u / hd : u % (hd / 16)) * 16;
        const int t0 = is_v ? inner : outer, t1 = is_v ? inner + 16 : outer + 1;
        const bool has_new = t0 < hi && t1 > lo, has_old = t0 < lo;
        if (!has_new && !(has_old && grew)) continue;
        int8_t *at = codes + (is_v ? ((int64_t)outer << A.C.shift) + inner : (int64_t)outer * hd + inner);
        union {
            uint4 w;
            int8_t c[16];
        } buf;
        if (t0 < lo || t1 > hi) buf.w = *(const uint4 *)at;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int t = is_v ? inner + e : outer, d = is_v ? outer : inner + e;
            if (t >= lo && t < hi) buf.c[e] = (int8_t)quantize_exact(x[(int64_t)t * ld + d], now, inv);
            else if (t < lo && grew) buf.c[e] = (int8_t)requantize_exact(buf.c[e], was, now, inv64);
        }
        *(uint4 *)at = buf.w;
    }
    if (tid == 0 && (grew || lo == 0)) *sp = now;
}

// ---- read ---------------------------------------------------------------------------

constexpr int kReadThreads = 256;
constexpr int kReadRows = 16;

struct ReadArgs {
    CacheArgs C;
    const int64_t *slots;
    float *k, *v;
    int64_t n, ldk, ldv;
};

// One workgroup: kReadRows slots of one KV head, keys and values.
__global__ __launch_bounds__(kReadThreads) void kv_read_kernel(ReadArgs A) {
    const int h = blockIdx.y, hd = A.C.hd, B = 1 << A.C.shift;
    const int64_t i0 = (int64_t)blockIdx.x * kReadRows;
    for (int u = threadIdx.x; u < kReadRows * hd; u += kReadThreads) {
        const int64_t i = i0 + u / hd;
        const int d = u % hd;
        if (i >= A.n) break;
        const int64_t slot = A.slots[i], page = slot >> A.C.shift;
        if (slot < 0 || page >= A.C.n_pages) continue;
        const int off = (int)(slot & (B - 1));
        const int64_t ph = page * A.C.n_kv + h, at = ph * ((int64_t)hd << A.C.shift);
        A.k[i * A.ldk + (int64_t)h * hd + d] = (float)A.C.k[at + (int64_t)off * hd + d] * A.C.ks[ph];
        A.v[i * A.ldv + (int64_t)h * hd + d] = (float)A.C.v[at + ((int64_t)d << A.C.shift) + off] * A.C.vs[ph];
    }
}

}  // namespace sihip
