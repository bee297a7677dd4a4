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
//
// Nothing but dependent loads bounds it: 64 requests with a token each take
// 6.0 us, 1000 with 24600 tokens 8.9 us, a launch with nothing to do 3.5 us.
// With 1024 threads the 64 take 6.3 us.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_plan_kernel(PlanArgs A) {
    extern __shared__ int32_t plan_lds[];
    __shared__ PlanSum wave_sum[THREADS / 64];
    __shared__ int wave_bad[THREADS / 64];
    int32_t *tok0 = plan_lds, *need0 = tok0 + A.n_req, *back0 = need0 + A.n_req;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int n_free = *A.n_free;

    // exclusive prefix sums: a span of requests per thread
    const int per = (A.n_req + THREADS - 1) / THREADS;
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
    for (int w = 0; w < THREADS / 64; w++) {
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
    const int64_t step = (int64_t)gridDim.x * THREADS;
    const int64_t first = (int64_t)blockIdx.x * THREADS + tid;
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

// The tokens lo .. hi - 1 of the jth page that gets new tokens of request r, which
// begins at position base; row q0 is position p0. None (lo = hi): the request has no
// such page, or only tokens past the host's bounds, which are not written (max_kv is at
// most what the table's rows hold).
struct PageSpan {
    int64_t q0, base;
    int p0, lo, hi, block;  // block: of the request's table row
};

__device__ inline PageSpan page_span(const BatchArgs &A, int r, int j, int shift) {
    const Span s = request_span(A, r);
    const int end = min(s.p0 + min(s.n, A.max_q), A.max_kv), b = (s.p0 >> shift) + j;
    const int64_t base = (int64_t)b << shift;
    PageSpan g = {s.q0, base, s.p0, 0, 0, b};
    if (end <= s.p0 || base >= end) return g;
    g.lo = (int)max((int64_t)s.p0 - base, (int64_t)0);
    g.hi = (int)min((int64_t)end - base, (int64_t)1 << shift);
    return g;
}

// ---- append ------------------------------------------------------------------------

struct AppendArgs {
    CacheArgs C;
    BatchArgs R;
    const float *k, *v;
    int64_t ldk, ldv;
    bool k_wide;  // rows of k and their heads are 16-byte aligned
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

// 16 values to codes. The sum with 1.5 2^23 leaves the product rounded to an
// integer, ties to even, in the low bits; what is within 10^-4 of a border (or
// no number) is rounded exactly, all 16 of the thread.
__device__ inline void quantize16(const float *x, float scale, float inv, uint32_t *w) {
    constexpr float kMagic = 12582912.0f;
    bool clear = true;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float r = fmaf(x[4 * i + e], inv, kMagic);
            const float d = fabsf(fmaf(x[4 * i + e], inv, kMagic - r));
            clear &= d <= 0.4999f;
            b[e] = __builtin_bit_cast(uint32_t, r);
        }
        const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u);
        w[i] = lo | hi << 16;
    }
    if (clear) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w[i] = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) w[i] |= (uint32_t)(uint8_t)quantize_exact(x[4 * i + e], scale, inv) << (8 * e);
    }
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
//
// A thread has 16 bytes of the page: 16 dims of a token (keys) or 16 tokens of
// a dim (values, so that the lanes of a wave read a row each time and write
// whole granules of the transposed page), U times; the f32 values stay in
// registers from the search for the largest to their rounding.
//
// Bound by memory: each new row is read once, each touched page written once.
// 5 prompt chunks, 5760 rows of 8 heads of 128, pages of 64: 59 MB in 19.5 us
// (3.0 TB/s); one 16-byte unit a thread, not 2 of half as many threads (22 us),
// as long as 1024 threads reach. One new token for 64 requests: 7.5 us, of
// which a launch with nothing to do takes 3.5; the rest are dependent loads.
// Where every page's scale grows, and its old codes are rounded again in f64,
// 10.3 us, and 21.3 for the chunks.
//
// Rope: none, or KeyRope (kvrope.h), by which keys are rotated on the way and a third layer of
// workgroups rotates the queries. (The body as a function that two kernels call took 82
// registers in place of 52, and prompts of 1000 tokens 37 us in place of 35.)
template <int U, int THREADS, class... Rope>
__global__ __launch_bounds__(THREADS) void kv_append_kernel(AppendArgs A, Rope... rope) {
    constexpr bool kRotates = sizeof...(Rope) > 0;
    __shared__ float wave_max[THREADS / 64];
    const int h = blockIdx.x % A.C.n_kv, j = blockIdx.x / A.C.n_kv, r = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const int tid = threadIdx.x, hd = A.C.hd;
    const PageSpan g = page_span(A.R, r, j, A.C.shift);
    const int64_t base = g.base;
    const int lo = g.lo, hi = g.hi;
    if (lo >= hi) return;
    if constexpr (kRotates) {
        if (blockIdx.z == 2) {
            (rope.template queries<THREADS>(g, hd, h), ...);
            return;
        }
    }
    const int64_t page = A.R.table[(int64_t)r * A.R.max_blocks + g.block];
    if (page < 0 || page >= A.C.n_pages) return;
    const int64_t ld = is_v ? A.ldv : A.ldk;
    // row of the page's token 0 (may lie before the first row)
    const float *x = (is_v ? A.v : A.k) + (g.q0 + base - g.p0) * ld + (int64_t)h * hd;
    float *sp = (is_v ? A.C.vs : A.C.ks) + page * A.C.n_kv + h;
    int8_t *codes = (is_v ? A.C.v : A.C.k) + (page * A.C.n_kv + h) * ((int64_t)hd << A.C.shift);
    const float was = lo > 0 ? *sp : 0.0f;

    const int units = (hd << A.C.shift) / 16, per_token = hd / 16;
    float val[U][16], top = 0.0f;
    union Codes {
        uint4 w;
        int8_t c[16];
    } buf[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int u = tid + THREADS * i;
        const int outer = is_v ? u % hd : u / per_token, inner = (is_v ? u / hd : u % per_token) * 16;
        const int t0 = is_v ? inner : outer, t1 = is_v ? inner + 16 : outer + 1;
        const bool has_new = u < units && t0 < hi && t1 > lo;
        if (u < units && t0 < hi && (t0 < lo || t1 > hi)) buf[i].w = *(const uint4 *)(codes + (is_v ? (outer << A.C.shift) + inner : outer * hd + inner));
        if (!has_new) {
#pragma unroll
            for (int e = 0; e < 16; e++) val[i][e] = 0.0f;
        } else if (is_v) {
#pragma unroll
            for (int e = 0; e < 16; e++) val[i][e] = inner + e >= lo && inner + e < hi ? x[(int64_t)(inner + e) * ld + outer] : 0.0f;
        } else if constexpr (kRotates) {
            (rope.key(x + (int64_t)outer * ld, (int)base + outer, inner, A.k_wide, val[i]), ...);
        } else if (A.k_wide) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float4 y = ((const float4 *)(x + (int64_t)outer * ld + inner))[e];
                val[i][4 * e] = y.x, val[i][4 * e + 1] = y.y, val[i][4 * e + 2] = y.z, val[i][4 * e + 3] = y.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) val[i][e] = x[(int64_t)outer * ld + inner + e];
        }
    }
#pragma unroll
    for (int i = 0; i < U; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float a = fabsf(val[i][e]);
            top = fmaxf(top, a < INFINITY ? a : 0.0f);
        }
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if ((tid & 63) == 0) wave_max[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) top = fmaxf(top, wave_max[w]);
    const float now = fmaxf(was, top < kTinyAmax ? 0.0f : top / 127.0f);
    const bool grew = now > was;
    const float inv = now > 0.0f ? 1.0f / now : 0.0f;

#pragma unroll
    for (int i = 0; i < U; i++) {
        const int u = tid + THREADS * i;
        const int outer = is_v ? u % hd : u / per_token, inner = (is_v ? u / hd : u % per_token) * 16;
        const int t0 = is_v ? inner : outer, t1 = is_v ? inner + 16 : outer + 1;
        const bool has_new = t0 < hi && t1 > lo, has_old = t0 < lo;
        if (u >= units || !(has_new || (has_old && grew))) continue;
        if (has_old && grew) {
            const double inv64 = 1.0 / (double)now;
#pragma unroll
            for (int e = 0; e < 16; e++)
                if ((is_v ? inner + e : outer) < lo) buf[i].c[e] = (int8_t)requantize_exact(buf[i].c[e], was, now, inv64);
        }
        Codes q;
        quantize16(val[i], now, inv, &q.w.x);
        if (t0 >= lo && t1 <= hi) {
            buf[i] = q;
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int t = is_v ? inner + e : outer;
                buf[i].c[e] = t >= lo && t < hi ? q.c[e] : buf[i].c[e];
            }
        }
        *(uint4 *)(codes + (is_v ? (outer << A.C.shift) + inner : outer * hd + inner)) = buf[i].w;
    }
    if (tid == 0 && (grew || lo == 0)) *sp = now;
}

// ---- read ---------------------------------------------------------------------------

constexpr int kReadThreads = 256;

struct ReadArgs {
    CacheArgs C;
    const int64_t *slots;
    float *k, *v;
    int64_t n, ldk, ldv;
    bool wide;  // rows of k and v and their heads are 16-byte aligned
};

// bytes `from` .. from + 15 of 32
__device__ inline uint4 read_window(uint4 a, uint4 b, int from) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int s = 4; s; s >>= 1)
        if (from & (4 * s))
#pragma unroll
            for (int i = 0; i + s < 8; i++) w[i] = w[i + s];
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = __builtin_amdgcn_alignbyte(w[i + 1], w[i], from & 3);
    return uint4{o[0], o[1], o[2], o[3]};
}

// One workgroup: ROWS slots of one KV head, keys (z = 0): four dims of a
// slot a thread; or values: two dims of 16 slots a thread, so that the lanes of
// a wave write rows. 16 slots that go on from one another lie in one or two
// 16-token segments of the transposed pages: two loads a dim. Any others are
// read byte by byte, all 32 loads of a thread before the first use.
//
// Bound by memory: 4 requests of 7000 tokens, 8 heads of 128: 97 MB in 22.5 us
// (4.3 TB/s, a large copy 4.8); a byte at a time for all slots 43 us. 600
// tokens of 4 heads of 64: 4.3 us with 16 slots a workgroup, 6.0 with 64.
template <int ROWS>
__global__ __launch_bounds__(kReadThreads) void kv_read_kernel(ReadArgs A) {
    __shared__ int64_t at[ROWS];  // first code of the page and head, or -1
    __shared__ int off[ROWS];     // place in the page
    __shared__ float scale[ROWS];
    __shared__ int run[ROWS / 16];  // whether the 16 slots go on from one another
    const int h = blockIdx.y, hd = A.C.hd, tid = threadIdx.x;
    const bool is_v = blockIdx.z != 0;
    const int64_t i0 = (int64_t)blockIdx.x * ROWS;
    if (tid < ROWS) {
        const int64_t slot = i0 + tid < A.n ? A.slots[i0 + tid] : -1, page = slot >> A.C.shift;
        const bool ok = slot >= 0 && page < A.C.n_pages;
        const int64_t ph = page * A.C.n_kv + h;
        at[tid] = ok ? ph * ((int64_t)hd << A.C.shift) : -1;
        off[tid] = (int)(slot & ((1 << A.C.shift) - 1));
        scale[tid] = ok ? (is_v ? A.C.vs : A.C.ks)[ph] : 0.0f;
        const int64_t s0 = __shfl(slot, tid & 48);
        const int left = 16 - (int)(s0 & 15), k = tid & 15;
        const int64_t s1 = __shfl(slot, (tid & 48) + (left & 15));
        const bool on = ok && (k < left ? slot == s0 + k : (s1 & 15) == 0 && slot == s1 + k - left);
        const uint64_t all = __ballot(on);
        if (k == 0) run[tid >> 4] = (all >> (tid & 48) & 0xffffu) == 0xffffu;
    }
    __syncthreads();
    if (!is_v) {
        const int per_row = hd / 4;
#pragma unroll 4
        for (int u = tid; u < ROWS * per_row; u += kReadThreads) {
            const int i = u / per_row, d = u % per_row * 4;
            if (at[i] < 0) continue;
            const char4 c = *(const char4 *)(A.C.k + at[i] + off[i] * hd + d);
            float *to = A.k + (i0 + i) * A.ldk + (int64_t)h * hd + d;
            const float s = scale[i];
            if (A.wide) {
                *(float4 *)to = float4{c.x * s, c.y * s, c.z * s, c.w * s};
            } else {
                to[0] = c.x * s;
                to[1] = c.y * s;
                to[2] = c.z * s;
                to[3] = c.w * s;
            }
        }
        return;
    }
    union Codes {
        uint4 w;
        int8_t c[16];
    };
    for (int u = tid; u < ROWS / 16 * (hd / 2); u += kReadThreads) {
        const int first = u / (hd / 2) * 16, d = u % (hd / 2) * 2;
        float *to = A.v + (i0 + first) * A.ldv + (int64_t)h * hd + d;
        if (run[first >> 4]) {
            const int from = off[first] & 15, left = 16 - from, next = first + (left & 15);
            const int8_t *a = A.C.v + at[first] + (off[first] & ~15) + (d << A.C.shift);
            const int8_t *b = A.C.v + at[next] + (off[next] & ~15) + (d << A.C.shift);
            const int step = 1 << A.C.shift;
            Codes x, y;
            x.w = read_window(*(const uint4 *)a, *(const uint4 *)b, from);
            y.w = read_window(*(const uint4 *)(a + step), *(const uint4 *)(b + step), from);
            const float sa = scale[first], sb = scale[next];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float s = i < left ? sa : sb;
                if (A.wide) {
                    *(float2 *)(to + i * A.ldv) = float2{x.c[i] * s, y.c[i] * s};
                } else {
                    to[i * A.ldv] = x.c[i] * s;
                    to[i * A.ldv + 1] = y.c[i] * s;
                }
            }
            continue;
        }
        int8_t x[16], y[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            // (a slot that is none reads the first page, and writes nothing)
            const int64_t from = at[first + i] < 0 ? 0 : at[first + i] + off[first + i];
            const int8_t *a = A.C.v + from + (d << A.C.shift);
            x[i] = a[0];
            y[i] = a[1 << A.C.shift];
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            if (at[first + i] < 0) continue;
            to[i * A.ldv] = x[i] * scale[first + i];
            to[i * A.ldv + 1] = y[i] * scale[first + i];
        }
    }
}

}  // namespace sihip
