// Entry points of the paged 8-bit KV cache (declarations in include/sihip.h):
// argument checks, launch sizes, workspaces. Every array is the caller's and
// every length is a device number, so the host checks what it can see (sizes,
// alignment, pointers) and the kernels check what they read (requests, table
// entries, slots) before they use it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "attnp.h"
#include "context.h"
#include "kvcache.h"

using namespace sihip;

namespace {

// The calls run on the context's device and give the caller's back.
struct OnDevice {
    int before = -1, device;
    explicit OnDevice(int d) : device(d) {
        if (hipGetDevice(&before) != hipSuccess) before = -1;
        if (before != d) (void)hipSetDevice(d);
    }
    ~OnDevice() {
        if (before >= 0 && before != device) (void)hipSetDevice(before);
    }
};

bool aligned(const void *p, uintptr_t n) { return (uintptr_t)p % n == 0; }

// log2 of a supported block, or -1
int block_shift(int64_t block) {
    for (int s = 4; s <= 8; s++)
        if (block == (int64_t)1 << s) return s;
    return -1;
}

int launched(sihip_ctx *ctx, const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SIHIP_OK : set_err(ctx, SIHIP_EDEVICE, "%s launch: %s", what, hipGetErrorString(e));
}

int check_cache(sihip_ctx *ctx, const char *fn, const sihip_kv_cache *c, CacheArgs &C) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale)
        return set_err(ctx, SIHIP_EINVAL, "%s: NULL cache", fn);
    const int shift = block_shift(c->block);
    if (shift < 0)
        return set_err(ctx, SIHIP_EINVAL, "%s: block %lld is not 16, 32, 64, 128 or 256", fn, (long long)c->block);
    if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
        return set_err(ctx, SIHIP_EINVAL, "%s: head_dim %lld is not a multiple of 16 up to 256", fn,
                       (long long)c->head_dim);
    if (c->n_head_kv < 1 || c->n_head_kv > 4096)
        return set_err(ctx, SIHIP_EINVAL, "%s: n_head_kv %lld outside 1..4096", fn, (long long)c->n_head_kv);
    if (c->n_pages < 1 || c->n_pages > INT32_MAX)
        return set_err(ctx, SIHIP_EINVAL, "%s: n_pages %lld outside 1..2^31-1", fn, (long long)c->n_pages);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return set_err(ctx, SIHIP_EINVAL, "%s: k and v must be 16-byte aligned, scales 4-byte", fn);
    C = {c->k, c->v, c->k_scale, c->v_scale, c->n_pages, (int)c->n_head_kv, (int)c->head_dim, shift};
    return SIHIP_OK;
}

int check_batch(sihip_ctx *ctx, const char *fn, const sihip_kv_batch *b, int64_t block, BatchArgs &R) {
    if (!b || !b->q_start || !b->kv_len || !b->table) return set_err(ctx, SIHIP_EINVAL, "%s: NULL batch", fn);
    if (b->n_req < 1 || b->n_req > kMaxRequests)
        return set_err(ctx, SIHIP_EINVAL, "%s: n_req %lld outside 1..%lld", fn, (long long)b->n_req,
                       (long long)kMaxRequests);
    if (b->max_blocks < 1 || b->max_blocks > INT32_MAX / block)
        return set_err(ctx, SIHIP_EINVAL, "%s: max_blocks %lld of %lld tokens pass 2^31 positions", fn,
                       (long long)b->max_blocks, (long long)block);
    if (b->n_tok < 0 || b->n_tok > INT32_MAX || b->max_q < 0 || b->max_q > INT32_MAX || b->max_kv < 0 ||
        b->max_kv > INT32_MAX)
        return set_err(ctx, SIHIP_EINVAL, "%s: n_tok %lld, max_q %lld or max_kv %lld outside 0..2^31-1", fn,
                       (long long)b->n_tok, (long long)b->max_q, (long long)b->max_kv);
    R = {b->q_start, b->kv_len, b->table, b->n_tok, (int)b->max_blocks,
         (int)std::min(b->max_q, b->n_tok), (int)std::min(b->max_kv, b->max_blocks * block)};
    return SIHIP_OK;
}

}  // namespace

extern "C" int sihip_kv_plan_dev(sihip_ctx *ctx, const sihip_kv_plan *p, void *stream) {
    if (!ctx || !p) return set_err(ctx, SIHIP_EINVAL, "kv_plan_dev: NULL argument");
    if (!p->len || !p->add || !p->free_pages || !p->n_free || !p->table || !p->q_start || !p->kv_len ||
        !p->n_free_out || !p->status || (p->n_tok > 0 && (!p->slot || !p->pos)))
        return set_err(ctx, SIHIP_EINVAL, "kv_plan_dev: NULL array");
    if (p->n_req < 1 || p->n_req > kMaxRequests)
        return set_err(ctx, SIHIP_EINVAL, "kv_plan_dev: n_req %lld outside 1..%lld", (long long)p->n_req,
                       (long long)kMaxRequests);
    const int shift = block_shift(p->block);
    if (shift < 0)
        return set_err(ctx, SIHIP_EINVAL, "kv_plan_dev: block %lld is not 16, 32, 64, 128 or 256",
                       (long long)p->block);
    if (p->n_tok < 0 || p->n_tok > INT32_MAX || p->n_pages < 1 || p->n_pages > INT32_MAX)
        return set_err(ctx, SIHIP_EINVAL, "kv_plan_dev: n_tok %lld or n_pages %lld out of range",
                       (long long)p->n_tok, (long long)p->n_pages);
    if (p->max_blocks < 1 || p->max_blocks > INT32_MAX / p->block)
        return set_err(ctx, SIHIP_EINVAL, "kv_plan_dev: max_blocks %lld of %lld tokens pass 2^31 positions",
                       (long long)p->max_blocks, (long long)p->block);
    if (p->kv_len == p->len || p->kv_len == p->add || p->n_free_out == p->n_free)
        return set_err(ctx, SIHIP_EINVAL, "kv_plan_dev: kv_len and n_free_out must not be inputs of the call");
    const OnDevice on(ctx->device);
    const PlanArgs A = {p->len, p->add, p->n_free, p->free_pages, p->table, p->q_start, p->kv_len, p->pos,
                        p->n_free_out, p->status, p->slot, p->n_tok, (int)p->n_req, (int)p->n_pages,
                        (int)p->max_blocks, shift};
    // few requests need few waves, which start and meet sooner
    const bool few = p->n_req <= 256;
    const int64_t threads = few ? 256 : 1024;
    const int64_t wgs = std::min<int64_t>(std::max<int64_t>(1, (p->n_tok + threads - 1) / threads), ctx->n_cu);
    hipLaunchKernelGGL(few ? kv_plan_kernel<256> : kv_plan_kernel<1024>, dim3((unsigned)wgs), dim3((unsigned)threads),
                       (size_t)p->n_req * 12, (hipStream_t)stream, A);
    return launched(ctx, "kv_plan");
}

extern "C" int sihip_kv_append_dev(sihip_ctx *ctx, const sihip_kv_cache *cache, const sihip_kv_batch *batch,
                                   const float *k, int64_t ldk, const float *v, int64_t ldv, void *stream) {
    if (!ctx) return set_err(ctx, SIHIP_EINVAL, "kv_append_dev: NULL argument");
    AppendArgs A;
    int rc = check_cache(ctx, "kv_append_dev", cache, A.C);
    if (!rc) rc = check_batch(ctx, "kv_append_dev", batch, cache->block, A.R);
    if (rc) return rc;
    const int64_t width = (int64_t)A.C.n_kv * A.C.hd;
    if (ldk < width || ldv < width)
        return set_err(ctx, SIHIP_EINVAL, "kv_append_dev: rows of %lld values at ldk %lld, ldv %lld",
                       (long long)width, (long long)ldk, (long long)ldv);
    if (A.R.max_q == 0) return SIHIP_OK;
    if (!k || !v || !aligned(k, 4) || !aligned(v, 4))
        return set_err(ctx, SIHIP_EINVAL, "kv_append_dev: k and v must be f32 arrays");
    A.k = k;
    A.v = v;
    A.ldk = ldk;
    A.ldv = ldv;
    A.k_wide = aligned(k, 16) && ldk % 4 == 0;
    // blocks of a request that max_q tokens can touch
    const int64_t blocks = std::min<int64_t>(((int64_t)A.R.max_q + cache->block - 2) / cache->block + 1, A.R.max_blocks);
    const int64_t gx = blocks * A.C.n_kv;
    if (gx * 1024 > UINT32_MAX)
        return set_err(ctx, SIHIP_EINVAL, "kv_append_dev: max_q %d of %d heads has no grid", A.R.max_q, A.C.n_kv);
    const OnDevice on(ctx->device);
    const dim3 grid((unsigned)gx, (unsigned)batch->n_req, 2);
    const hipStream_t st = (hipStream_t)stream;
    const int64_t units = cache->block * A.C.hd / 16;
    if (units <= 128) hipLaunchKernelGGL((kv_append_kernel<1, 128>), grid, dim3(128), 0, st, A);
    else if (units <= 256) hipLaunchKernelGGL((kv_append_kernel<1, 256>), grid, dim3(256), 0, st, A);
    else if (units <= 512) hipLaunchKernelGGL((kv_append_kernel<1, 512>), grid, dim3(512), 0, st, A);
    else if (units <= 1024) hipLaunchKernelGGL((kv_append_kernel<1, 1024>), grid, dim3(1024), 0, st, A);
    else if (units <= 2048) hipLaunchKernelGGL((kv_append_kernel<2, 1024>), grid, dim3(1024), 0, st, A);
    else hipLaunchKernelGGL((kv_append_kernel<4, 1024>), grid, dim3(1024), 0, st, A);
    return launched(ctx, "kv_append");
}

extern "C" int sihip_kv_read_dev(sihip_ctx *ctx, const sihip_kv_cache *cache, const int64_t *slots, int64_t n,
                                 float *k, int64_t ldk, float *v, int64_t ldv, void *stream) {
    if (!ctx) return set_err(ctx, SIHIP_EINVAL, "kv_read_dev: NULL argument");
    ReadArgs A;
    const int rc = check_cache(ctx, "kv_read_dev", cache, A.C);
    if (rc) return rc;
    const int64_t width = (int64_t)A.C.n_kv * A.C.hd;
    if (n < 0 || n > INT32_MAX || ldk < width || ldv < width)
        return set_err(ctx, SIHIP_EINVAL, "kv_read_dev: %lld rows of %lld values at ldk %lld, ldv %lld", (long long)n,
                       (long long)width, (long long)ldk, (long long)ldv);
    if (n == 0) return SIHIP_OK;
    if (!slots || !k || !v || !aligned(slots, 8) || !aligned(k, 4) || !aligned(v, 4))
        return set_err(ctx, SIHIP_EINVAL, "kv_read_dev: slots must be an int64 array, k and v f32 arrays");
    A.slots = slots;
    A.k = k;
    A.v = v;
    A.n = n;
    A.ldk = ldk;
    A.ldv = ldv;
    A.wide = aligned(k, 16) && ldk % 4 == 0 && aligned(v, 16) && ldv % 4 == 0;
    // 64 slots a workgroup use the lines of a page that they load; while those
    // are too few workgroups to fill the device, 16
    const bool few = (n + 63) / 64 * A.C.n_kv * 2 < 4 * ctx->n_cu;
    const int64_t rows = few ? 16 : 64, gx = (n + rows - 1) / rows;
    if (gx * kReadThreads > UINT32_MAX)
        return set_err(ctx, SIHIP_EINVAL, "kv_read_dev: %lld rows have no grid", (long long)n);
    const OnDevice on(ctx->device);
    hipLaunchKernelGGL(few ? kv_read_kernel<16> : kv_read_kernel<64>, dim3((unsigned)gx, (unsigned)A.C.n_kv, 2),
                       dim3(kReadThreads), 0, (hipStream_t)stream, A);
    return launched(ctx, "kv_read");
}

// ---- attention ------------------------------------------------------------------

namespace {

// counters at the front of a caller's workspace, whatever the call's size
constexpr size_t kCounterBytes = (size_t)kGemmCounters * 4;

// One launch: the kernel for few rows of a request (16-row blocks) or the one
// for many (blocks of 128 or 256).
struct AttnPLaunch {
    AttnPArgs A;
    int waves = 0;      // of 32 rows in a large row block, 0: 16-row blocks
    int row_waves = 0;  // waves that share a 16-row block's chunks
    int64_t blocks = 0, gx = 0, pieces = 0;  // row blocks, the grid, parts of split blocks
    size_t part_bytes = 0;
};

struct AttnPPlan {
    AttnPLaunch l[2];
    int n = 0;
    size_t part_bytes() const { return (n > 0 ? l[0].part_bytes : 0) + (n > 1 ? l[1].part_bytes : 0); }
};

// Rows of a request up to which it counts as one with few, where a batch has both.
constexpr int kApFewRows = 64;

// Waves of a large row block, 0: 16-row blocks throughout. The work is 16-row
// blocks times 64-key chunks (as far as the host knows the lengths: bounds)
// times the head's width. us, 16-row blocks against the large ones:
//   32 heads of 128: 512 rows 24 / 50, 1024 51 / 72, 1500 86 / 99, 1800 114 / 116,
//     2048 132 / 120; 190 behind 8000 keys 96 / 107, 256 behind 8000 105 / 85, 64
//     behind 30000 118 / 77; window of 512 140 / 119
//     rows of few keys, however many: 200 prompts of up to 256 311 / 362, 50 of up
//     to 512 184 / 205, 8 of up to 1024 128 / 125
//   14 heads of 64 on 2: 1200 27 / 33, 4096 133 / 124; 32 on 8: 4096 239 / 171
//   wider than 128 the large blocks' sums would leave one wave a SIMD: 16 heads of
//     256, 4096 rows 467, 627 in a build that had them
int attn_waves(const sihip_ctx *ctx, const AttnPArgs &A, int64_t rows, int64_t all_rows) {
    if (A.C.hd > 128) return 0;
    const int waves = ap_tile_waves(A.C.hd);
    if (ctx->opt.attnp_large >= 0) return ctx->opt.attnp_large ? waves : 0;
    if (rows <= 32) return 0;
    int64_t keys = A.R.max_kv - A.R.max_q / 2;  // of a row, on average, without a window
    if (A.window) keys = std::min<int64_t>(keys, (int64_t)A.window + 64);
    if (keys < 384) return 0;
    const double work = (double)(all_rows / 16 * A.C.n_kv) * ((double)keys / 64) * A.C.hd;
    return work < 45e3 * 128 ? 0 : waves;
}

// Blocks, pieces and grid of a launch over requests of up to `rows` rows,
// `all_rows` together.
int plan_launch(sihip_ctx *ctx, AttnPLaunch &L, int64_t rows, int64_t all_rows) {
    AttnPArgs &A = L.A;
    const int block_rows = L.waves ? 32 * L.waves : kApRows;
    A.n_tiles = (int)((rows + block_rows - 1) / block_rows);
    A.ranks = (int)std::min<int64_t>((int64_t)A.R.max_kv * A.G / block_rows, 1 << 30);
    // row blocks of all requests: as many as the longest has each, and, listed,
    // no more than the step's rows fill
    L.blocks = (int64_t)A.n_req * A.n_tiles;
    if (A.placed) L.blocks = std::min(L.blocks, all_rows / block_rows + A.n_req);
    const int64_t items = L.blocks * A.C.n_kv;
    A.chunk = L.waves || A.C.hd <= 128 ? 6 : 5;
    const int64_t chunks = std::max<int64_t>(1, ((int64_t)A.R.max_kv + (1 << A.chunk) - 1) >> A.chunk);
    const int64_t forced = ctx->opt.attnp_splits;
    if (L.waves || !A.placed) {
        // splits of a row block's keys: until every CU has its workgroups, none
        // shorter than four chunks
        L.row_waves = 4;
        const int64_t per_cu = L.waves ? 8 / L.waves : 4;
        int64_t n = (per_cu * ctx->n_cu + items - 1) / std::max<int64_t>(items, 1);
        if (forced > 0) n = forced;
        n = std::max<int64_t>(1, std::min<int64_t>(n, 64));
        A.per_split = (int)std::max<int64_t>((chunks + n - 1) / n, forced > 0 ? 1 : 4);
        A.n_split = (int)((chunks + A.per_split - 1) / A.per_split);
        A.whole = 0;
        L.pieces = items * A.n_split;
        L.gx = L.waves ? (A.placed ? L.blocks : A.n_tiles) * A.C.n_kv : (int64_t)A.n_tiles * A.n_split;
    } else {
        // Four waves share a piece, or, where there are row blocks enough, each
        // has its own. Workgroups that the pieces are made for, of single tokens
        // by the number of row blocks: the host knows no more. Few blocks: one a
        // CU; more: more, as the pieces of blocks of different lengths end at
        // different times. us with 1 / 1.5 / 3 a CU, heads of 128, blocks of up to
        // so many keys: 8 of 131072 46 / 56 / 65; 32 of 30000 41 / 35 / 40; 64 of
        // 16000 36 / 31 / 36; 128 of 16000 64 / 51 / 59; 248 of 8191 45 / 49 / 44;
        // 256 of 8191 49 / 41 / 45; 400 of 8191 67 / 73 / 63; 512 of 8191 89 / 88 /
        // 81. Blocks that are all of one length would do better with one: 128 of
        // 8000 46 / 54 / 58, 256 of 4095 43 / 48 / 58, 512 of 4095 100 / 100 / 110.
        // The row blocks of prompts fill the CUs by themselves, and are as long as
        // each other (128 rows behind 4000 keys 37 us with one, 52 with three).
        const int64_t w = ctx->opt.attnp_row_waves;
        L.row_waves = w == 1 || w == 4 ? (int)w : items >= 4 * ctx->n_cu ? 1 : 4;
        A.slots = (A.R.max_q > 1 ? (L.row_waves == 1 ? 8 : 2) : L.row_waves == 1 ? 16 : items < 64 ? 2 : items < 256 ? 3 : 6) *
                  ctx->n_cu / 2;
        A.per_split = L.row_waves == 1 ? 6 : L.row_waves;
        A.whole = L.row_waves == 1 ? 8 : 2 * L.row_waves;
        if (forced > 0) {
            A.slots = (int)std::min<int64_t>(forced * std::max<int64_t>(items, 1), 1 << 20);
            A.per_split = 1;
            A.whole = 0;
        }
        A.n_split = chunks > std::max(A.whole, A.per_split) ? INT32_MAX : 1;
        L.pieces = items + A.slots;
        L.gx = A.n_split > 1 ? L.pieces : items;
    }
    // pieces of 16-row blocks join by counters, one for each at most
    if (!L.waves && L.pieces > kGemmCounters) {
        A.n_split = 1;
        A.per_split = INT32_MAX;
        L.gx = A.placed ? items : A.n_tiles;
    }
    L.part_bytes = A.n_split > 1 ? (size_t)L.pieces * block_rows * (A.C.hd / 4 + 1) * 16 : 0;
    if (L.gx * 512 > UINT32_MAX)
        return set_err(ctx, SIHIP_EINVAL, "attn_paged_dev: max_q %d of %d heads has no grid", A.R.max_q, A.G * A.C.n_kv);
    return SIHIP_OK;
}

int plan_attn(sihip_ctx *ctx, const sihip_kv_cache *cache, const sihip_kv_batch *batch, const sihip_attn_paged *a,
              AttnPPlan &P) {
    const char *fn = "attn_paged_dev";
    if (!ctx || !a) return set_err(ctx, SIHIP_EINVAL, "%s: NULL argument", fn);
    AttnPArgs A = {};
    int rc = check_cache(ctx, fn, cache, A.C);
    if (!rc) rc = check_batch(ctx, fn, batch, cache->block, A.R);
    if (rc) return rc;
    if (a->n_head < 1 || a->n_head > 4096 || a->n_head % A.C.n_kv)
        return set_err(ctx, SIHIP_EINVAL, "%s: n_head %lld must be a multiple of n_head_kv %d (<= 4096)", fn,
                       (long long)a->n_head, A.C.n_kv);
    const int64_t width = a->n_head * A.C.hd;
    if (a->ldq < width || a->ldo < width)
        return set_err(ctx, SIHIP_EINVAL, "%s: rows of %lld values at ldq %lld, ldo %lld", fn, (long long)width,
                       (long long)a->ldq, (long long)a->ldo);
    if (!std::isfinite(a->kq_scale) || !std::isfinite(a->softcap) || a->softcap < 0)
        return set_err(ctx, SIHIP_EINVAL, "%s: kq_scale %g or softcap %g", fn, (double)a->kq_scale,
                       (double)a->softcap);
    if (a->window < 0) return set_err(ctx, SIHIP_EINVAL, "%s: window %lld", fn, (long long)a->window);
    if (A.R.max_q == 0) return SIHIP_OK;
    if (!a->q || !a->out || !aligned(a->q, 4) || !aligned(a->out, 4))
        return set_err(ctx, SIHIP_EINVAL, "%s: q and out must be f32 arrays", fn);
    A.G = (int)(a->n_head / A.C.n_kv);
    const int64_t rows = (int64_t)A.R.max_q * A.G, all_rows = A.R.n_tok * A.G;
    if (rows > INT32_MAX)
        return set_err(ctx, SIHIP_EINVAL, "%s: max_q %d times %d heads a KV head pass 2^31 rows", fn, A.R.max_q, A.G);
    A.q = a->q;
    A.out = a->out;
    A.ldq = a->ldq;
    A.ldo = a->ldo;
    A.q_vec = aligned(a->q, 16) && a->ldq % 4 == 0;
    A.out_vec = aligned(a->out, 16) && a->ldo % 4 == 0;
    A.slopes = a->slopes;
    A.prefix = a->prefix;
    A.n_req = (int)batch->n_req;
    A.window = (int)std::min<int64_t>(a->window, INT32_MAX);
    const double scale = std::fabs((double)a->kq_scale), log2e = 1.4426950408889634;
    A.sign = a->kq_scale < 0 ? -1.0f : 1.0f;
    A.scale2 = (float)(scale * log2e);
    A.cap = (float)std::min((double)a->softcap * log2e, (double)FLT_MAX);
    A.cap_in = a->softcap > 0 ? (float)std::min(2.0 * scale / a->softcap * log2e, (double)FLT_MAX) : 0.0f;
    A.placed = A.n_req <= 64 * kPlaceRegs;
    A.least = 0;
    A.most = INT32_MAX;
    P.l[0].A = A;
    P.l[0].waves = attn_waves(ctx, A, rows, all_rows);
    P.n = 1;
    // Lengths that differ: a request of few rows would fill little of a large
    // block, and go through all its keys in it alone
    if (P.l[0].waves && A.placed && A.n_req > 1 && A.R.n_tok < (int64_t)A.n_req * A.R.max_q && rows > kApFewRows) {
        P.l[0].A.least = kApFewRows + 1;
        P.l[1].A = A;
        P.l[1].A.most = kApFewRows;
        P.n = 2;
        rc = plan_launch(ctx, P.l[1], kApFewRows, std::min<int64_t>(all_rows, (int64_t)A.n_req * kApFewRows));
        if (rc) return rc;
    }
    return plan_launch(ctx, P.l[0], rows, all_rows);
}

int launch_attn(sihip_ctx *ctx, const AttnPLaunch &L, hipStream_t st) {
    const AttnPArgs &A = L.A;
    const int hd = A.C.hd, z = A.placed ? 1 : A.n_req;
    if (L.waves) {
        const dim3 grid((unsigned)L.gx, (unsigned)A.n_split, (unsigned)z), t(L.waves * 64);
        if (hd <= 64) hipLaunchKernelGGL(attnp_tiles_kernel<4>, grid, t, 0, st, A);
        else if (hd <= 96) hipLaunchKernelGGL(attnp_tiles_kernel<6>, grid, t, 0, st, A);
        else hipLaunchKernelGGL(attnp_tiles_kernel<8>, grid, t, 0, st, A);
        if (A.n_split > 1) {
            const int per_wg = kApJoinThreads / (32 * L.waves);  // four-dim columns
            const dim3 jg((unsigned)L.gx, (unsigned)((hd / 4 + per_wg - 1) / per_wg), (unsigned)z);
            if (L.waves == 4) hipLaunchKernelGGL(attnp_join_kernel<128>, jg, dim3(kApJoinThreads), 0, st, A);
            else hipLaunchKernelGGL(attnp_join_kernel<256>, jg, dim3(kApJoinThreads), 0, st, A);
        }
    } else {
        const dim3 grid((unsigned)L.gx, A.placed ? 1u : (unsigned)A.C.n_kv, (unsigned)z), t(L.row_waves * 64);
#define SIHIP_APR(NK, TT)                                                                                  \
    if (L.row_waves == 1) hipLaunchKernelGGL((attnp_rows_kernel<NK, TT, 1>), grid, t, 0, st, A);           \
    else hipLaunchKernelGGL((attnp_rows_kernel<NK, TT, 4>), grid, t, 0, st, A);
        if (hd <= 64) { SIHIP_APR(1, 4) }
        else if (hd <= 128) { SIHIP_APR(2, 4) }
        else if (hd <= 192) { SIHIP_APR(3, 2) }
        else { SIHIP_APR(4, 2) }
#undef SIHIP_APR
    }
    return launched(ctx, "attn_paged");
}

}  // namespace

extern "C" int sihip_attn_paged_workspace(sihip_ctx *ctx, const sihip_kv_cache *cache, const sihip_kv_batch *batch,
                                          const sihip_attn_paged *args, uint64_t *bytes) {
    if (!bytes) return set_err(ctx, SIHIP_EINVAL, "attn_paged_workspace: NULL argument");
    AttnPPlan P;
    const int rc = plan_attn(ctx, cache, batch, args, P);
    if (rc) return rc;
    *bytes = P.part_bytes() ? kCounterBytes + P.part_bytes() : 0;
    return SIHIP_OK;
}

extern "C" int sihip_attn_paged_dev(sihip_ctx *ctx, const sihip_kv_cache *cache, const sihip_kv_batch *batch,
                                    const sihip_attn_paged *args, void *stream) {
    AttnPPlan P;
    int rc = plan_attn(ctx, cache, batch, args, P);
    if (rc || P.n == 0) return rc;
    const OnDevice on(ctx->device);
    const hipStream_t st = (hipStream_t)stream;
    const size_t bytes = P.part_bytes();
    const bool shared = bytes && !args->workspace;
    uint32_t *cnt = nullptr;
    uint8_t *part = nullptr;
    if (shared) {
        try {
            rc = ensure(ctx, &ctx->d_attn, &ctx->d_attn_cap, bytes, st);
        } catch (...) {
            rc = set_err(ctx, SIHIP_ENOMEM, "attn_paged_dev: out of host memory");
        }
        if (!rc) rc = order_before(ctx, ctx->order, st);
        if (rc) return rc;
        cnt = ctx->d_gcnt;
        part = (uint8_t *)ctx->d_attn;
    } else if (bytes) {
        if (args->workspace_bytes < kCounterBytes + bytes || !aligned(args->workspace, 16))
            return set_err(ctx, SIHIP_EINVAL, "attn_paged_dev: a workspace of %zu bytes, 16-byte aligned, is needed",
                           kCounterBytes + bytes);
        cnt = (uint32_t *)args->workspace;
        part = (uint8_t *)args->workspace + kCounterBytes;
    }
    for (int i = 0; i < P.n; i++) {
        P.l[i].A.cnt = cnt;
        P.l[i].A.part = (float *)part;
        part += P.l[i].part_bytes;
        rc = launch_attn(ctx, P.l[i], st);
        if (rc) return rc;
    }
    return shared ? order_after(ctx, ctx->order, st) : SIHIP_OK;
}
