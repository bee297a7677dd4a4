// What the entry points of the paged caches share on the host: argument
// checks, and the launches and workspaces of attention. Every array is the caller's and
// every length is a device number, so the host checks what it can see (sizes,
// alignment, pointers) and the kernels check what they read (requests, table
// entries, slots) before they use it.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "attnp.h"
#include "kvcache.h"
#include "launch.h"
#include "rope.h"

// one copy for the library's translation units, not exported (context.h)
#pragma GCC visibility push(hidden)

namespace sihip {

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

// The second launch of large row blocks whose keys were split (kvcache.hip).
void launch_join(const AttnPLaunch &L, hipStream_t st);

namespace {

// log2 of a supported block, or -1
int block_shift(int64_t block) {
    for (int s = 4; s <= 8; s++)
        if (block == (int64_t)1 << s) return s;
    return -1;
}

// Sizes that both caches have, head_dim in steps of `dims`.
int check_sizes(sihip_ctx *ctx, const char *fn, int64_t block, int64_t head_dim, int dims, int64_t n_head_kv, int64_t n_pages) {
    if (block_shift(block) < 0)
        return set_err(ctx, SIHIP_EINVAL, "%s: block %lld is not 16, 32, 64, 128 or 256", fn, (long long)block);
    if (head_dim < dims || head_dim > 256 || head_dim % dims)
        return set_err(ctx, SIHIP_EINVAL, "%s: head_dim %lld is not a multiple of %d up to 256", fn, (long long)head_dim, dims);
    if (n_head_kv < 1 || n_head_kv > 4096)
        return set_err(ctx, SIHIP_EINVAL, "%s: n_head_kv %lld outside 1..4096", fn, (long long)n_head_kv);
    if (n_pages < 1 || n_pages > INT32_MAX)
        return set_err(ctx, SIHIP_EINVAL, "%s: n_pages %lld outside 1..2^31-1", fn, (long long)n_pages);
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

// Rotated queries of more than twice what the L2s hold are written past them. By the step's room, which the host knows: a step of
// fewer rows loses nothing by it. us of an append and the attention that reads its queries next, through / past the L2s, 32 heads of
// 128 on 8, over 4 and 8 bits: a row 16.3 / 16.5 and 15.7 / 15.9; 64 single tokens behind 600 keys 26.5 / 26.0 and 25.9 /
// 25.6, behind 8191 71.9 / 71.8 and 99.1 / 98.4; 1008 rows 75.1 / 74.5 and 63.9 / 63.3.
constexpr int64_t kPastBytes = 64 << 20;

// The new rows of a step for a cache of n_kv heads of hd dims. Without tokens
// (R.max_q 0) arrays may be missing.
int check_rows(sihip_ctx *ctx, const char *fn, const sihip_kv_rows *a, const BatchArgs &R, int n_kv, int hd, RopeArgs &P,
               RopeQueries &Q) {
    if (!a) return set_err(ctx, SIHIP_EINVAL, "%s: NULL argument", fn);
    const int64_t width = (int64_t)n_kv * hd;
    if (a->ldk < width || a->ldv < width)
        return set_err(ctx, SIHIP_EINVAL, "%s: rows of %lld values at ldk %lld, ldv %lld", fn, (long long)width,
                       (long long)a->ldk, (long long)a->ldv);
    P = {};
    Q = {};
    if (a->rope) {
        if (a->rope_dim < 2 || a->rope_dim % 2 || a->rope_dim > hd)
            return set_err(ctx, SIHIP_EINVAL, "%s: rope_dim %lld is not even and in 2..%d", fn, (long long)a->rope_dim, hd);
        if (a->rope_len < R.max_kv)
            return set_err(ctx, SIHIP_EINVAL, "%s: rope_len %lld is below the %d positions of the batch", fn,
                           (long long)a->rope_len, R.max_kv);
        if (!aligned(a->rope, 4)) return set_err(ctx, SIHIP_EINVAL, "%s: rope must be an f32 array", fn);
        P = {a->rope, (int)a->rope_dim / 2, a->rope_neighbours != 0, aligned(a->rope, 16) && a->rope_dim % 8 == 0};
    }
    if (a->q) {
        if (!a->rope) return set_err(ctx, SIHIP_EINVAL, "%s: queries without a rotation", fn);
        if (a->n_head < 1 || a->n_head > 4096 || a->n_head % n_kv)
            return set_err(ctx, SIHIP_EINVAL, "%s: n_head %lld must be a multiple of n_head_kv %d (<= 4096)", fn,
                           (long long)a->n_head, n_kv);
        const int64_t wide = a->n_head * hd;
        if (a->ldq < wide || a->ldq_out < wide)
            return set_err(ctx, SIHIP_EINVAL, "%s: rows of %lld values at ldq %lld, ldq_out %lld", fn, (long long)wide,
                           (long long)a->ldq, (long long)a->ldq_out);
        if (!a->q_out || !aligned(a->q, 4) || !aligned(a->q_out, 4))
            return set_err(ctx, SIHIP_EINVAL, "%s: q and q_out must be f32 arrays", fn);
        if (a->q == a->q_out && a->ldq != a->ldq_out)
            return set_err(ctx, SIHIP_EINVAL, "%s: in place, ldq %lld and ldq_out %lld must be equal", fn, (long long)a->ldq,
                           (long long)a->ldq_out);
        Q = {a->q, a->q_out, a->ldq, a->ldq_out, (int)(a->n_head / n_kv),
             aligned(a->q, 16) && aligned(a->q_out, 16) && a->ldq % 4 == 0 && a->ldq_out % 4 == 0,
             R.n_tok * wide * 4 > kPastBytes};
    }
    if (R.max_q > 0 && (!a->k || !a->v || !aligned(a->k, 4) || !aligned(a->v, 4)))
        return set_err(ctx, SIHIP_EINVAL, "%s: k and v must be f32 arrays", fn);
    return SIHIP_OK;
}

// Workgroups of an append along x: the blocks of a request that max_q tokens can
// touch, each KV head. 0: nothing to do.
int append_grid(sihip_ctx *ctx, const char *fn, const BatchArgs &R, int n_kv, int64_t block, int64_t &gx) {
    const int64_t blocks = std::min<int64_t>(((int64_t)R.max_q + block - 2) / block + 1, R.max_blocks);
    gx = R.max_q ? blocks * n_kv : 0;
    if (gx * 1024 > UINT32_MAX) return set_err(ctx, SIHIP_EINVAL, "%s: max_q %d of %d heads has no grid", fn, R.max_q, n_kv);
    return SIHIP_OK;
}

// ---- attention ------------------------------------------------------------------

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
//     256, 4096 rows 467, 627 in a build that had them (over 4 bits 770, and none was built)
// and over 4 bits (one threshold for both: of these it has the slower side for 2048 rows with the window, and for 1300 of
// heads of 96):
//   32 heads of 128: 1500 rows 102 / 111, 1800 136 / 132, 2048 158 / 144, 3000 298 / 202; 190 behind 8000 keys 120 /
//     125, 256 behind 8000 123 / 96, 64 behind 30000 133 / 87; window of 512, 2048 rows 82 / 67; 200 prompts of up to
//     256 312 / 385, 50 of up to 512 192 / 217, 8 of up to 1024 106 / 91; heads of 96: 1300 85 / 80, 2048 156 / 128
//   heads of 64: 32 on 8: 2048 105 / 107, 3000 199 / 159
int attn_waves(const sihip_ctx *ctx, const AttnPArgs &A, int waves, int64_t rows, int64_t all_rows) {
    if (A.C.hd > 128) return 0;
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
int plan_launch(sihip_ctx *ctx, const char *fn, AttnPLaunch &L, int64_t rows, int64_t all_rows) {
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
        return set_err(ctx, SIHIP_EINVAL, "%s: max_q %d of %d heads has no grid", fn, A.R.max_q, A.G * A.C.n_kv);
    return SIHIP_OK;
}

// C: the cache, which the caller has checked; waves: of a large row block.
int plan_attn(sihip_ctx *ctx, const char *fn, const CacheArgs &C, int waves, const sihip_kv_batch *batch, const sihip_attn_paged *a,
              AttnPPlan &P) {
    if (!a) return set_err(ctx, SIHIP_EINVAL, "%s: NULL argument", fn);
    AttnPArgs A = {};
    A.C = C;
    int rc = check_batch(ctx, fn, batch, (int64_t)1 << C.shift, A.R);
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
    P.l[0].waves = attn_waves(ctx, A, waves, rows, all_rows);
    P.n = 1;
    // Lengths that differ: a request of few rows would fill little of a large
    // block, and go through all its keys in it alone
    if (P.l[0].waves && A.placed && A.n_req > 1 && A.R.n_tok < (int64_t)A.n_req * A.R.max_q && rows > kApFewRows) {
        P.l[0].A.least = kApFewRows + 1;
        P.l[1].A = A;
        P.l[1].A.most = kApFewRows;
        P.n = 2;
        rc = plan_launch(ctx, fn, P.l[1], kApFewRows, std::min<int64_t>(all_rows, (int64_t)A.n_req * kApFewRows));
        if (rc) return rc;
    }
    return plan_launch(ctx, fn, P.l[0], rows, all_rows);
}

// The launches of a call, launch(L) each.
template <class Launch>
int run_attn(sihip_ctx *ctx, const char *fn, AttnPPlan &P, const sihip_attn_paged *args, hipStream_t st, Launch launch) {
    return with_workspace(ctx, fn, P.part_bytes(), args->workspace, args->workspace_bytes, st, [&](uint32_t *cnt, uint8_t *part) {
        int rc = SIHIP_OK;
        for (int i = 0; i < P.n && !rc; i++) {
            P.l[i].A.cnt = cnt;
            P.l[i].A.part = (float *)part;
            part += P.l[i].part_bytes;
            rc = launch(P.l[i]);
        }
        return rc;
    });
}

}  // namespace
}  // namespace sihip

#pragma GCC visibility pop
