// Entry points of the paged 8-bit KV cache (declarations in include/sihip.h).
#include "kvhost.h"
#include "kvrope.h"

using namespace sihip;

namespace {

int check_cache(sihip_ctx *ctx, const char *fn, const sihip_kv_cache *c, CacheArgs &C) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale)
        return set_err(ctx, SIHIP_EINVAL, "%s: NULL cache", fn);
    const int rc = check_sizes(ctx, fn, c->block, c->head_dim, 16, c->n_head_kv, c->n_pages);
    if (rc) return rc;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return set_err(ctx, SIHIP_EINVAL, "%s: k and v must be 16-byte aligned, scales 4-byte", fn);
    C = {c->k, c->v, c->k_scale, c->v_scale, c->n_pages, (int)c->n_head_kv, (int)c->head_dim, block_shift(c->block)};
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
    int64_t gx;
    rc = append_grid(ctx, "kv_append_dev", A.R, A.C.n_kv, cache->block, gx);
    if (rc) return rc;
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

extern "C" int sihip_kv_append_rope_dev(sihip_ctx *ctx, const sihip_kv_cache *cache, const sihip_kv_batch *batch,
                                        const sihip_kv_rows *rows, void *stream) {
    const char *fn = "kv_append_rope_dev";
    if (!ctx) return set_err(ctx, SIHIP_EINVAL, "%s: NULL argument", fn);
    AppendArgs A;
    KeyRope X;
    int64_t gx = 0;
    int rc = check_cache(ctx, fn, cache, A.C);
    if (!rc) rc = check_batch(ctx, fn, batch, cache->block, A.R);
    if (!rc) rc = check_rows(ctx, fn, rows, A.R, A.C.n_kv, A.C.hd, X.P, X.Q);
    if (!rc && !rows->rope) rc = set_err(ctx, SIHIP_EINVAL, "%s: NULL rope", fn);
    if (!rc) rc = append_grid(ctx, fn, A.R, A.C.n_kv, cache->block, gx);
    if (rc || !gx) return rc;
    A.k = rows->k;
    A.v = rows->v;
    A.ldk = rows->ldk;
    A.ldv = rows->ldv;
    A.k_wide = aligned(A.k, 16) && A.ldk % 4 == 0;
    const OnDevice on(ctx->device);
    const dim3 grid((unsigned)gx, (unsigned)batch->n_req, X.Q.q ? 3 : 2);
    const hipStream_t st = (hipStream_t)stream;
    const int64_t units = cache->block * A.C.hd / 16;
    if (units <= 128) hipLaunchKernelGGL((kv_append_kernel<1, 128, KeyRope>), grid, dim3(128), 0, st, A, X);
    else if (units <= 256) hipLaunchKernelGGL((kv_append_kernel<1, 256, KeyRope>), grid, dim3(256), 0, st, A, X);
    else if (units <= 512) hipLaunchKernelGGL((kv_append_kernel<1, 512, KeyRope>), grid, dim3(512), 0, st, A, X);
    else if (units <= 1024) hipLaunchKernelGGL((kv_append_kernel<1, 1024, KeyRope>), grid, dim3(1024), 0, st, A, X);
    else if (units <= 2048) hipLaunchKernelGGL((kv_append_kernel<2, 1024, KeyRope>), grid, dim3(1024), 0, st, A, X);
    else hipLaunchKernelGGL((kv_append_kernel<4, 1024, KeyRope>), grid, dim3(1024), 0, st, A, X);
    return launched(ctx, "kv_append_rope");
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

void sihip::launch_join(const AttnPLaunch &L, hipStream_t st) {
    const AttnPArgs &A = L.A;
    const int per_wg = kApJoinThreads / (32 * L.waves);  // four-dim columns
    const dim3 grid((unsigned)L.gx, (unsigned)((A.C.hd / 4 + per_wg - 1) / per_wg), A.placed ? 1u : (unsigned)A.n_req);
    if (L.waves == 4) hipLaunchKernelGGL(attnp_join_kernel<128>, grid, dim3(kApJoinThreads), 0, st, A);
    else hipLaunchKernelGGL(attnp_join_kernel<256>, grid, dim3(kApJoinThreads), 0, st, A);
}

namespace {

int launch_attn(sihip_ctx *ctx, const AttnPLaunch &L, hipStream_t st) {
    const AttnPArgs &A = L.A;
    const int hd = A.C.hd, z = A.placed ? 1 : A.n_req;
    if (L.waves) {
        const dim3 grid((unsigned)L.gx, (unsigned)A.n_split, (unsigned)z), t(L.waves * 64);
        if (hd <= 64) hipLaunchKernelGGL(attnp_tiles_kernel<4>, grid, t, 0, st, A);
        else if (hd <= 96) hipLaunchKernelGGL(attnp_tiles_kernel<6>, grid, t, 0, st, A);
        else hipLaunchKernelGGL(attnp_tiles_kernel<8>, grid, t, 0, st, A);
        if (A.n_split > 1) launch_join(L, st);
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

int plan_attn8(sihip_ctx *ctx, const sihip_kv_cache *cache, const sihip_kv_batch *batch, const sihip_attn_paged *a,
               AttnPPlan &P) {
    const char *fn = "attn_paged_dev";
    if (!ctx) return set_err(ctx, SIHIP_EINVAL, "%s: NULL argument", fn);
    CacheArgs C;
    const int rc = check_cache(ctx, fn, cache, C);
    return rc ? rc : plan_attn(ctx, fn, C, ap_tile_waves(C.hd), batch, a, P);
}

}  // namespace

extern "C" int sihip_attn_paged_workspace(sihip_ctx *ctx, const sihip_kv_cache *cache, const sihip_kv_batch *batch,
                                          const sihip_attn_paged *args, uint64_t *bytes) {
    if (!bytes) return set_err(ctx, SIHIP_EINVAL, "attn_paged_workspace: NULL argument");
    AttnPPlan P;
    const int rc = plan_attn8(ctx, cache, batch, args, P);
    if (rc) return rc;
    *bytes = P.part_bytes() ? kCounterBytes + P.part_bytes() : 0;
    return SIHIP_OK;
}

extern "C" int sihip_attn_paged_dev(sihip_ctx *ctx, const sihip_kv_cache *cache, const sihip_kv_batch *batch,
                                    const sihip_attn_paged *args, void *stream) {
    AttnPPlan P;
    const int rc = plan_attn8(ctx, cache, batch, args, P);
    if (rc || P.n == 0) return rc;
    return run_attn(ctx, "attn_paged_dev", P, args, (hipStream_t)stream,
                    [&](const AttnPLaunch &L) { return launch_attn(ctx, L, (hipStream_t)stream); });
}
