// Entry points of the paged 4-bit KV cache (declarations in include/sihip.h).
#include "attnp4.h"
#include "kvcache4.h"
#include "kvhost.h"

using namespace sihip;

namespace {

int check_cache4(sihip_ctx *ctx, const char *fn, const sihip_kv4_cache *c, Cache4Args &C) {
    if (!ctx) return set_err(ctx, SIHIP_EINVAL, "%s: NULL argument", fn);
    if (!c || !c->k || !c->v || !c->k_sub || !c->v_sub || !c->k_scale || !c->v_scale)
        return set_err(ctx, SIHIP_EINVAL, "%s: NULL cache", fn);
    const int rc = check_sizes(ctx, fn, c->block, c->head_dim, 32, c->n_head_kv, c->n_pages);
    if (rc) return rc;
    for (const void *p : {(const void *)c->k, (const void *)c->v, (const void *)c->k_sub, (const void *)c->v_sub,
                          (const void *)c->k_scale, (const void *)c->v_scale})
        if (!aligned(p, 16)) return set_err(ctx, SIHIP_EINVAL, "%s: the cache's arrays must be 16-byte aligned", fn);
    C = {c->k, c->v, c->k_sub, c->v_sub, c->k_scale, c->v_scale, c->n_pages, (int)c->n_head_kv, (int)c->head_dim,
         block_shift(c->block)};
    return SIHIP_OK;
}

}  // namespace

extern "C" int sihip_kv4_append_dev(sihip_ctx *ctx, const sihip_kv4_cache *cache, const sihip_kv_batch *batch,
                                    const sihip_kv_rows *rows, void *stream) {
    const char *fn = "kv4_append_dev";
    Append4Args A;
    int64_t gx = 0;
    int rc = check_cache4(ctx, fn, cache, A.C);
    if (!rc) rc = check_batch(ctx, fn, batch, cache->block, A.R);
    if (!rc) rc = check_rows(ctx, fn, rows, A.R, A.C.n_kv, A.C.hd, A.P, A.Q);
    if (!rc) rc = append_grid(ctx, fn, A.R, A.C.n_kv, cache->block, gx);
    if (rc || !gx) return rc;
    A.k = rows->k;
    A.v = rows->v;
    A.ldk = rows->ldk;
    A.ldv = rows->ldv;
    A.wide = aligned(A.k, 16) && A.ldk % 4 == 0 && aligned(A.v, 16) && A.ldv % 4 == 0;
    const OnDevice on(ctx->device);
    hipLaunchKernelGGL(kv4_append_kernel, dim3((unsigned)gx, (unsigned)batch->n_req, A.Q.q ? 3 : 2), dim3(k4Threads), 0,
                       (hipStream_t)stream, A);
    return launched(ctx, "kv4_append");
}

extern "C" int sihip_kv4_read_dev(sihip_ctx *ctx, const sihip_kv4_cache *cache, const int64_t *slots, int64_t n,
                                  float *k, int64_t ldk, float *v, int64_t ldv, void *stream) {
    const char *fn = "kv4_read_dev";
    Read4Args A;
    const int rc = check_cache4(ctx, fn, cache, A.C);
    if (rc) return rc;
    const int64_t width = (int64_t)A.C.n_kv * A.C.hd;
    if (n < 0 || n > INT32_MAX || ldk < width || ldv < width)
        return set_err(ctx, SIHIP_EINVAL, "%s: %lld rows of %lld values at ldk %lld, ldv %lld", fn, (long long)n,
                       (long long)width, (long long)ldk, (long long)ldv);
    if (n == 0) return SIHIP_OK;
    if (!slots || !k || !v || !aligned(slots, 8) || !aligned(k, 4) || !aligned(v, 4))
        return set_err(ctx, SIHIP_EINVAL, "%s: slots must be an int64 array, k and v f32 arrays", fn);
    A.slots = slots;
    A.k = k;
    A.v = v;
    A.n = n;
    A.ldk = ldk;
    A.ldv = ldv;
    A.wide = aligned(k, 16) && ldk % 4 == 0 && aligned(v, 16) && ldv % 4 == 0;
    // (as sihip_kv_read_dev chooses)
    const bool few = (n + 63) / 64 * A.C.n_kv * 2 < 4 * ctx->n_cu;
    const int64_t slots_per = few ? 16 : 64, gx = (n + slots_per - 1) / slots_per;
    if (gx * kReadThreads > UINT32_MAX)
        return set_err(ctx, SIHIP_EINVAL, "%s: %lld rows have no grid", fn, (long long)n);
    const OnDevice on(ctx->device);
    hipLaunchKernelGGL(few ? kv4_read_kernel<16> : kv4_read_kernel<64>, dim3((unsigned)gx, (unsigned)A.C.n_kv, 2),
                       dim3(kReadThreads), 0, (hipStream_t)stream, A);
    return launched(ctx, "kv4_read");
}

// ---- attention ------------------------------------------------------------------

namespace {

int plan_attn4(sihip_ctx *ctx, const sihip_kv4_cache *cache, const sihip_kv_batch *batch, const sihip_attn_paged *a,
               Cache4Args &C, AttnPPlan &P) {
    const char *fn = "attn_paged4_dev";
    const int rc = check_cache4(ctx, fn, cache, C);
    if (rc) return rc;
    return plan_attn(ctx, fn, {(int8_t *)C.k, (int8_t *)C.v, nullptr, nullptr, C.n_pages, C.n_kv, C.hd, C.shift}, ap4_tile_waves(C.hd), batch, a,
                     P);
}

int launch_attn4(sihip_ctx *ctx, const Cache4Args &C, const AttnPLaunch &L, hipStream_t st) {
    Attn4Args A;
    (AttnPArgs &)A = L.A;
    A.ksub = C.ksub;
    A.vsub = C.vsub;
    A.kd = C.ks;
    A.vd = C.vs;
    const int hd = C.hd, z = A.placed ? 1 : A.n_req;
    if (L.waves) {
        const dim3 grid((unsigned)L.gx, (unsigned)A.n_split, (unsigned)z), t(L.waves * 64);
        if (hd <= 64) hipLaunchKernelGGL(attnp4_tiles_kernel<4>, grid, t, 0, st, A);
        else if (hd <= 96) hipLaunchKernelGGL(attnp4_tiles_kernel<6>, grid, t, 0, st, A);
        else hipLaunchKernelGGL(attnp4_tiles_kernel<8>, grid, t, 0, st, A);
        if (A.n_split > 1) launch_join(L, st);
        return launched(ctx, "attn_paged4");
    }
    const dim3 grid((unsigned)L.gx, A.placed ? 1u : (unsigned)C.n_kv, (unsigned)z), t(L.row_waves * 64);
    // Up to 8 rows of heads up to 64, 4 of heads up to 128, 2 of wider ones: a column for each of
    // their groups of dims
    const int64_t rows = (int64_t)A.R.max_q * A.G;
#define SIHIP_AP4G(KD, NK, ND, TT, NG)                                                                                 \
    if (rows <= 16 / NG) {                                                                                             \
        if (L.row_waves == 1) hipLaunchKernelGGL((attnp4_groups_kernel<KD, NK, ND, TT, 1, NG>), grid, t, 0, st, A);    \
        else hipLaunchKernelGGL((attnp4_groups_kernel<KD, NK, ND, TT, 4, NG>), grid, t, 0, st, A);                     \
        return launched(ctx, "attn_paged4");                                                                           \
    }
    if (hd <= 64) { SIHIP_AP4G(16, 1, 4, 4, 2) }
    else if (hd <= 128) { SIHIP_AP4G(32, 1, 8, 4, 4) }
    else if (hd <= 192) { SIHIP_AP4G(32, 2, 12, 2, 8) }
    else { SIHIP_AP4G(32, 2, 16, 2, 8) }
#undef SIHIP_AP4G
#define SIHIP_AP4R(KD, NK, ND, TT)                                                                                     \
    if (L.row_waves == 1) hipLaunchKernelGGL((attnp4_rows_kernel<KD, NK, ND, TT, 1>), grid, t, 0, st, A);              \
    else hipLaunchKernelGGL((attnp4_rows_kernel<KD, NK, ND, TT, 4>), grid, t, 0, st, A);
    if (hd <= 64) { SIHIP_AP4R(16, 1, 4, 4) }
    else if (hd <= 128) { SIHIP_AP4R(32, 1, 8, 4) }
    else if (hd <= 192) { SIHIP_AP4R(32, 2, 12, 2) }
    else { SIHIP_AP4R(32, 2, 16, 2) }
#undef SIHIP_AP4R
    return launched(ctx, "attn_paged4");
}

}  // namespace

extern "C" int sihip_attn_paged4_workspace(sihip_ctx *ctx, const sihip_kv4_cache *cache, const sihip_kv_batch *batch,
                                           const sihip_attn_paged *args, uint64_t *bytes) {
    if (!bytes) return set_err(ctx, SIHIP_EINVAL, "attn_paged4_workspace: NULL argument");
    AttnPPlan P;
    Cache4Args C;
    const int rc = plan_attn4(ctx, cache, batch, args, C, P);
    if (rc) return rc;
    *bytes = P.part_bytes() ? kCounterBytes + P.part_bytes() : 0;
    return SIHIP_OK;
}

extern "C" int sihip_attn_paged4_dev(sihip_ctx *ctx, const sihip_kv4_cache *cache, const sihip_kv_batch *batch,
                                     const sihip_attn_paged *args, void *stream) {
    AttnPPlan P;
    Cache4Args C;
    const int rc = plan_attn4(ctx, cache, batch, args, C, P);
    if (rc || P.n == 0) return rc;
    return run_attn(ctx, "attn_paged4_dev", P, args, (hipStream_t)stream,
                    [&](const AttnPLaunch &L) { return launch_attn4(ctx, C, L, (hipStream_t)stream); });
}
