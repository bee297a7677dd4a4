// Entry points of log probabilities (declarations in include/sihip.h).
#include "logprobs.h"

#include <algorithm>

#include "launch.h"

using namespace sihip;

namespace {

// Checks, and the splits of a row: until the device has two workgroups a CU, and none shorter than one round of
// loads. Each split ends with reductions and a choice, in turn, that no loads cover. us with 1 / 2 / 4 /
// 8 a CU: 500 rows of 151936, no tokens chosen 53 / 50 / 53 / 54, 20 tokens 80 / 67 / 82 / 73; 64 of 151936 14 / 12 / 14 / 22 and
// 23 / 19 / 22 / 35; 200 of 151936 24 / 24 / 26 / 27 and 40 / 36 / 36 / 44; 64 of 32003, which have 8 splits at
// most, 7.3 / 7.9 / 7.8 / 7.6 and 13.1 / 13.8 / 13.8 / 13.9.
int plan_logprobs(sihip_ctx *ctx, const sihip_logprobs *a, LogprobArgs &A, size_t &part_bytes) {
    const char *fn = "logprobs_dev";
    if (!ctx || !a) return set_err(ctx, SIHIP_EINVAL, "%s: NULL argument", fn);
    if (a->n_rows < 0 || a->n_rows >= 1 << 24 || a->n_vocab < 1 || a->n_vocab > INT32_MAX || a->ld < a->n_vocab)
        return set_err(ctx, SIHIP_EINVAL, "%s: %lld rows of %lld logits at ld %lld", fn, (long long)a->n_rows,
                       (long long)a->n_vocab, (long long)a->ld);
    if (a->n_token < 0 || a->n_token > INT32_MAX || a->n_top < 0 || a->n_top > kLpMostTop || a->n_top > a->n_vocab)
        return set_err(ctx, SIHIP_EINVAL, "%s: n_token %lld, n_top %lld (at most %d and n_vocab)", fn, (long long)a->n_token,
                       (long long)a->n_top, kLpMostTop);
    part_bytes = 0;
    A = {};
    if (a->n_rows == 0) return SIHIP_OK;
    if (!a->logits || !aligned(a->logits, 4) || !aligned(a->token, 4) || !aligned(a->logprob, 4) || !aligned(a->entropy, 4) ||
        !aligned(a->top_id, 4) || !aligned(a->top_logprob, 4))
        return set_err(ctx, SIHIP_EINVAL, "%s: NULL logits, or an array that is not 4-byte aligned", fn);
    if (a->n_token > 0 && !a->token != !a->logprob)
        return set_err(ctx, SIHIP_EINVAL, "%s: token and logprob go together", fn);
    if (a->n_top > 0 && (!a->top_id || !a->top_logprob)) return set_err(ctx, SIHIP_EINVAL, "%s: NULL top_id or top_logprob", fn);
    A.x = a->logits;
    A.ld = a->ld;
    A.n = a->n_vocab;
    A.token = a->token;
    A.n_token = a->n_token;
    A.logprob = a->n_token ? a->logprob : nullptr;
    A.entropy = a->entropy;
    A.n_top = (int)a->n_top;
    A.top_id = a->top_id;
    A.top_logprob = a->top_logprob;
    const int64_t granules = (A.n + 6) / 4, round = kLpThreads * kLpGroup;  // (a row may begin inside one)
    const int64_t want = (2 * ctx->n_cu + a->n_rows - 1) / a->n_rows, most = (granules + round - 1) / round;
    const int64_t n = std::max<int64_t>(1, std::min<int64_t>({want, most, A.n_top ? kLpMostSplits : kLpThreads}));
    A.per_split = ((granules + n - 1) / n + 3) / 4 * 4;  // (whole 64 bytes, of splits of one length)
    A.n_split = (int)((granules + A.per_split - 1) / A.per_split);
    if (A.n_split > 1) part_bytes = (size_t)a->n_rows * lp_part_bytes(A.n_top, A.n_split);
    return SIHIP_OK;
}

}  // namespace

extern "C" int sihip_logprobs_workspace(sihip_ctx *ctx, const sihip_logprobs *args, uint64_t *bytes) {
    if (!bytes) return set_err(ctx, SIHIP_EINVAL, "logprobs_workspace: NULL argument");
    LogprobArgs A;
    size_t part;
    const int rc = plan_logprobs(ctx, args, A, part);
    if (rc) return rc;
    *bytes = part ? kCounterBytes + part : 0;
    return SIHIP_OK;
}

extern "C" int sihip_logprobs_dev(sihip_ctx *ctx, const sihip_logprobs *args, void *stream) {
    LogprobArgs A;
    size_t part_bytes;
    const int rc = plan_logprobs(ctx, args, A, part_bytes);
    if (rc || args->n_rows == 0) return rc;
    const hipStream_t st = (hipStream_t)stream;
    return with_workspace(ctx, "logprobs_dev", part_bytes, args->workspace, args->workspace_bytes, st,
                          [&](uint32_t *cnt, uint8_t *part) {
                              A.cnt = cnt;
                              A.part = part;
                              const dim3 grid((unsigned)(args->n_rows * A.n_split));
                              if (A.n_top) hipLaunchKernelGGL(logprobs_kernel<true>, grid, dim3(kLpThreads), 0, st, A);
                              else hipLaunchKernelGGL(logprobs_kernel<false>, grid, dim3(kLpThreads), 0, st, A);
                              return launched(ctx, "logprobs");
                          });
}
