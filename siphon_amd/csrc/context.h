// The state of a context and what its entry points share: options, error
// messages, workspaces and the order of launches that use them. Included by
// every translation unit of libsiphon_hip.so.
#pragma once

#include <hip/hip_runtime.h>

#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <vector>

#include "../../include/sihip.h"

// Tuning knobs, read once from the environment at sihip_init (variable
// SIHIP_<NAME>) and changed afterwards only through sihip_set_option; a
// negative value means "the built-in rule".
struct Options {
    int64_t wg_per_cu = -1;    // matvec workgroups per CU when rows exceed waves (rule: 2)
    int64_t wave_target = -1;  // row tiles a matvec layout aims for (rule: 800)
    int64_t split_elems = -1;  // column-slice length in elements, 0: none (rule: kSliceElems)
    int64_t tile_cols = -1;    // matvec tile width at upload (rule: choose_G)
    int64_t gemm_min_m = -1;   // smallest M on the matrix cores (rule: 5)
    int64_t gemm_mt = -1;      // GEMM m-tile rows / 32 (rule: by M)
    int64_t gemm_sbk = -1;     // GEMM K-slice length in super-blocks, 0: none (rule: by tiles)
    int64_t gemm2_min_m = -1;  // smallest M on the 16x16 Q4_K GEMM (rule: kGemm2MinM)
    int64_t gemm2_waves = -1;  // waves per SIMD of the 16x16 GEMMs, 1 or 2 (rule: 2)
    int64_t gemm6_min_m = -1;  // smallest M on the Q6_K GEMM (rule: kGemm6MinM)
    int64_t gemmh_min_m = -1;  // smallest M on the F16 GEMM (rule: kGemmhMinM)
    int64_t gemmq_min_m = -1;  // smallest M on the Q4_0/Q5_0/Q8_0 GEMM (rule: kGemmqMinM)
    int64_t gemmq_xmode = -1;  // Q8_0-pair GEMM record mode 0 or 1 (gemmq_kernel XM; rule: 1 where it fits)
    int64_t gemmq_fuse = -1;   // Q8_0-pair GEMM quantizing X itself (XM 2) at 16-row m blocks, 0: off (rule: on)
    int64_t gemmh_fuse = -1;   // F16 GEMM converting X itself (XF) at 16-row m blocks, 0: off (rule: on)
    int64_t attn_fuse = -1;    // decode attention in one launch up to 512 k positions, at most kAttnFuseCap, 0: three (rule: attn_fuse_max)
    int64_t gemm2s_max_m = -1; // largest M on the small-M Q4_K GEMM, 0: none (rule: 16)
    int64_t gemmks_max_m = -1; // largest M on the small-M K-quant GEMM, 0: none (rule: 16)
    int64_t gemmks_q4k = -1;   // Q4_K small M on gemmks.h (1) or gemm2s.h (0) (rule: 0)
    int64_t gemms_waves = -1;  // waves per workgroup of the small-M GEMMs, 4 or 8 (rule: by rows)
    int64_t gemmkf_max_m = -1; // largest M on the fused small-M K-quant launch, 0: none (rule: 8)
    int64_t gemmkf_sbk = -1;   // its K-slice length in super-blocks, 0: fewest slices (rule: by tiles)
    int64_t gemmsk_max_m = -1; // largest M on the short-prompt K-quant GEMM, 0: none (rule: kGemmSKMaxM)
    int64_t gemmd_min_m = -1;  // smallest M on the F16 and Q8_0-pair GEMM of prompts, 0: never (rule: kGemmDMinM)
    int64_t gemmx_min_m = -1;  // smallest M on the K-quant GEMM of longer prompts, 0: never (rule: past GEMMSK_MAX_M)
    int64_t ring_mt = -1;      // m tiles of the ring-buffered GEMMs (gemmx.h, gemmd.h), where they have that instance (rule: plan_tiles)
    int64_t ring_sbk = -1;     // their K-slice length in steps, 0: none (rule: plan_tiles)
    int64_t gemm_group = -1;   // Q4_K matrices over one X in one 16x16 GEMM launch, 0: off (rule: on)
    int64_t attnp_large = -1;  // paged attention: large row blocks (1), blocks of 16 rows (0) (rule: attn_waves)
    int64_t attnp_row_waves = -1; // paged attention: waves that share a 16-row block's keys (1, 4) (rule: plan_launch)
    int64_t attnp_splits = -1; // paged attention: splits of a row block's keys, 1..64 (rule: plan_launch)
    int64_t q80_scalar = -1;   // Q8_0 activations by the scalar quantizer (reference
                               // kernels.c:542-558, its SI_SCALAR mode), 1: on (rule: off)
};

// Order of launches that share mutable device state across streams: a
// context's GEMM and attention workspaces, a column-sliced weight's partial
// sums and arrival counters. While all of them come on one stream nothing
// is added. The first launch on a second stream waits for the device to
// drain (hipDeviceSynchronize; no stream handle of an earlier call is
// touched, since the caller may have destroyed it); from then on the state
// carries an event recorded after each of its launches, and a launch on
// another stream than the last one waits for that event. Launches made
// during a graph capture are neither recorded nor made to wait: a captured
// sequence is ordered by its graph, and its replays must not overlap eager
// use of the same state on another stream.
struct StreamOrder {
    hipStream_t last = nullptr;
    bool used = false;
    bool multi = false;
    hipEvent_t ev = nullptr;
};

struct sihip_ctx {
    int device;
    int n_cu;
    size_t lds_limit;
    hipStream_t stream;  // for host-pointer entry points
    char err[512];
    Options opt;
    void *d_in = nullptr;
    size_t d_in_cap = 0;
    void *d_out = nullptr;
    size_t d_out_cap = 0;
    uint8_t *h_stage = nullptr;  // pinned staging of sihip_gemv (kStageBytes), made on first use
    uint8_t *h_stage_dev = nullptr;  // its device address
    bool h_stage_tried = false;
    uint32_t h_seq = 0;  // calls that used it
    void *d_aux = nullptr;
    size_t d_aux_cap = 0;
    void *d_ws = nullptr;  // prefill GEMM: quantized activation planes
    size_t d_ws_cap = 0;
    void *d_gpart = nullptr;  // prefill GEMM K slices: partial sums
    size_t d_gpart_cap = 0;
    uint32_t *d_gcnt = nullptr;  // prefill GEMM K slices: arrival counters (zero between calls)
    void *d_attn = nullptr;  // decode attention: scores and f16 probabilities
    size_t d_attn_cap = 0;
    // workspaces replaced by larger ones: a graph captured earlier may still
    // hold their addresses, so they stay allocated until sihip_shutdown
    std::vector<void *> retired;
    // this device's copy of the static scratch of sihip_gemm_dev_noalloc
    uint8_t *scratch = nullptr;
    StreamOrder order;  // of the launches using the workspaces above
};

// Arrival counters of K-sliced GEMM tiles, allocated (and zeroed) at
// sihip_init; launches with more tiles than this are not sliced.
constexpr int64_t kGemmCounters = 65536;

// What follows is one copy for the library's translation units and not exported
// from it: the host's process may hold the same names.
#pragma GCC visibility push(hidden)

// the last failure of sihip_init, and of calls without a context
inline char g_init_err[512];

inline int set_err(sihip_ctx *ctx, int code, const char *fmt, ...) {
    char *dst = ctx ? ctx->err : g_init_err;
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(dst, 512, fmt, ap);
    va_end(ap);
    return code;
}

#define HIP_OK(ctx, call)                                                              \
    do {                                                                               \
        hipError_t e_ = (call);                                                        \
        if (e_ != hipSuccess)                                                          \
            return set_err((ctx), SIHIP_EDEVICE, "%s: %s", #call, hipGetErrorString(e_)); \
    } while (0)

// True if work on st is being captured into a graph (allocations and
// synchronous calls are not allowed then).
inline bool capturing(hipStream_t st) {
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &cs) != hipSuccess) return false;
    return cs != hipStreamCaptureStatusNone;
}

// Before a launch on stream st that uses the state ordered by o.
inline int order_before(sihip_ctx *ctx, StreamOrder &o, hipStream_t st) {
    if (!o.used || o.last == st || capturing(st)) return SIHIP_OK;
    if (!o.multi) {
        HIP_OK(ctx, hipDeviceSynchronize());
        HIP_OK(ctx, hipEventCreateWithFlags(&o.ev, hipEventDisableTiming));
        o.multi = true;
        return SIHIP_OK;
    }
    HIP_OK(ctx, hipStreamWaitEvent(st, o.ev, 0));
    return SIHIP_OK;
}

// After that launch was enqueued.
inline int order_after(sihip_ctx *ctx, StreamOrder &o, hipStream_t st) {
    if (capturing(st)) return SIHIP_OK;
    o.used = true;
    o.last = st;
    if (o.multi) HIP_OK(ctx, hipEventRecord(o.ev, st));
    return SIHIP_OK;
}

inline void order_free(StreamOrder &o) {
    if (o.ev) (void)hipEventDestroy(o.ev);
    o = StreamOrder();
}

// A context workspace of at least `bytes`. Growing it allocates a new
// buffer and retires the old one (kept until sihip_shutdown, since a graph
// captured before may reference it); under graph capture growing is an
// error, as allocation is not allowed there.
inline int ensure(sihip_ctx *ctx, void **buf, size_t *cap, size_t bytes, hipStream_t st = nullptr) {
    if (*cap >= bytes) return SIHIP_OK;
    if (st && capturing(st))
        return set_err(ctx, SIHIP_EINVAL,
                       "workspace of %zu bytes needed during graph capture (it holds %zu): run "
                       "the call once outside capture first, or use sihip_gemm_dev_noalloc",
                       bytes, *cap);
    void *nb = nullptr;
    if (hipMalloc(&nb, bytes) != hipSuccess)
        return set_err(ctx, SIHIP_ENOMEM, "device allocation of %zu bytes failed", bytes);
    if (*buf) ctx->retired.push_back(*buf);
    *buf = nb;
    *cap = bytes;
    return SIHIP_OK;
}

#pragma GCC visibility pop
