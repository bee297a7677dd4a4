// What entry points on device pointers share on the host: the device they run
// on, launch errors, and the workspace of kernels whose workgroups join through memory.
#pragma once

#include <hip/hip_runtime.h>

#include "context.h"

// one copy for the library's translation units, not exported (context.h)
#pragma GCC visibility push(hidden)

namespace sihip {

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

inline bool aligned(const void *p, uintptr_t n) { return (uintptr_t)p % n == 0; }

inline int launched(sihip_ctx *ctx, const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SIHIP_OK : set_err(ctx, SIHIP_EDEVICE, "%s launch: %s", what, hipGetErrorString(e));
}

// counters at the front of a caller's workspace, whatever the call's size
constexpr size_t kCounterBytes = (size_t)kGemmCounters * 4;

// Runs launch(counters, parts) with `bytes` of parts: in the caller's workspace, or in
// the context's, whose users are ordered. bytes 0: with neither.
template <class Launch>
int with_workspace(sihip_ctx *ctx, const char *fn, size_t bytes, void *own, uint64_t own_bytes, hipStream_t st, Launch launch) {
    const OnDevice on(ctx->device);
    if (!bytes) return launch(nullptr, nullptr);
    if (own) {
        if (own_bytes < kCounterBytes + bytes || !aligned(own, 16))
            return set_err(ctx, SIHIP_EINVAL, "%s: a workspace of %zu bytes, 16-byte aligned, is needed", fn,
                           kCounterBytes + bytes);
        return launch((uint32_t *)own, (uint8_t *)own + kCounterBytes);
    }
    int rc;
    try {
        rc = ensure(ctx, &ctx->d_attn, &ctx->d_attn_cap, bytes, st);
    } catch (...) {
        rc = set_err(ctx, SIHIP_ENOMEM, "%s: out of host memory", fn);
    }
    if (!rc) rc = order_before(ctx, ctx->order, st);
    if (!rc) rc = launch(ctx->d_gcnt, (uint8_t *)ctx->d_attn);
    return rc ? rc : order_after(ctx, ctx->order, st);
}

}  // namespace sihip

#pragma GCC visibility pop
