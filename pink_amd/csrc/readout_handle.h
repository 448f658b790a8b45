// What the sources of the read-out share: the handle that pink_hip_readout_* work on, its workspace and errors, and sums over a wave.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <new>

#include "pink_hip.h"

struct pink_hip_readout {
    pink_hip_readout_config cfg;
    hipStream_t own, stream;
    void *work;
    size_t work_bytes;
    bool recorded;                 // a graph holds the address of `work`
    struct Former *former;         // workspaces that graphs hold and calls have outgrown
    char err[320];
};

struct Former {
    void *work;
    Former *next;
};

inline thread_local char g_readout_error[320];

namespace {

constexpr uint32_t kMaxSize = 1u << 20;

// Sums and maxima over a wave by DPP, within rows of sixteen and across them into lane 63: no LDS round trips.  The order is fixed.
#define PINK_DPP_ALL(op)                                       \
    op(0xb1, 0xf);      /* quad_perm [1, 0, 3, 2] */           \
    op(0x4e, 0xf);      /* quad_perm [2, 3, 0, 1] */           \
    op(0x141, 0xf);     /* row_half_mirror */                  \
    op(0x140, 0xf);     /* row_mirror */                       \
    op(0x142, 0xa);     /* row_bcast:15 into rows 1 and 3 */   \
    op(0x143, 0xc)      /* row_bcast:31 into rows 2 and 3 */

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v)
{
#define PINK_DPP_MAX(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false))
    PINK_DPP_ALL(PINK_DPP_MAX);
#undef PINK_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ float wave_sum(float v)
{
#define PINK_DPP_ADD(ctrl, rows) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, rows, 0xf, false))
    PINK_DPP_ALL(PINK_DPP_ADD);
#undef PINK_DPP_ADD
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

__device__ __forceinline__ float wave_max(float v)
{
    constexpr int kLeast = (int)0xff800000;                // minus infinity, for rows that a step leaves alone
#define PINK_DPP_MAX(ctrl, rows) v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(kLeast, __float_as_int(v), ctrl, rows, 0xf, false)))
    PINK_DPP_ALL(PINK_DPP_MAX);
#undef PINK_DPP_MAX
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Zeros, by a kernel: a recorded memset has not always been replayed right in graphs.
__global__ __launch_bounds__(256) void k_clear(uint8_t *at, uint64_t bytes)
{
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < bytes; i += (uint64_t)gridDim.x * 256) at[i] = 0;
}

int fail(pink_hip_readout *r, int code, const char *what, const char *why = nullptr)
{
    char *const to = r ? r->err : g_readout_error;
    std::snprintf(to, 320, why ? "%s: %s" : "%s", what, why);
    if (code == PINK_HIP_ENOMEM || code == PINK_HIP_EDEVICE) (void)hipGetLastError();          // (returned here, it is no later launch's)
    return code;
}

#define HIP_TRY(r, call)                                                                                              \
    do {                                                                                                              \
        const hipError_t e_ = (call);                                                                                 \
        if (e_ != hipSuccess)                                                                                         \
            return fail(r, e_ == hipErrorOutOfMemory ? PINK_HIP_ENOMEM : PINK_HIP_EDEVICE, #call, hipGetErrorString(e_)); \
    } while (0)

#define TRY(expr)                            \
    do {                                     \
        const int rc_ = (expr);              \
        if (rc_ != PINK_HIP_OK) return rc_;  \
    } while (0)

#define REFUSE(r, condition, what)                                   \
    do {                                                             \
        if (condition) return fail(r, PINK_HIP_EINVAL, what);        \
    } while (0)

int launched(pink_hip_readout *r, const char *what)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PINK_HIP_OK : fail(r, PINK_HIP_EDEVICE, what, hipGetErrorString(e));
}

// A launch has at most 2^32 - 1 threads.
bool too_many(uint64_t blocks, uint32_t threads) { return blocks * threads > 0xffffffffu; }

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

size_t element_bytes(const pink_hip_readout *r) { return r->cfg.element == PINK_HIP_ELEMENT_BFLOAT ? 2 : 4; }

// The workspace holds so many bytes from here on.  One whose address a recorded graph may hold is kept beside the next until the handle
// is destroyed.
int grow(pink_hip_readout *r, size_t bytes)
{
    hipStreamCaptureStatus capture;
    HIP_TRY(r, hipStreamIsCapturing(r->stream, &capture));
    if (capture != hipStreamCaptureStatusNone) {
        if (bytes > r->work_bytes) return fail(r, PINK_HIP_ESTATE, "a recorded call needs a larger workspace: pink_hip_readout_reserve before");
        r->recorded = true;
    }
    if (bytes <= r->work_bytes) return PINK_HIP_OK;
    HIP_TRY(r, hipStreamSynchronize(r->stream));
    if (r->recorded) {
        Former *const kept = new (std::nothrow) Former{r->work, r->former};
        if (!kept) return fail(r, PINK_HIP_ENOMEM, "pink_hip_readout: out of memory");
        r->former = kept;
    } else if (r->work) {
        HIP_TRY(r, hipFree(r->work));
    }
    r->work = nullptr;
    r->work_bytes = 0;
    r->recorded = false;
    HIP_TRY(r, hipMalloc(&r->work, bytes));
    r->work_bytes = bytes;
    return PINK_HIP_OK;
}

}  // namespace
