// What the files of the C ABI (capi.hip, capi_mx.hip) share: error reporting, the
// device's set-up and the argument checks' macros.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

namespace xpuint8 {

// sets the thread's error message, returns code
int fail(int code, const std::string& msg);
// set-up of the current device, once; 0 or an error code
int ensure_device();
// 0, or error 5 with what failed
int launched(hipError_t e, const char* what);

inline hipStream_t as_stream(const void* s) {
    return static_cast<hipStream_t>(const_cast<void*>(s));
}

constexpr int64_t kMaxDim = (int64_t(1) << 31) - 1;

// Every buffer is read and written with 16-byte vector accesses.
#define XPU_NONNULL(p)                                          \
    if (!(p)) return fail(6, #p " must not be null");           \
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0)               \
    return fail(6, #p " must be 16-byte aligned")
#define XPU_ALIGNED_OPT(p)                                      \
    if ((p) && reinterpret_cast<uintptr_t>(p) % 16 != 0)        \
    return fail(6, #p " must be 16-byte aligned")
#define XPU_TRY(expr)              \
    do {                           \
        const int rc_ = (expr);    \
        if (rc_ != 0) return rc_;  \
    } while (0)

}  // namespace xpuint8
