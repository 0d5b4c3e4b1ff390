// What the library's translation units share: the error buffer and its macros, the context handle.
#pragma once
#include "../../include/t2mi.h"
#include <hip/hip_runtime.h>
#include <stddef.h>

// fills the thread's message (t2_last_error) and returns `code`; defined in t2mi.hip
__attribute__((visibility("hidden"), format(printf, 2, 3))) int fail(int code, const char* fmt, ...);

#define HIP_TRY(expr)                                                                              \
    do {                                                                                           \
        hipError_t e_ = (expr);                                                                    \
        if (e_ != hipSuccess)                                                                      \
            return fail(e_ == hipErrorOutOfMemory ? T2_ENOMEM : T2_EHIP, "%s failed: %s (%s:%d)", #expr, \
                        hipGetErrorString(e_), __FILE__, __LINE__);                                \
    } while (0)

#define T2_TRY(expr)              \
    do {                          \
        int r_ = (expr);          \
        if (r_ != T2_OK) return r_; \
    } while (0)

struct t2_ctx {
    int device;
    hipStream_t stream;
    bool own_stream;
    float* red_ws = nullptr;   // partial sums of the loss reductions (train.h)
    void* voc_ws = nullptr;    // Griffin-Lim workspace (vocoder.h), grown on demand
    size_t voc_ws_bytes = 0;
    unsigned long long scan_wait_ticks = 200000000ull;     // option scan_wait_us, of the 100 MHz clock (recurrence.hip)
};

// Makes the context's device current for the length of a call and the caller's again behind it.
struct DeviceScope {
    int before = -1;
    hipError_t err;
    explicit DeviceScope(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;
    }
    ~DeviceScope() { if (before >= 0) (void)hipSetDevice(before); }
};
