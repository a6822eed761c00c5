// What the library's other translation units need from the one that owns the contexts
// (ngraph_hip.hip): the stream launches go to at this moment (a recording redirects it), the
// device, and the text of the last failure.  Not part of the C ABI.
#pragma once
#include <hip/hip_runtime.h>

#include "ngraph_hip.h"

#define NGH_INTERNAL __attribute__((visibility("hidden")))

namespace ngh {

struct ContextView {
    hipStream_t stream;
    int device;
    int cus;
    bool capturing;
};

NGH_INTERNAL ContextView view_of(const ngh_context* ctx);
// Records the message for ngh_last_error and returns `code`.
NGH_INTERNAL int report(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// Launches go to the context's device whatever device the calling thread has current.
class DeviceScope {
public:
    explicit DeviceScope(int device) {
        if (hipGetDevice(&before_) != hipSuccess) before_ = -1;
        changed_ = before_ != device;
        ok_ = !changed_ || hipSetDevice(device) == hipSuccess;
    }
    ~DeviceScope() {
        if (changed_ && before_ >= 0) (void)hipSetDevice(before_);
    }
    bool ok() const { return ok_; }

private:
    int before_ = -1;
    bool changed_ = false, ok_ = false;
};

// Bytes a view of `rows` rows of `width` elements, `stride` elements apart, spans.
inline unsigned long long span_bytes(int64_t rows, int64_t width, int64_t stride, int itemsize) {
    if (rows <= 0 || width <= 0) return 0;
    const __int128 bytes = ((__int128)(rows - 1) * stride + width) * itemsize;
    return bytes < (__int128)1 << 62 ? (unsigned long long)bytes : 1ull << 62;
}

// A grid has fewer than 2^32 threads; calls over more rows than that are launched in slices.
constexpr long long kMostThreads = 1LL << 31;

inline bool spans_overlap(const void* a, unsigned long long an, const void* b, unsigned long long bn) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return an && bn && x < y + bn && y < x + an;
}

}  // namespace ngh

#define NGH_HIP_TRY(expr)                                                                                     \
    do {                                                                                                      \
        hipError_t e_ = (expr);                                                                               \
        if (e_ != hipSuccess)                                                                                 \
            return ngh::report(e_ == hipErrorOutOfMemory ? NGH_E_NOMEM : NGH_E_RUNTIME, "%s failed: %s", #expr, \
                               hipGetErrorString(e_));                                                        \
    } while (0)
