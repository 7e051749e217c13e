// xq_host.h — host-side helpers of the C entry points: storage sizes, alignment,
// error messages.
#pragma once

#include <stdarg.h>
#include <stdio.h>

#include "xq_kernels.h"

namespace xq {

inline size_t type_size(int t) {  // ggml_type_size: bytes of one element or block
    switch (t) {
    case XQ_TYPE_F32: return 4;
    case XQ_TYPE_F16:
    case XQ_TYPE_BF16: return 2;
    case XQ_TYPE_Q8_0: return 34;
    case XQ_TYPE_Q4_0: return 18;
    case XQ_TYPE_E5M2: return 1;
    default: return 0;
    }
}

inline size_t record_bytes(int t, int64_t d) {
    switch (t) {
    case XQ_TYPE_F32: return (size_t)d * 4;
    case XQ_TYPE_F16:
    case XQ_TYPE_BF16: return (size_t)d * 2;
    case XQ_TYPE_Q8_0: return (size_t)(d / 32) * 34;
    case XQ_TYPE_Q4_0: return (size_t)(d / 32) * 18;
    case XQ_TYPE_E5M2: return (size_t)d;
    default: return 0;
    }
}

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

// Sets the calling thread's message; XQ_OK clears it.
inline xq_status failf(xq_status st, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return set_error(st, buf);
}
inline xq_status done_ok() { return set_error(XQ_OK, ""); }

}  // namespace xq
