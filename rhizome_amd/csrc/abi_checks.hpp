// abi_checks.hpp -- argument checks shared by the C boundaries' files.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "gdr_internal.hpp"

namespace rhz {
namespace abi {

inline rhz_status fail(rhz_status s, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return rhz::record_error(s, buf);
}

inline rhz_status ok() { return rhz::record_error(RHZ_OK, ""); }

inline rhz_status hip_status(hipError_t e, const char* what) {
    if (e == hipSuccess) return ok();
    return fail(RHZ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

constexpr int64_t kMaxIndex = INT32_MAX;

inline bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

// A buffer of a call, for the checks that run over all of them.
struct Buffer {
    const char* name;
    const void* p;
    size_t bytes;
    size_t align;
    bool needed, written;
};

// Every needed buffer given, every one aligned, and none that is written
// overlapping another.
inline rhz_status check_buffers(const Buffer* b, int n) {
    for (int i = 0; i < n; ++i) {
        if (b[i].needed && !b[i].p) return fail(RHZ_ERR_INVALID_ARG, "%s is NULL", b[i].name);
        if (misaligned(b[i].p, b[i].align)) return fail(RHZ_ERR_INVALID_ARG, "%s is not aligned", b[i].name);
    }
    for (int i = 0; i < n; ++i) {
        if (!b[i].written || !b[i].p) continue;
        const uintptr_t i0 = reinterpret_cast<uintptr_t>(b[i].p), i1 = i0 + b[i].bytes;
        for (int j = 0; j < n; ++j) {
            const uintptr_t j0 = reinterpret_cast<uintptr_t>(b[j].p), j1 = j0 + b[j].bytes;
            if (j != i && b[j].p && i0 < j1 && j0 < i1)
                return fail(RHZ_ERR_INVALID_ARG, "%s overlaps %s", b[i].name, b[j].name);
        }
    }
    return ok();
}

inline rhz_status check_workspace(const void* p, size_t have, size_t need) {
    if (need == 0) return ok();
    if (!p) return fail(RHZ_ERR_WORKSPACE, "workspace is NULL (%zu bytes needed)", need);
    if (have < need) return fail(RHZ_ERR_WORKSPACE, "workspace has %zu bytes, %zu needed", have, need);
    if (misaligned(p, 256)) return fail(RHZ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    return ok();
}

}  // namespace abi
}  // namespace rhz
