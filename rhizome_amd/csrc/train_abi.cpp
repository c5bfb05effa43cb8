// train_abi.cpp -- the extern "C" boundary of the training operators
// (rhizome_train.h): argument validation, complete before any HIP call, and
// dispatch to the kernel launchers.

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "gdr_internal.hpp"
#include "rhizome_train.h"

namespace {

rhz_status fail(rhz_status s, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return rhz::record_error(s, buf);
}

rhz_status ok() { return rhz::record_error(RHZ_OK, ""); }

rhz_status hip_status(hipError_t e, const char* what) {
    if (e == hipSuccess) return ok();
    return fail(RHZ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

constexpr int64_t kMaxIndex = INT32_MAX;

bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

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
rhz_status check_buffers(const Buffer* b, int n) {
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

rhz_status check_backward(const rhz_gdr_prefill_backward_args* a) {
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    if (a->batch < 1) return fail(RHZ_ERR_INVALID_ARG, "batch must be >= 1 (got %d)", a->batch);
    if (a->seq_len < 0) return fail(RHZ_ERR_INVALID_ARG, "seq_len must be >= 0 (got %d)", a->seq_len);
    if (a->heads < 1) return fail(RHZ_ERR_INVALID_ARG, "heads must be >= 1 (got %d)", a->heads);
    if (a->d_k < 1) return fail(RHZ_ERR_INVALID_ARG, "d_k must be >= 1 (got %d)", a->d_k);
    if (a->d_v < 1) return fail(RHZ_ERR_INVALID_ARG, "d_v must be >= 1 (got %d)", a->d_v);
    if (a->dtype != RHZ_F32 && a->dtype != RHZ_BF16)
        return fail(RHZ_ERR_INVALID_ARG, "dtype must be RHZ_F32 or RHZ_BF16 (got %d)", a->dtype);
    if (a->gate_kind != RHZ_GATE_LOG_ALPHA && a->gate_kind != RHZ_GATE_ALPHA)
        return fail(RHZ_ERR_INVALID_ARG, "gate_kind must be RHZ_GATE_LOG_ALPHA or RHZ_GATE_ALPHA (got %d)",
                    a->gate_kind);
    if (a->d_k > 128) return fail(RHZ_ERR_UNSUPPORTED, "d_k = %d exceeds the backward pass's 128", a->d_k);
    if (a->d_v > 1024) return fail(RHZ_ERR_UNSUPPORTED, "d_v = %d exceeds the supported 1024", a->d_v);
    const int64_t tokens = a->cu_seqlens ? (int64_t)a->seq_len : (int64_t)a->batch * a->seq_len;
    if (tokens * a->heads > kMaxIndex)
        return fail(RHZ_ERR_INVALID_ARG, "tokens * heads = %lld exceeds 2^31 - 1", (long long)(tokens * a->heads));
    if ((int64_t)a->batch * a->heads > kMaxIndex / 128)
        return fail(RHZ_ERR_INVALID_ARG, "batch * heads = %lld is too large", (long long)a->batch * a->heads);
    return ok();
}
}  // namespace

extern "C" {

rhz_status rhz_gdr_prefill_backward_workspace_size(const rhz_gdr_prefill_backward_args* a, size_t* bytes) {
    if (!bytes) return fail(RHZ_ERR_INVALID_ARG, "bytes is NULL");
    const rhz_status s = check_backward(a);
    if (s != RHZ_OK) return s;
    *bytes = rhz::backward_workspace_bytes(*a);
    return ok();
}

rhz_status rhz_gdr_prefill_backward(const rhz_gdr_prefill_backward_args* a, void* stream) {
    rhz_status s = check_backward(a);
    if (s != RHZ_OK) return s;
    const size_t tokens = a->cu_seqlens ? (size_t)a->seq_len : (size_t)a->batch * a->seq_len;
    if (tokens == 0 && !a->grad_initial_state) return ok();
    const size_t es = a->dtype == RHZ_F32 ? 4 : 2, rows = tokens * a->heads;
    const size_t nk = rows * a->d_k * es, nv = rows * a->d_v * es;
    const size_t ns = (size_t)a->batch * a->heads * a->d_v * a->d_k * 4;
    const bool any = tokens > 0;
    const Buffer b[] = {
        {"q", a->q, nk, es, any, false},
        {"k", a->k, nk, es, any, false},
        {"v", a->v, nv, es, any, false},
        {"gate", a->gate, rows * 4, 4, any, false},
        {"beta", a->beta, rows * 4, 4, any, false},
        {"grad_o", a->grad_o, nv, es, any, false},
        {"cu_seqlens", a->cu_seqlens, ((size_t)a->batch + 1) * 4, 4, false, false},
        {"initial_state", a->initial_state, ns, 4, false, false},
        {"grad_final_state", a->grad_final_state, ns, 4, false, false},
        {"grad_q", a->grad_q, nk, es, any, true},
        {"grad_k", a->grad_k, nk, es, any, true},
        {"grad_v", a->grad_v, nv, es, any, true},
        {"grad_gate", a->grad_gate, rows * es, es, any, true},
        {"grad_beta", a->grad_beta, rows * es, es, any, true},
        {"grad_initial_state", a->grad_initial_state, ns, 4, false, true},
        {"workspace", a->workspace, a->workspace_bytes, 1, false, true},
    };
    if ((s = check_buffers(b, sizeof b / sizeof b[0])) != RHZ_OK) return s;
    const size_t need = rhz::backward_workspace_bytes(*a);
    if (need) {
        if (!a->workspace) return fail(RHZ_ERR_WORKSPACE, "workspace is NULL (%zu bytes needed)", need);
        if (a->workspace_bytes < need)
            return fail(RHZ_ERR_WORKSPACE, "workspace has %zu bytes, %zu needed", a->workspace_bytes, need);
        if (reinterpret_cast<uintptr_t>(a->workspace) & 255u)
            return fail(RHZ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    }
    return hip_status(rhz::launch_backward(*a, static_cast<hipStream_t>(stream)), "prefill backward launch");
}

}  // extern "C"
