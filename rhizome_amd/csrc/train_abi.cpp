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

rhz_status check_workspace(const void* p, size_t have, size_t need) {
    if (need == 0) return ok();
    if (!p) return fail(RHZ_ERR_WORKSPACE, "workspace is NULL (%zu bytes needed)", need);
    if (have < need) return fail(RHZ_ERR_WORKSPACE, "workspace has %zu bytes, %zu needed", have, need);
    if (misaligned(p, 256)) return fail(RHZ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
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
    if (rhz::exceeds(tokens, a->heads, kMaxIndex))
        return fail(RHZ_ERR_INVALID_ARG, "tokens * heads = %lld * %d exceeds 2^31 - 1", (long long)tokens, a->heads);
    if ((int64_t)a->batch * a->heads > kMaxIndex / 128)
        return fail(RHZ_ERR_INVALID_ARG, "batch * heads = %lld is too large", (long long)a->batch * a->heads);
    return ok();
}

rhz_status check_conv_backward(const rhz_gdr_conv_prepare_backward_args* a) {
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    if (a->batch < 1) return fail(RHZ_ERR_INVALID_ARG, "batch must be >= 1 (got %d)", a->batch);
    if (a->seq_len < 0) return fail(RHZ_ERR_INVALID_ARG, "seq_len must be >= 0 (got %d)", a->seq_len);
    if (a->heads < 1) return fail(RHZ_ERR_INVALID_ARG, "heads must be >= 1 (got %d)", a->heads);
    if (a->d_k < 1 || a->d_v < 1)
        return fail(RHZ_ERR_INVALID_ARG, "d_k and d_v must be >= 1 (got %d, %d)", a->d_k, a->d_v);
    if (a->dtype != RHZ_F32 && a->dtype != RHZ_BF16)
        return fail(RHZ_ERR_INVALID_ARG, "dtype must be RHZ_F32 or RHZ_BF16 (got %d)", a->dtype);
    if (!std::isfinite(a->q_scale)) return fail(RHZ_ERR_INVALID_ARG, "q_scale must be finite");
    if (a->d_k > 512 || a->d_v > 1024)
        return fail(RHZ_ERR_UNSUPPORTED, "d_k = %d, d_v = %d exceed the supported 512 and 1024", a->d_k, a->d_v);
    if (!rhz::conv_prepare_supported(a->dtype, a->d_k, a->d_v)) {
        const int n = a->dtype == RHZ_F32 ? 4 : 8;
        return fail(RHZ_ERR_UNSUPPORTED, "d_k = %d, d_v = %d: need multiples of %d with d_k / %d a power of two up to 64",
                    a->d_k, a->d_v, n, n);
    }
    const int64_t C = (int64_t)a->heads * (2 * a->d_k + a->d_v);
    const int64_t tokens = a->cu_seqlens ? a->seq_len : (int64_t)a->batch * a->seq_len;
    if (rhz::exceeds(tokens, C, kMaxIndex) || rhz::exceeds(a->batch, C * 3, kMaxIndex) || C * 4 > kMaxIndex)
        return fail(RHZ_ERR_INVALID_ARG, "tokens * channels and batch * channels * 3 must stay below 2^31");
    return ok();
}

rhz_status check_norm(int rows, int dim, int dtype, float eps) {
    if (rows < 0) return fail(RHZ_ERR_INVALID_ARG, "rows must be >= 0 (got %d)", rows);
    if (dim < 1) return fail(RHZ_ERR_INVALID_ARG, "dim must be >= 1 (got %d)", dim);
    if (dtype != RHZ_F32 && dtype != RHZ_BF16)
        return fail(RHZ_ERR_INVALID_ARG, "dtype must be RHZ_F32 or RHZ_BF16 (got %d)", dtype);
    if (dim > 8192) return fail(RHZ_ERR_UNSUPPORTED, "dim = %d exceeds the supported 8192", dim);
    if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(RHZ_ERR_INVALID_ARG, "eps must be >= 0 and finite");
    if ((int64_t)rows * dim > kMaxIndex) return fail(RHZ_ERR_INVALID_ARG, "rows * dim exceeds 2^31 - 1");
    return ok();
}

rhz_status norm_backward(const rhz_norm_backward_args* a, bool layer, void* stream) {
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    rhz_status s = check_norm(a->rows, a->dim, a->dtype, a->eps);
    if (s != RHZ_OK) return s;
    if (!layer && a->grad_bias) return fail(RHZ_ERR_INVALID_ARG, "RMSNorm has no bias: grad_bias must be NULL");
    const bool any = a->rows > 0;
    const size_t es = a->dtype == RHZ_F32 ? 4 : 2, n = (size_t)a->rows * a->dim * es, nd = (size_t)a->dim * 4;
    const Buffer b[] = {
        {"grad_y", a->grad_y, n, es, any, false},
        {"x", a->x, n, es, any, false},
        {"weight", a->weight, nd, 4, any, false},
        {"grad_x", a->grad_x, n, es, any, true},
        {"grad_weight", a->grad_weight, nd, 4, true, true},
        {"grad_bias", a->grad_bias, nd, 4, false, true},
        {"workspace", a->workspace, a->workspace_bytes, 1, false, true},
    };
    if ((s = check_buffers(b, sizeof b / sizeof b[0])) != RHZ_OK) return s;
    if ((s = check_workspace(a->workspace, a->workspace_bytes, rhz::norm_backward_workspace_bytes(*a))) != RHZ_OK)
        return s;
    return hip_status(rhz::launch_norm_backward(*a, layer, static_cast<hipStream_t>(stream)), "norm backward launch");
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
    if ((s = check_workspace(a->workspace, a->workspace_bytes, rhz::backward_workspace_bytes(*a))) != RHZ_OK) return s;
    return hip_status(rhz::launch_backward(*a, static_cast<hipStream_t>(stream)), "prefill backward launch");
}

rhz_status rhz_gdr_conv_prepare_backward_workspace_size(const rhz_gdr_conv_prepare_backward_args* a, size_t* bytes) {
    if (!bytes) return fail(RHZ_ERR_INVALID_ARG, "bytes is NULL");
    const rhz_status s = check_conv_backward(a);
    if (s != RHZ_OK) return s;
    *bytes = rhz::conv_prepare_backward_workspace_bytes(*a);
    return ok();
}

rhz_status rhz_gdr_conv_prepare_backward(const rhz_gdr_conv_prepare_backward_args* a, void* stream) {
    rhz_status s = check_conv_backward(a);
    if (s != RHZ_OK) return s;
    const size_t tokens = a->cu_seqlens ? (size_t)a->seq_len : (size_t)a->batch * a->seq_len;
    const size_t es = a->dtype == RHZ_F32 ? 4 : 2, rows = tokens * a->heads;
    const size_t C = (size_t)a->heads * (2 * a->d_k + a->d_v), ns = (size_t)a->batch * C * 12;
    const bool any = tokens > 0;
    const Buffer b[] = {
        {"x", a->x, tokens * C * es, 16, any, false},
        {"weight", a->weight, C * 16, 4, true, false},
        {"bias", a->bias, C * 4, 4, false, false},
        {"cu_seqlens", a->cu_seqlens, ((size_t)a->batch + 1) * 4, 4, false, false},
        {"initial_state", a->initial_state, ns, 4, false, false},
        {"beta_logit", a->beta_logit, rows * 4, 4, any, false},
        {"alpha_logit", a->alpha_logit, rows * 4, 4, any, false},
        {"a_log", a->a_log, (size_t)a->heads * 4, 4, any, false},
        {"grad_q", a->grad_q, rows * a->d_k * es, 16, any, false},
        {"grad_k", a->grad_k, rows * a->d_k * es, 16, any, false},
        {"grad_v", a->grad_v, rows * a->d_v * es, 16, any, false},
        {"grad_beta", a->grad_beta, rows * es, es, any, false},
        {"grad_g", a->grad_g, rows * es, es, any, false},
        {"grad_final_state", a->grad_final_state, ns, 4, false, false},
        {"grad_x", a->grad_x, tokens * C * es, 16, any, true},
        {"grad_weight", a->grad_weight, C * 16, 4, true, true},
        {"grad_bias", a->grad_bias, C * 4, 4, false, true},
        {"grad_beta_logit", a->grad_beta_logit, rows * 4, 4, any, true},
        {"grad_alpha_logit", a->grad_alpha_logit, rows * 4, 4, any, true},
        {"grad_a_log", a->grad_a_log, (size_t)a->heads * 4, 4, true, true},
        {"grad_initial_state", a->grad_initial_state, ns, 4, false, true},
        {"workspace", a->workspace, a->workspace_bytes, 1, false, true},
    };
    if ((s = check_buffers(b, sizeof b / sizeof b[0])) != RHZ_OK) return s;
    if ((s = check_workspace(a->workspace, a->workspace_bytes, rhz::conv_prepare_backward_workspace_bytes(*a))) != RHZ_OK)
        return s;
    return hip_status(rhz::launch_conv_prepare_backward(*a, static_cast<hipStream_t>(stream)),
                      "conv prepare backward launch");
}

rhz_status rhz_layernorm(const rhz_layernorm_args* a, void* stream) {
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    rhz_status s = check_norm(a->rows, a->dim, a->dtype, a->eps);
    if (s != RHZ_OK) return s;
    if (a->rows == 0) return ok();
    const size_t es = a->dtype == RHZ_F32 ? 4 : 2, n = (size_t)a->rows * a->dim * es, nd = (size_t)a->dim * 4;
    const Buffer b[] = {
        {"y", a->y, n, es, true, true},
        {"weight", a->weight, nd, 4, true, false},
        {"bias", a->bias, nd, 4, false, false},
        {"x", a->x, n, es, true, false},  // last: y may be x itself
    };
    if ((s = check_buffers(b, a->x == a->y && a->x ? 3 : 4)) != RHZ_OK) return s;
    return hip_status(rhz::launch_layernorm(*a, static_cast<hipStream_t>(stream)), "layernorm launch");
}

rhz_status rhz_norm_backward_workspace_size(const rhz_norm_backward_args* a, size_t* bytes) {
    if (!bytes) return fail(RHZ_ERR_INVALID_ARG, "bytes is NULL");
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    const rhz_status s = check_norm(a->rows, a->dim, a->dtype, a->eps);
    if (s != RHZ_OK) return s;
    *bytes = rhz::norm_backward_workspace_bytes(*a);
    return ok();
}

rhz_status rhz_layernorm_backward(const rhz_norm_backward_args* a, void* stream) {
    return norm_backward(a, true, stream);
}

rhz_status rhz_rmsnorm_heads_backward(const rhz_norm_backward_args* a, void* stream) {
    return norm_backward(a, false, stream);
}

}  // extern "C"
