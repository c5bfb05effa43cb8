// attn_abi.cpp -- the extern "C" boundary of the latent attention
// (rhizome_attention.h): argument validation, complete before any HIP call,
// and dispatch to the kernel launchers.

#include <cmath>
#include <cstdint>

#include "abi_checks.hpp"
#include "gdr_internal.hpp"
#include "rhizome_attention.h"

using namespace rhz::abi;

namespace {

// Tiles address 128 rows by 32-bit byte offsets.
constexpr int64_t kMaxTokenStride = 1 << 22;

size_t value_bytes(int dtype) { return dtype == RHZ_F32 ? 4 : 2; }

rhz_status check_dtype(int dtype) {
    if (dtype == RHZ_F32 || dtype == RHZ_BF16) return ok();
    return fail(RHZ_ERR_INVALID_ARG, "dtype must be RHZ_F32 or RHZ_BF16 (got %d)", dtype);
}

rhz_status check_flag(const char* name, int v) {
    if (v == 0 || v == 1) return ok();
    return fail(RHZ_ERR_INVALID_ARG, "%s must be 0 or 1 (got %d)", name, v);
}

// Elements from the first to the last of [n, heads, dim] with these strides, or
// -1 beyond what 63 bits hold in bytes.
int64_t extent(int64_t n, int64_t stride, int64_t heads, int64_t head_stride, int64_t dim) {
    if (n == 0) return 0;
    const int64_t most = INT64_MAX / 32;
    if (rhz::exceeds(stride, n, most) || rhz::exceeds(head_stride, heads, most)) return -1;
    return (n - 1) * stride + (heads - 1) * head_stride + dim;
}

// No two rows of `dim` values share an element.
bool disjoint(int64_t n, int64_t stride, int64_t heads, int64_t head_stride, int64_t dim) {
    const bool by_token = (heads <= 1 || head_stride >= dim) && (n <= 1 || stride >= extent(1, 0, heads, head_stride, dim));
    const bool by_head = (n <= 1 || stride >= dim) && (heads <= 1 || head_stride >= extent(n, stride, 1, 0, dim));
    return by_token || by_head;
}

rhz_status check_rope(const rhz_rope_args* a) {
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    if (a->tokens < 0) return fail(RHZ_ERR_INVALID_ARG, "tokens must be >= 0 (got %d)", a->tokens);
    if (a->heads < 1) return fail(RHZ_ERR_INVALID_ARG, "heads must be >= 1 (got %d)", a->heads);
    if (a->rot < 2 || a->rot % 2) return fail(RHZ_ERR_INVALID_ARG, "rot must be even and >= 2 (got %d)", a->rot);
    if (a->rot > 1024) return fail(RHZ_ERR_UNSUPPORTED, "rot = %d exceeds the supported 1024", a->rot);
    if (a->offset < 0 || a->dim < 1 || a->offset > a->dim || a->rot > a->dim - a->offset)
        return fail(RHZ_ERR_INVALID_ARG, "channels [%d, %d + %d) are not in [0, %d)", a->offset, a->offset, a->rot, a->dim);
    if ((int64_t)a->heads * a->dim > INT32_MAX / 4096)
        return fail(RHZ_ERR_UNSUPPORTED, "heads * dim = %lld exceeds 2^19 - 1", (long long)a->heads * a->dim);
    rhz_status s = check_dtype(a->dtype);
    if (s == RHZ_OK) s = check_flag("interleaved", a->interleaved);
    if (s == RHZ_OK) s = check_flag("inverse", a->inverse);
    if (s != RHZ_OK) return s;
    if (!std::isfinite(a->magnitude)) return fail(RHZ_ERR_INVALID_ARG, "magnitude must be finite");
    if (a->x_token_stride < 0 || a->x_head_stride < 0 || a->y_token_stride < 0 || a->y_head_stride < 0)
        return fail(RHZ_ERR_INVALID_ARG, "strides must be >= 0");
    return ok();
}

rhz_status check_paged(int batch, int page_size, int num_pages, int max_pages) {
    if (batch < 1) return fail(RHZ_ERR_INVALID_ARG, "batch must be >= 1 (got %d)", batch);
    if (page_size < 1 || num_pages < 1 || max_pages < 1)
        return fail(RHZ_ERR_INVALID_ARG, "page_size, num_pages and max_pages must be >= 1 (got %d, %d, %d)", page_size,
                    num_pages, max_pages);
    if ((int64_t)page_size * num_pages > INT32_MAX)
        return fail(RHZ_ERR_INVALID_ARG, "page_size * num_pages = %lld exceeds 2^31 - 1", (long long)page_size * num_pages);
    return ok();
}

rhz_status check_append(const rhz_latent_append_args* a) {
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    rhz_status s = check_paged(a->batch, a->page_size, a->num_pages, a->max_pages);
    if (s == RHZ_OK) s = check_dtype(a->dtype);
    if (s == RHZ_OK) s = check_flag("interleaved", a->interleaved);
    if (s != RHZ_OK) return s;
    if (a->seq_len < 0) return fail(RHZ_ERR_INVALID_ARG, "seq_len must be >= 0 (got %d)", a->seq_len);
    if (a->d_c < 1 || a->d_r < 0) return fail(RHZ_ERR_INVALID_ARG, "d_c must be >= 1 and d_r >= 0 (got %d, %d)", a->d_c, a->d_r);
    if (a->d_c > 4096 || a->d_r > 1024)
        return fail(RHZ_ERR_UNSUPPORTED, "d_c = %d, d_r = %d exceed the supported 4096 and 1024", a->d_c, a->d_r);
    if (a->turns && a->d_r % 2) return fail(RHZ_ERR_INVALID_ARG, "d_r must be even to be turned (got %d)", a->d_r);
    if (!std::isfinite(a->magnitude)) return fail(RHZ_ERR_INVALID_ARG, "magnitude must be finite");
    if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return fail(RHZ_ERR_INVALID_ARG, "eps must be >= 0 and finite");
    const int64_t tokens = a->cu_seqlens ? (int64_t)a->seq_len : (int64_t)a->batch * a->seq_len;
    if (tokens > INT32_MAX) return fail(RHZ_ERR_INVALID_ARG, "%lld new tokens: at most 2^31 - 1", (long long)tokens);
    if (a->latent_stride < 0 || a->k_rope_stride < 0) return fail(RHZ_ERR_INVALID_ARG, "strides must be >= 0");
    if (extent(tokens, a->latent_stride, 1, 0, a->d_c) < 0 || extent(tokens, a->k_rope_stride, 1, 0, a->d_r) < 0)
        return fail(RHZ_ERR_INVALID_ARG, "strides are too large");
    return ok();
}

rhz_status check_decode(const rhz_latent_decode_args* a) {
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    rhz_status s = check_paged(a->batch, a->page_size, a->num_pages, a->max_pages);
    if (s == RHZ_OK) s = check_dtype(a->dtype);
    if (s != RHZ_OK) return s;
    if (a->steps < 1 || a->heads < 1)
        return fail(RHZ_ERR_INVALID_ARG, "steps and heads must be >= 1 (got %d, %d)", a->steps, a->heads);
    if (a->d_c < 1 || a->d_r < 0) return fail(RHZ_ERR_INVALID_ARG, "d_c must be >= 1 and d_r >= 0 (got %d, %d)", a->d_c, a->d_r);
    if (a->steps > RHZ_MULTISTEP_MAX || a->heads > 1024)
        return fail(RHZ_ERR_UNSUPPORTED, "steps = %d, heads = %d exceed the supported %d and 1024", a->steps, a->heads,
                    RHZ_MULTISTEP_MAX);
    if (a->d_c > 512 || a->d_r > 64)
        return fail(RHZ_ERR_UNSUPPORTED, "d_c = %d, d_r = %d exceed the supported 512 and 64", a->d_c, a->d_r);
    if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return fail(RHZ_ERR_INVALID_ARG, "scale must be > 0 and finite");
    if ((int64_t)a->batch * a->steps * a->heads > INT32_MAX)
        return fail(RHZ_ERR_INVALID_ARG, "batch * steps * heads exceeds 2^31 - 1");
    return ok();
}

rhz_status check_prefill(const rhz_latent_prefill_args* a) {
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    if (a->batch < 1) return fail(RHZ_ERR_INVALID_ARG, "batch must be >= 1 (got %d)", a->batch);
    if (a->seq_len < 0 || a->seq_len_k < 0)
        return fail(RHZ_ERR_INVALID_ARG, "seq_len and seq_len_k must be >= 0 (got %d, %d)", a->seq_len, a->seq_len_k);
    if (a->heads < 1) return fail(RHZ_ERR_INVALID_ARG, "heads must be >= 1 (got %d)", a->heads);
    if (a->d_n < 1 || a->d_r < 0 || a->d_v < 1)
        return fail(RHZ_ERR_INVALID_ARG, "d_n and d_v must be >= 1 and d_r >= 0 (got %d, %d, %d)", a->d_n, a->d_v, a->d_r);
    rhz_status s = check_dtype(a->dtype);
    if (s == RHZ_OK) s = check_flag("causal", a->causal);
    if (s != RHZ_OK) return s;
    if (a->d_n > 192 || a->d_r > 192 || a->d_n + a->d_r > 192 || a->d_v > 128)
        return fail(RHZ_ERR_UNSUPPORTED, "d_n + d_r = %lld, d_v = %d exceed the supported 192 and 128",
                    (long long)a->d_n + a->d_r, a->d_v);
    if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return fail(RHZ_ERR_INVALID_ARG, "scale must be > 0 and finite");
    if (a->cu_seqlens_k && !a->cu_seqlens) return fail(RHZ_ERR_INVALID_ARG, "cu_seqlens_k without cu_seqlens");
    if (a->cu_seqlens && !a->cu_seqlens_k && a->seq_len != a->seq_len_k)
        return fail(RHZ_ERR_INVALID_ARG, "seq_len = %d and seq_len_k = %d differ without cu_seqlens_k", a->seq_len, a->seq_len_k);
    const int64_t queries = a->cu_seqlens ? (int64_t)a->seq_len : (int64_t)a->batch * a->seq_len;
    const int64_t keys = a->cu_seqlens ? (int64_t)a->seq_len_k : (int64_t)a->batch * a->seq_len_k;
    // room for tile numbers and ends beyond the last row
    if (queries > INT32_MAX - 256 || keys > INT32_MAX - 256)
        return fail(RHZ_ERR_INVALID_ARG, "%lld queries, %lld keys: at most 2^31 - 257", (long long)queries, (long long)keys);
    const int64_t strides[] = {a->q_token_stride, a->q_head_stride, a->k_token_stride, a->k_head_stride,
                               a->v_token_stride, a->v_head_stride, a->k_rope_stride};
    for (const int64_t x : strides)
        if (x < 0) return fail(RHZ_ERR_INVALID_ARG, "strides must be >= 0");
    if (a->q_token_stride > kMaxTokenStride || a->k_token_stride > kMaxTokenStride || a->v_token_stride > kMaxTokenStride ||
        a->k_rope_stride > kMaxTokenStride || (int64_t)a->heads * a->d_v > kMaxTokenStride)
        return fail(RHZ_ERR_UNSUPPORTED, "tokens are more than %lld elements apart", (long long)kMaxTokenStride);
    if (extent(queries, a->q_token_stride, a->heads, a->q_head_stride, a->d_n + a->d_r) < 0 ||
        extent(keys, a->k_token_stride, a->heads, a->k_head_stride, a->d_n) < 0 ||
        extent(keys, a->v_token_stride, a->heads, a->v_head_stride, a->d_v) < 0)
        return fail(RHZ_ERR_INVALID_ARG, "strides are too large");
    return ok();
}

struct PrefillSizes {
    size_t queries, keys, es, q, k, v, r, o, lse, cu;
};

PrefillSizes prefill_sizes(const rhz_latent_prefill_args& a) {
    PrefillSizes n;
    n.queries = a.cu_seqlens ? (size_t)a.seq_len : (size_t)a.batch * a.seq_len;
    n.keys = a.cu_seqlens ? (size_t)a.seq_len_k : (size_t)a.batch * a.seq_len_k;
    n.es = value_bytes(a.dtype);
    n.q = extent(n.queries, a.q_token_stride, a.heads, a.q_head_stride, a.d_n + a.d_r) * n.es;
    n.k = extent(n.keys, a.k_token_stride, a.heads, a.k_head_stride, a.d_n) * n.es;
    n.v = extent(n.keys, a.v_token_stride, a.heads, a.v_head_stride, a.d_v) * n.es;
    n.r = extent(n.keys, a.k_rope_stride, 1, 0, a.d_r) * n.es;
    n.o = n.queries * a.heads * a.d_v * n.es;
    n.lse = n.queries * a.heads * 4;
    n.cu = ((size_t)a.batch + 1) * 4;
    return n;
}

}  // namespace

extern "C" {

rhz_status rhz_rope_frequencies(const rhz_rope_frequency_args* a, double* turns, float* magnitude) {
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    if (!turns) return fail(RHZ_ERR_INVALID_ARG, "turns is NULL");
    if (!magnitude) return fail(RHZ_ERR_INVALID_ARG, "magnitude is NULL");
    if (a->dim < 2 || a->dim % 2) return fail(RHZ_ERR_INVALID_ARG, "dim must be even and >= 2 (got %d)", a->dim);
    if (a->dim > 1024) return fail(RHZ_ERR_UNSUPPORTED, "dim = %d exceeds the supported 1024", a->dim);
    if (a->scaling < RHZ_ROPE_PLAIN || a->scaling > RHZ_ROPE_BY_PARTS)
        return fail(RHZ_ERR_INVALID_ARG, "scaling is no rhz_rope_scaling (got %d)", a->scaling);
    if (!(a->theta > 1.0) || !std::isfinite(a->theta)) return fail(RHZ_ERR_INVALID_ARG, "theta must be > 1 and finite");
    if (a->scaling != RHZ_ROPE_PLAIN && (!(a->factor >= 1.0) || !std::isfinite(a->factor)))
        return fail(RHZ_ERR_INVALID_ARG, "factor must be >= 1 and finite");
    if (a->scaling == RHZ_ROPE_BY_PARTS) {
        if (!(a->trained_length >= 1.0) || !std::isfinite(a->trained_length))
            return fail(RHZ_ERR_INVALID_ARG, "trained_length must be >= 1 and finite");
        if (!(a->slow >= 0.0) || !(a->fast > a->slow) || !std::isfinite(a->fast))
            return fail(RHZ_ERR_INVALID_ARG, "need fast > slow >= 0, finite");
    }
    const double two_pi = 6.283185307179586476925;
    *magnitude = a->scaling == RHZ_ROPE_BY_PARTS ? float(0.1 * std::log(a->factor) + 1.0) : 1.f;
    for (int i = 0; i < a->dim / 2; ++i) {
        double f = std::pow(a->theta, -2.0 * i / a->dim) / two_pi;
        if (a->scaling == RHZ_ROPE_LINEAR) {
            f /= a->factor;
        } else if (a->scaling == RHZ_ROPE_BY_PARTS) {
            // the share that keeps its frequency, by the pair's turns over the trained length
            const double x = (a->trained_length * f - a->slow) / (a->fast - a->slow);
            const double keep = x < 0.0 ? 0.0 : x > 1.0 ? 1.0 : x;
            f *= keep + (1.0 - keep) / a->factor;
        }
        turns[i] = f;
    }
    return ok();
}

rhz_status rhz_rope(const rhz_rope_args* a, void* stream) {
    rhz_status s = check_rope(a);
    if (s != RHZ_OK) return s;
    if (a->tokens == 0) return ok();
    const int64_t nx = extent(a->tokens, a->x_token_stride, a->heads, a->x_head_stride, a->dim);
    const int64_t ny = extent(a->tokens, a->y_token_stride, a->heads, a->y_head_stride, a->dim);
    if (nx < 0 || ny < 0) return fail(RHZ_ERR_INVALID_ARG, "strides are too large");
    if (!disjoint(a->tokens, a->y_token_stride, a->heads, a->y_head_stride, a->dim))
        return fail(RHZ_ERR_INVALID_ARG, "y's rows overlap each other");
    const bool in_place = a->x == a->y && a->x;
    if (in_place && (a->x_token_stride != a->y_token_stride || a->x_head_stride != a->y_head_stride))
        return fail(RHZ_ERR_INVALID_ARG, "in place, x and y need the same strides");
    const size_t es = value_bytes(a->dtype);
    const Buffer b[] = {
        {"y", a->y, (size_t)ny * es, es, true, true},
        {"positions", a->positions, (size_t)a->tokens * 4, 4, true, false},
        {"turns", a->turns, (size_t)a->rot / 2 * 8, 8, true, false},
        {"x", a->x, (size_t)nx * es, es, true, false},  // last: y may be x itself
    };
    if ((s = check_buffers(b, in_place ? 3 : 4)) != RHZ_OK) return s;
    return hip_status(rhz::launch_rope(*a, static_cast<hipStream_t>(stream)), "rope launch");
}

rhz_status rhz_latent_append(const rhz_latent_append_args* a, void* stream) {
    rhz_status s = check_append(a);
    if (s != RHZ_OK) return s;
    const size_t tokens = a->cu_seqlens ? (size_t)a->seq_len : (size_t)a->batch * a->seq_len;
    if (tokens == 0) return ok();
    const size_t es = value_bytes(a->dtype);
    const Buffer b[] = {
        {"latent", a->latent, (size_t)extent(tokens, a->latent_stride, 1, 0, a->d_c) * es, es, true, false},
        {"k_rope", a->d_r ? a->k_rope : nullptr, (size_t)extent(tokens, a->k_rope_stride, 1, 0, a->d_r) * es, es, a->d_r > 0,
         false},
        {"cu_seqlens", a->cu_seqlens, ((size_t)a->batch + 1) * 4, 4, false, false},
        {"lengths", a->lengths, (size_t)a->batch * 4, 4, true, false},
        {"page_table", a->page_table, (size_t)a->batch * a->max_pages * 4, 4, true, false},
        {"turns", a->turns, (size_t)a->d_r / 2 * 8, 8, false, false},
        {"norm_scale", a->norm_scale, (size_t)a->d_c * 4, 4, false, false},
        {"cache", a->cache, (size_t)a->num_pages * a->page_size * (a->d_c + a->d_r) * es, es, true, true},
    };
    if ((s = check_buffers(b, sizeof b / sizeof b[0])) != RHZ_OK) return s;
    return hip_status(rhz::launch_latent_append(*a, static_cast<hipStream_t>(stream)), "latent append launch");
}

rhz_status rhz_latent_decode_workspace_size(const rhz_latent_decode_args* a, size_t* bytes) {
    if (!bytes) return fail(RHZ_ERR_INVALID_ARG, "bytes is NULL");
    const rhz_status s = check_decode(a);
    if (s != RHZ_OK) return s;
    *bytes = rhz::latent_decode_workspace_bytes(*a);
    return ok();
}

rhz_status rhz_latent_decode(const rhz_latent_decode_args* a, void* stream) {
    rhz_status s = check_decode(a);
    if (s != RHZ_OK) return s;
    const size_t es = value_bytes(a->dtype), rows = (size_t)a->batch * a->steps * a->heads, D = (size_t)a->d_c + a->d_r;
    const Buffer b[] = {
        {"q", a->q, rows * D * es, es, true, false},
        {"cache", a->cache, (size_t)a->num_pages * a->page_size * D * es, es, true, false},
        {"page_table", a->page_table, (size_t)a->batch * a->max_pages * 4, 4, true, false},
        {"lengths", a->lengths, (size_t)a->batch * 4, 4, true, false},
        {"o", a->o, rows * a->d_c * es, es, true, true},
        {"lse", a->lse, rows * 4, 4, false, true},
        {"workspace", a->workspace, a->workspace_bytes, 1, false, true},
    };
    if ((s = check_buffers(b, sizeof b / sizeof b[0])) != RHZ_OK) return s;
    if ((s = check_workspace(a->workspace, a->workspace_bytes, rhz::latent_decode_workspace_bytes(*a))) != RHZ_OK) return s;
    return hip_status(rhz::launch_latent_decode(*a, static_cast<hipStream_t>(stream)), "latent decode launch");
}

rhz_status rhz_latent_prefill(const rhz_latent_prefill_args* a, void* stream) {
    rhz_status s = check_prefill(a);
    if (s != RHZ_OK) return s;
    const PrefillSizes n = prefill_sizes(*a);
    if (n.queries == 0) return ok();
    const bool keys = n.keys > 0;
    const Buffer b[] = {
        {"q", a->q, n.q, n.es, true, false},
        {"k", a->k, n.k, n.es, keys, false},
        {"v", a->v, n.v, n.es, keys, false},
        {"k_rope", a->d_r ? a->k_rope : nullptr, n.r, n.es, keys && a->d_r > 0, false},
        {"cu_seqlens", a->cu_seqlens, n.cu, 4, false, false},
        {"cu_seqlens_k", a->cu_seqlens_k, n.cu, 4, false, false},
        {"o", a->o, n.o, n.es, true, true},
        {"lse", a->lse, n.lse, 4, true, true},
    };
    if ((s = check_buffers(b, sizeof b / sizeof b[0])) != RHZ_OK) return s;
    return hip_status(rhz::launch_latent_prefill(*a, static_cast<hipStream_t>(stream)), "latent prefill launch");
}

rhz_status rhz_latent_prefill_backward_workspace_size(const rhz_latent_prefill_backward_args* a, size_t* bytes) {
    if (!bytes) return fail(RHZ_ERR_INVALID_ARG, "bytes is NULL");
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    const rhz_status s = check_prefill(&a->forward);
    if (s != RHZ_OK) return s;
    *bytes = rhz::latent_prefill_backward_workspace_bytes(*a);
    return ok();
}

rhz_status rhz_latent_prefill_backward(const rhz_latent_prefill_backward_args* a, void* stream) {
    if (!a) return fail(RHZ_ERR_INVALID_ARG, "args is NULL");
    const rhz_latent_prefill_args& f = a->forward;
    rhz_status s = check_prefill(&f);
    if (s != RHZ_OK) return s;
    const PrefillSizes n = prefill_sizes(f);
    if (n.queries == 0 && n.keys == 0) return ok();
    const bool queries = n.queries > 0, keys = n.keys > 0, rope = keys && f.d_r > 0;
    const size_t rows_q = n.queries * f.heads, rows_k = n.keys * f.heads;
    const Buffer b[] = {
        {"q", f.q, n.q, n.es, queries, false},
        {"k", f.k, n.k, n.es, keys, false},
        {"v", f.v, n.v, n.es, keys, false},
        {"k_rope", f.d_r ? f.k_rope : nullptr, n.r, n.es, rope, false},
        {"cu_seqlens", f.cu_seqlens, n.cu, 4, false, false},
        {"cu_seqlens_k", f.cu_seqlens_k, n.cu, 4, false, false},
        {"o", f.o, n.o, n.es, queries, false},
        {"lse", f.lse, n.lse, 4, queries, false},
        {"grad_o", a->grad_o, n.o, n.es, queries, false},
        {"grad_lse", a->grad_lse, n.lse, 4, false, false},
        {"grad_q", a->grad_q, rows_q * (f.d_n + f.d_r) * n.es, n.es, queries, true},
        {"grad_k", a->grad_k, rows_k * f.d_n * n.es, n.es, keys, true},
        {"grad_v", a->grad_v, rows_k * f.d_v * n.es, n.es, keys, true},
        {"grad_k_rope", f.d_r ? a->grad_k_rope : nullptr, n.keys * f.d_r * n.es, n.es, rope, true},
        {"workspace", a->workspace, a->workspace_bytes, 1, false, true},
    };
    if ((s = check_buffers(b, sizeof b / sizeof b[0])) != RHZ_OK) return s;
    if ((s = check_workspace(a->workspace, a->workspace_bytes, rhz::latent_prefill_backward_workspace_bytes(*a))) != RHZ_OK)
        return s;
    return hip_status(rhz::launch_latent_prefill_backward(*a, static_cast<hipStream_t>(stream)),
                      "latent prefill backward launch");
}

}  // extern "C"
