// latent_cache.hip -- rotary positions, and new tokens into the paged cache of
// latents.  Both move bytes: what is counted is that every value is read and
// written once, 16 bytes at a time, and that an angle is formed once for all
// heads.
#include <algorithm>

#include "gdr_internal.hpp"
#include "gdr_rows.hpp"

namespace rhz {
namespace {

// (cos, sin) of `turns` turns times a position, times the magnitude.  The
// product is reduced to half a turn in 64 bits: at a position of 2^31 its rounding
// is 2^-25 of a turn at most, at a million 2^-36, before fp32 takes the rest.
__device__ __forceinline__ float2 rotation(double turns, int position, float magnitude) {
    const double t = turns * position;
    float s, c;
    sincospif(2.f * float(t - rint(t)), &s, &c);
    return make_float2(c * magnitude, s * magnitude);
}

struct RopeParams {
    const void* x;
    const int* positions;
    const double* turns;
    void* y;
    long xt, xh, yt, yh;
    int tokens, heads, dim, offset, rot, copy, per_block;  // tokens of a workgroup
    float magnitude, sign;
};

constexpr int kThreads = 256, kTokenPairs = 2048;

// A workgroup forms the angles of its tokens in LDS, then goes over their heads:
// 8192 tokens, 32 heads of 192 channels, 64 of them turned, 37 us for 201 MB, 5.4
// TB/s (the card's copies reach 4.7; part of x stays in its caches).  Values one by
// one where they are not aligned to 16 bytes: 94 us.
// An item is what one thread does at once: E pairs of channels of a head (half
// layout: chunks of both halves; interleaved: a chunk is E / 2 pairs) or one
// chunk that is copied.
template <typename T, bool VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeParams a) {
    using V = Vec<T, VEC>;
    constexpr int E = V::N;
    __shared__ float2 angle[kTokenPairs];
    const int tid = threadIdx.x, half = a.rot / 2;
    const long t0 = (long)blockIdx.x * a.per_block;
    const int n = (int)min((long)a.per_block, a.tokens - t0);
    for (int i = tid; i < n * half; i += kThreads) {
        const int t = i / half;
        float2 v = rotation(a.turns[i - t * half], a.positions[t0 + t], a.magnitude);
        v.y *= a.sign;
        angle[i] = v;
    }
    __syncthreads();
    const unsigned turned = INTER && VEC ? a.rot / E : half / E;
    const unsigned copied = a.copy ? (a.dim - a.rot) / E : 0;
    const unsigned per_head = turned + copied, total = n * a.heads * per_head;
    for (unsigned i = tid; i < total; i += kThreads) {
        const unsigned row = i / per_head, k = i - row * per_head, t = row / a.heads, h = row - t * a.heads;
        const T* x = (const T*)a.x + (t0 + t) * a.xt + h * a.xh;
        T* y = (T*)a.y + (t0 + t) * a.yt + h * a.yh;
        if (k >= turned) {
            int d = (k - turned) * E;
            if (d >= a.offset) d += a.rot;
            float v[E];
            V::load(x + d, v);
            V::store(y + d, v);
            continue;
        }
        const float2* cs = angle + t * half;
        if constexpr (INTER && VEC) {
            const int d = a.offset + k * E;
            float v[E];
            V::load(x + d, v);
#pragma unroll
            for (int j = 0; j < E; j += 2) {
                const float2 r = cs[(k * E + j) / 2];
                const float p = v[j], q = v[j + 1];
                v[j] = p * r.x - q * r.y;
                v[j + 1] = p * r.y + q * r.x;
            }
            V::store(y + d, v);
        } else {
            const int d = a.offset + (INTER ? 2 * k : k * E), e = INTER ? d + 1 : d + half;
            float p[E], q[E];
            V::load(x + d, p);
            V::load(x + e, q);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const float2 r = cs[k * E + j];
                const float u = p[j] * r.x - q[j] * r.y;
                q[j] = p[j] * r.y + q[j] * r.x;
                p[j] = u;
            }
            V::store(y + d, p);
            V::store(y + e, q);
        }
    }
}

template <typename T>
hipError_t rope(const RopeParams& p, bool vec, bool inter, hipStream_t stream) {
    const int64_t blocks = ((int64_t)p.tokens + p.per_block - 1) / p.per_block;
    if (check_grid(blocks, kThreads) != hipSuccess) return hipErrorInvalidConfiguration;
    const unsigned n = (unsigned)blocks;
    if (vec && inter)
        rope_kernel<T, true, true><<<n, kThreads, 0, stream>>>(p);
    else if (vec)
        rope_kernel<T, true, false><<<n, kThreads, 0, stream>>>(p);
    else if (inter)
        rope_kernel<T, false, true><<<n, kThreads, 0, stream>>>(p);
    else
        rope_kernel<T, false, false><<<n, kThreads, 0, stream>>>(p);
    return hipGetLastError();
}

// ------------------------------------------------------------------- append
struct AppendParams {
    const void *latent, *key;
    const int *cu, *lengths, *table;
    const double* turns;
    const float* norm;
    void* cache;
    long ls, ks, tokens;
    int batch, len, d_c, d_r, page, num_pages, max_pages, inter;
    float magnitude, eps;
};

// Chunks of a lane that stay in registers: 1024 bf16 or 512 fp32 latents (128 of
// either where a chunk is one value), those behind are read twice.  With eight, for
// 4096, the registers leave room for fewer waves: 10333 tokens of 512 + 64, 11.0 us
// instead of 10.1.
constexpr int kMaxChunks = 2;

// A wave a token: the latent is read once and kept in registers while its norm is
// formed.  10333 tokens of 512 + 64, 24 MB: 10.1 us, values one by one 13.4; one
// token each of 8 sequences 4.4.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void latent_append_kernel(AppendParams a) {
    using V = Vec<T, VEC>;
    constexpr int E = V::N;
    const int lane = threadIdx.x & 63;
    const long t = (long)blockIdx.x * (kThreads / kWave) + (threadIdx.x >> 6);
    if (t >= a.tokens) return;
    // The token's values are on their way while its place is looked up.
    const T* x = (const T*)a.latent + t * a.ls;
    const int chunks = a.d_c / E;
    typename V::Raw keep[kMaxChunks];
#pragma unroll
    for (int k = 0; k < kMaxChunks; ++k) {
        const int i = k * kWave + lane;
        if (i < chunks) keep[k] = V::load_raw(x + i * E);
    }
    const T* r = (const T*)a.key + t * a.ks;
    const int half = a.d_r / 2;
    const auto pair = [&](int i) { return a.inter ? 2 * i : i; };
    const auto partner = [&](int i) { return a.inter ? 2 * i + 1 : i + half; };
    float p0 = 0.f, q0 = 0.f;
    double f0 = 0.0;
    if (a.turns && lane < half) p0 = Elem<T>::load(r, pair(lane)), q0 = Elem<T>::load(r, partner(lane)), f0 = a.turns[lane];
    int seq, left;  // tokens of the sequence from this one on
    if (a.cu) {
        seq = 0;  // sequences that end at or before t
        for (int b0 = 0; b0 < a.batch; b0 += kWave) {
            const int b = b0 + lane;
            const int n = __popcll(__ballot(b < a.batch && a.cu[min(b, a.batch - 1) + 1] <= t));
            seq += n;
            if (n < kWave) break;
        }
        if (seq >= a.batch) return;
        int t0, t1;
        seq_bounds(a.cu, seq, a.len, t0, t1);
        if (t < t0 || t >= t1) return;
        left = t1 - (int)t;
    } else {
        seq = int(t / a.len);
        left = a.len - int(t % a.len);
    }
    const long pos = (long)a.lengths[seq] - left;
    if (pos < 0 || pos / a.page >= a.max_pages) return;
    const int page = a.table[(long)seq * a.max_pages + pos / a.page];
    if (page < 0 || page >= a.num_pages) return;
    T* out = (T*)a.cache + ((long)page * a.page + pos % a.page) * (a.d_c + a.d_r);
    float sum = 0.f, f = 1.f;
    if (a.norm) {
#pragma unroll
        for (int k = 0; k < kMaxChunks; ++k) {
            if (k * kWave + lane >= chunks) continue;
            float v[E];
            V::unpack(keep[k], v);
#pragma unroll
            for (int j = 0; j < E; ++j) sum = fmaf(v[j], v[j], sum);
        }
        for (int i = kMaxChunks * kWave + lane; i < chunks; i += kWave) {
            float v[E];
            V::load(x + i * E, v);
#pragma unroll
            for (int j = 0; j < E; ++j) sum = fmaf(v[j], v[j], sum);
        }
        f = 1.f / sqrtf(row_sum<64>(sum) / a.d_c + a.eps);
    }
    const auto put = [&](int i, float (&v)[E]) {
        if (a.norm)
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] *= f * a.norm[i * E + j];
        V::store(out + i * E, v);
    };
#pragma unroll
    for (int k = 0; k < kMaxChunks; ++k) {
        const int i = k * kWave + lane;
        if (i >= chunks) continue;
        float v[E];
        V::unpack(keep[k], v);
        put(i, v);
    }
    for (int i = kMaxChunks * kWave + lane; i < chunks; i += kWave) {
        float v[E];
        V::load(x + i * E, v);
        put(i, v);
    }
    out += a.d_c;
    if (!a.turns) {
        for (int d = lane; d < a.d_r; d += kWave) out[d] = r[d];
        return;
    }
    for (int i = lane; i < half; i += kWave) {
        if (i != lane) p0 = Elem<T>::load(r, pair(i)), q0 = Elem<T>::load(r, partner(i)), f0 = a.turns[i];
        const float2 cs = rotation(f0, (int)pos, a.magnitude);
        Elem<T>::store(out, pair(i), p0 * cs.x - q0 * cs.y);
        Elem<T>::store(out, partner(i), p0 * cs.y + q0 * cs.x);
    }
}

}  // namespace

hipError_t launch_rope(const rhz_rope_args& a, hipStream_t stream) {
    if (a.tokens == 0) return hipSuccess;
    const int e = a.dtype == RHZ_F32 ? 4 : 8;
    const bool vec = (a.interleaved ? a.rot % e == 0 : a.rot / 2 % e == 0) && a.offset % e == 0 && a.dim % e == 0 &&
                     a.x_token_stride % e == 0 && a.x_head_stride % e == 0 && a.y_token_stride % e == 0 &&
                     a.y_head_stride % e == 0 && aligned16(a.x) && aligned16(a.y);
    RopeParams p = {a.x, a.positions, a.turns, a.y, a.x_token_stride, a.x_head_stride, a.y_token_stride, a.y_head_stride,
                    a.tokens, a.heads, a.dim, a.offset, a.rot, a.x != a.y, 1, a.magnitude, a.inverse ? -1.f : 1.f};
    // some three chunks a thread, and the angles in LDS
    const int64_t chunks = (int64_t)a.heads * a.dim / (vec ? e : 1);
    const int64_t want = std::max<int64_t>(1, 3 * kThreads / std::max<int64_t>(chunks, 1));
    p.per_block = (int)std::min<int64_t>(want, kTokenPairs / (a.rot / 2));
    return a.dtype == RHZ_F32 ? rope<float>(p, vec, a.interleaved, stream) : rope<uint16_t>(p, vec, a.interleaved, stream);
}

hipError_t launch_latent_append(const rhz_latent_append_args& a, hipStream_t stream) {
    const int64_t tokens = a.cu_seqlens ? (int64_t)a.seq_len : (int64_t)a.batch * a.seq_len;
    if (tokens == 0) return hipSuccess;
    const int e = a.dtype == RHZ_F32 ? 4 : 8;
    const bool vec = a.d_c % e == 0 && a.d_r % e == 0 && a.latent_stride % e == 0 && aligned16(a.latent) && aligned16(a.cache);
    const AppendParams p = {a.latent, a.k_rope, a.cu_seqlens, a.lengths, a.page_table, a.turns, a.norm_scale, a.cache,
                            a.latent_stride, a.k_rope_stride, (long)tokens, a.batch, a.seq_len, a.d_c, a.d_r, a.page_size,
                            a.num_pages, a.max_pages, a.interleaved, a.magnitude, a.eps};
    const int64_t blocks = (tokens + kThreads / kWave - 1) / (kThreads / kWave);
    if (check_grid(blocks, kThreads) != hipSuccess) return hipErrorInvalidConfiguration;
    const unsigned n = (unsigned)blocks;
    if (a.dtype == RHZ_F32) {
        if (vec)
            latent_append_kernel<float, true><<<n, kThreads, 0, stream>>>(p);
        else
            latent_append_kernel<float, false><<<n, kThreads, 0, stream>>>(p);
    } else {
        if (vec)
            latent_append_kernel<uint16_t, true><<<n, kThreads, 0, stream>>>(p);
        else
            latent_append_kernel<uint16_t, false><<<n, kThreads, 0, stream>>>(p);
    }
    return hipGetLastError();
}

}  // namespace rhz
