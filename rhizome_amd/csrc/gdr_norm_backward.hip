// gdr_norm_backward.hip -- layer norm, its backward pass, and the backward pass
// of the per-head RMSNorm (norm.rs:8-13, 48-59), for gfx950.
//
// Per row of n values, r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r
// (RMSNorm: mu = 0), t = dy * w:
//
//   layer norm   y = xh * w + b
//   dx = r (t - mean(t) - xh mean(t * xh))      (RMSNorm: without mean(t))
//   dw = sum over rows of dy * xh,  db = sum over rows of dy.
//
// All are bound by HBM: a row is read once into registers, where its sums are
// taken (the variance from the centred values), and its output written once.
// The rows of a block run along its persistent threads, each of which keeps
// its columns' share of dw and db in registers; the blocks' shares go to the
// workspace and a second kernel adds them in a fixed order.
//
// bf16, of a copy's 5.2 TB/s: layer norm of 16384 rows of 2048, 0.13 GB in 29 us
// (4.6 TB/s); its backward pass, 0.21 GB in 43 us (4.9) and 4 us for the sums;
// RMSNorm's backward pass of 262144 rows of 128, 0.20 GB in 39 us (5.1) and 4 us.

#include <algorithm>

#include "gdr_internal.hpp"
#include "gdr_rows.hpp"

namespace rhz {
namespace {

struct NormParams {
    const void *dy, *x;
    const float *w, *b;
    void* out;    // y, or dx
    float* part;  // backward: [blocks][2 or 1][dim]
    int rows, dim;
    float eps;
};

// A group of G threads per row (256: the whole block), NV vectors each.
template <int G>
__device__ __forceinline__ float group_total(float x, float* red) {
    if constexpr (G <= 64) {
        return row_sum<G>(x);
    } else {
        x = row_sum<64>(x);
        __syncthreads();  // the previous sum has been read
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
        __syncthreads();
        return (red[0] + red[1]) + (red[2] + red[3]);
    }
}

template <typename T, bool VEC, int G, int NV>
struct Rows {
    using V = Vec<T, VEC>;
    static constexpr int N = V::N;
    static constexpr int kGroups = 256 / G;                        // rows of a block at once
    static constexpr int kUnroll = NV >= 4 || G > 64 ? 1 : 4 / NV;  // of a group
    static constexpr bool kKeepW = NV * N <= 32;                   // the weights stay in registers
    static __device__ __forceinline__ void load_raw(typename V::Raw (&r)[NV], const T* row, int li, int dim) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (li + G * i) * N;
            r[i] = j < dim ? V::load_raw(row + j) : typename V::Raw{};
        }
    }
    static __device__ __forceinline__ void unpack(const typename V::Raw (&r)[NV], float (&x)[NV][N]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) V::unpack(r[i], x[i]);
    }
    static __device__ __forceinline__ void weights(float (&w)[NV][N], const float* p, int li, int dim) {
#pragma unroll
        for (int i = 0; i < NV; ++i) weights1(w[i], p, (li + G * i) * N, dim);
    }
    static __device__ __forceinline__ void weights1(float (&w)[N], const float* p, int j, int dim) {
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = p && j < dim ? p[j + e] : 0.f;
    }
    // x - mu and r of a row; columns beyond the row stay zero
    template <bool CENTER>
    static __device__ __forceinline__ float stats(float (&x)[NV][N], int li, int dim, float eps, float* red) {
        if constexpr (CENTER) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) s += x[i][e];
            const float mu = group_total<G>(s, red) / (float)dim;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) x[i][e] = (li + G * i) * N < dim ? x[i][e] - mu : 0.f;
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) ss += x[i][e] * x[i][e];
        return 1.f / sqrtf(group_total<G>(ss, red) / (float)dim + eps);
    }
};

template <typename T, bool VEC, int G, int NV>
__global__ __launch_bounds__(256) void layernorm_kernel(NormParams p) {
    using R = Rows<T, VEC, G, NV>;
    using V = typename R::V;
    constexpr int N = R::N, U = R::kUnroll, RPB = R::kGroups;
    __shared__ float red[4];
    const int li = threadIdx.x % G, row0 = blockIdx.x * RPB * U + threadIdx.x / G;
    typename V::Raw raw[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (row0 + u * RPB < p.rows)
            R::load_raw(raw[u], static_cast<const T*>(p.x) + (long)(row0 + u * RPB) * p.dim, li, p.dim);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int row = row0 + u * RPB;
        if (row >= p.rows) break;  // uniform over the group
        float x[NV][N];
        R::unpack(raw[u], x);
        const float r = R::template stats<true>(x, li, p.dim, p.eps, red);
        T* y = static_cast<T*>(p.out) + (long)row * p.dim;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (li + G * i) * N;
            if (j >= p.dim) continue;
            float w[N], b[N], o[N];
            R::weights1(w, p.w, j, p.dim);
            R::weights1(b, p.b, j, p.dim);
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] = x[i][e] * r * w[e] + b[e];
            V::template store<true>(y + j, o);
        }
    }
}

template <typename T, bool VEC, int G, int NV, bool CENTER>
__global__ __launch_bounds__(256) void norm_backward_kernel(NormParams p) {
    using R = Rows<T, VEC, G, NV>;
    using V = typename R::V;
    constexpr int N = R::N, U = R::kUnroll, RPB = R::kGroups;
    __shared__ float red[4];
    __shared__ float cols[CENTER ? 2 : 1][(G < 64 ? G : 64) * NV * N];
    const int li = threadIdx.x % G, grp = threadIdx.x / G;
    float aw[NV][N], ab[NV][N], w[NV][N];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) aw[i][e] = ab[i][e] = 0.f;
    if constexpr (R::kKeepW) R::weights(w, p.w, li, p.dim);
    typename V::Raw rx[U][NV], ry[U][NV];
    // rows go up to 2^31 - 1 (dim = 1) and the counter two steps beyond: unsigned
    const unsigned rows = p.rows;
    auto load = [&](unsigned first) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned row = first + u * RPB;
            if (row < rows) {
                R::load_raw(rx[u], static_cast<const T*>(p.x) + (long)row * p.dim, li, p.dim);
                R::load_raw(ry[u], static_cast<const T*>(p.dy) + (long)row * p.dim, li, p.dim);
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i) rx[u][i] = ry[u][i] = typename V::Raw{};
            }
        }
    };
    const unsigned step = gridDim.x * RPB * U;
    unsigned base = blockIdx.x * RPB * U;  // the same for the whole block
    load(base + grp);
    for (; base < rows; base += step) {
        float x[U][NV][N], y[U][NV][N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            R::unpack(rx[u], x[u]);
            R::unpack(ry[u], y[u]);
        }
        load(base + step + grp);  // rows beyond the last are zero
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned row = base + grp + u * RPB;
            float r = R::template stats<CENTER>(x[u], li, p.dim, p.eps, red);
            if (row >= rows) r = 0.f;  // no row: nothing is added, with eps = 0 too
            float st = 0.f, sx = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float wi[N];
                if constexpr (R::kKeepW) {
#pragma unroll
                    for (int e = 0; e < N; ++e) wi[e] = w[i][e];
                } else {
                    R::weights1(wi, p.w, (li + G * i) * N, p.dim);
                }
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    x[u][i][e] *= r;
                    aw[i][e] += y[u][i][e] * x[u][i][e];
                    if constexpr (CENTER) ab[i][e] += y[u][i][e];
                    y[u][i][e] *= wi[e];
                    st += y[u][i][e];
                    sx += y[u][i][e] * x[u][i][e];
                }
            }
            const float mx = group_total<G>(sx, red) / (float)p.dim;
            const float mt = CENTER ? group_total<G>(st, red) / (float)p.dim : 0.f;
            if (row < rows) {
                T* o = static_cast<T*>(p.out) + (long)row * p.dim;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int j = (li + G * i) * N;
                    if (j >= p.dim) continue;
                    float d[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) d[e] = r * (y[u][i][e] - mt - x[u][i][e] * mx);
                    V::template store<true>(o + j, d);
                }
            }
        }
    }
    // the block's share of dw (and db): over a wave's groups by lane exchange,
    // over the waves through LDS in their order
    float* part = p.part + (long)blockIdx.x * (CENTER ? 2 : 1) * p.dim;
    if constexpr (G <= 64) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e)
#pragma unroll
                for (int off = G; off < 64; off <<= 1) {
                    aw[i][e] += __shfl_xor(aw[i][e], off, kWave);
                    if constexpr (CENTER) ab[i][e] += __shfl_xor(ab[i][e], off, kWave);
                }
        for (int wv = 0; wv < 4; ++wv) {
            if (int(threadIdx.x >> 6) == wv && int(threadIdx.x & 63) < G) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const int j = (li + G * i) * N + e;
                        cols[0][j] = wv ? cols[0][j] + aw[i][e] : aw[i][e];
                        if constexpr (CENTER) cols[CENTER][j] = wv ? cols[CENTER][j] + ab[i][e] : ab[i][e];
                    }
            }
            __syncthreads();
        }
        for (int j = threadIdx.x; j < p.dim; j += 256) {
            part[j] = cols[0][j];
            if constexpr (CENTER) part[p.dim + j] = cols[CENTER][j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int j = (li + G * i) * N + e;
                if (j < p.dim) {
                    part[j] = aw[i][e];
                    if constexpr (CENTER) part[p.dim + j] = ab[i][e];
                }
            }
    }
}

// out[c] = sum over b of part[b][c], c < cols (dw's, then db's): 64 columns
// and 16 slices of the blocks to a workgroup.
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* part, int blocks, int cols, int dim, float* dw,
                                                           float* db) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    float x = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int b = slice; b < blocks; b += 16) x += part[(long)b * cols + c];
    }
    s[slice][lane] = x;
    __syncthreads();
    if (slice == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 16; ++i) x += s[i][lane];
        if (c < dim) {
            if (dw) dw[c] = x;
        } else if (db) {
            db[c - dim] = x;
        }
    }
}

constexpr int kNormBlocks = 512;  // two per CU (four: 16384 rows of 2048 backward 54 us instead of 47)

struct NormShape {
    bool vec;
    int g, nv, unroll;
};
// Lanes per row and vectors per lane: as few lanes as hold the row in one
// vector each, a wave with up to four (scalar: sixteen), then the block.  bf16,
// layer norm and its backward pass: rows of 64 on 8 lanes 28 and 52 us, on 16
// lanes 44 and 81 (524288 rows); of 2048 on a wave 28 and 47 us, on a block 34
// and 112 (16384 rows); of 4096 on a wave 29 and 92 us, on a block 27 and 62.
NormShape norm_shape(int dtype, int dim, bool vec) {
    const int n = dtype == RHZ_F32 ? 4 : 8;
    if (vec && dim % n == 0) {
        const int v = dim / n;
        if (v <= 8) return {true, 8, 1, 4};
        if (v <= 16) return {true, 16, 1, 4};
        if (v <= 32) return {true, 32, 1, 4};
        if (v <= 64) return {true, 64, 1, 4};
        if (v <= 128) return {true, 64, 2, 2};
        if (v <= 256) return {true, 64, 4, 1};
        if (v <= 512) return {true, 256, 2, 1};
        if (v <= 1024) return {true, 256, 4, 1};
        return {true, 256, 8, 1};
    }
    if (dim <= 64) return {false, 16, 4, 1};
    if (dim <= 256) return {false, 64, 4, 1};
    if (dim <= 1024) return {false, 64, 16, 1};
    if (dim <= 2048) return {false, 256, 8, 1};
    return {false, 256, 32, 1};
}
int64_t norm_blocks(const NormShape& s, int64_t rows) {
    const int64_t per = (256 / s.g) * s.unroll;
    return (rows + per - 1) / per;
}

template <template <typename, bool, int, int> class K, typename T>
hipError_t go_norm(const NormParams& p, const NormShape& s, int64_t blocks, hipStream_t st) {
    if (blocks <= 0) return hipSuccess;
    if (const hipError_t e = check_grid(blocks, 256); e != hipSuccess) return e;
#define RHZ_NORM(VEC, G, NV) \
    if (s.vec == VEC && s.g == G && s.nv == NV) \
        hipLaunchKernelGGL((K<T, VEC, G, NV>::fn), dim3((unsigned)blocks), dim3(256), 0, st, p)
    RHZ_NORM(true, 8, 1);
    RHZ_NORM(true, 16, 1);
    RHZ_NORM(true, 32, 1);
    RHZ_NORM(true, 64, 1);
    RHZ_NORM(true, 64, 2);
    RHZ_NORM(true, 64, 4);
    RHZ_NORM(true, 256, 2);
    RHZ_NORM(true, 256, 4);
    RHZ_NORM(true, 256, 8);
    RHZ_NORM(false, 16, 4);
    RHZ_NORM(false, 64, 4);
    RHZ_NORM(false, 64, 16);
    RHZ_NORM(false, 256, 8);
    RHZ_NORM(false, 256, 32);
#undef RHZ_NORM
    return hipGetLastError();
}
template <typename T, bool VEC, int G, int NV>
struct LayerK {
    static constexpr auto fn = layernorm_kernel<T, VEC, G, NV>;
};
template <typename T, bool VEC, int G, int NV>
struct LayerBackK {
    static constexpr auto fn = norm_backward_kernel<T, VEC, G, NV, true>;
};
template <typename T, bool VEC, int G, int NV>
struct RmsBackK {
    static constexpr auto fn = norm_backward_kernel<T, VEC, G, NV, false>;
};

}  // namespace

hipError_t launch_layernorm(const rhz_layernorm_args& a, hipStream_t st) {
    const NormShape s = norm_shape(a.dtype, a.dim, aligned16(a.x) && aligned16(a.y));
    const NormParams p{nullptr, a.x, a.weight, a.bias, a.y, nullptr, a.rows, a.dim, a.eps};
    const int64_t blocks = norm_blocks(s, a.rows);
    if (a.dtype == RHZ_F32) return go_norm<LayerK, float>(p, s, blocks, st);
    return go_norm<LayerK, uint16_t>(p, s, blocks, st);
}

// The shares of the most blocks that a call of these sizes can have, whatever its alignment.
size_t norm_backward_workspace_bytes(const rhz_norm_backward_args& a) {
    return (size_t)std::min<int64_t>(a.rows, kNormBlocks) * 2 * a.dim * 4;
}

hipError_t launch_norm_backward(const rhz_norm_backward_args& a, bool layer, hipStream_t st) {
    const NormShape s = norm_shape(a.dtype, a.dim, aligned16(a.x) && aligned16(a.grad_y) && aligned16(a.grad_x));
    float* part = static_cast<float*>(a.workspace);
    const NormParams p{a.grad_y, a.x, a.weight, nullptr, a.grad_x, part, a.rows, a.dim, a.eps};
    const int64_t blocks = std::min<int64_t>(norm_blocks(s, a.rows), kNormBlocks);
    hipError_t e;
    if (layer)
        e = a.dtype == RHZ_F32 ? go_norm<LayerBackK, float>(p, s, blocks, st)
                               : go_norm<LayerBackK, uint16_t>(p, s, blocks, st);
    else
        e = a.dtype == RHZ_F32 ? go_norm<RmsBackK, float>(p, s, blocks, st)
                               : go_norm<RmsBackK, uint16_t>(p, s, blocks, st);
    if (e != hipSuccess) return e;
    const int cols = (layer ? 2 : 1) * a.dim;
    hipLaunchKernelGGL(column_sums_kernel, dim3((cols + 63) / 64), dim3(1024), 0, st, part, (int)blocks, cols, a.dim,
                       a.grad_weight, a.grad_bias);
    return hipGetLastError();
}

}  // namespace rhz
