// gdr_conv_backward.hip -- backward pass of the Local block's prologue
// (rhz_gdr_conv_prepare: causal conv1d of width 4, q and k row norms, gates;
// delta.rs:232-243, elementwise.rs:5-12, 36-42, 125-128), for gfx950.
//
// Per channel y_t = sum_j w_j x_{t-3+j} + b, where x before a sequence's start
// is its carried state.  With dy_t the gradient of the convolved value,
//
//   q row: f = q_scale / |y|,  dy = f (dq - y (y.dq) / |y|^2);  k the same with 1 / |y|;  v: dy = dv
//   dx_p = sum_j w_j dy_{p+3-j} over the sequence's tokens, + the carried state's gradient for its last three
//   dw_j = sum_t dy_t x_{t-3+j},  db = sum_t dy_t
//   dbeta_logit = dbeta s (1 - s), s = sigmoid;  g = -softplus(a) softplus(l):
//   dl = -dg softplus(a) sigmoid(l),  da = -sum dg sigmoid(a) softplus(l).
//
// Bound by HBM: x, dq, dk and dv are read once (and three tokens on either side
// of a span again) and dx is written once; the convolution is formed again
// rather than kept.  A thread owns the channels of one 16-byte access along a
// span of tokens: dy_t adds to the four open dx_{t-3} .. dx_t, the first of
// which is then complete.  Spans are long, so that the spans' shares of dw and
// db, which go through the workspace, stay small next to the tensors.
//
// 16384 tokens of 6144 channels in bf16: 140 us for 0.65 GB (4.6 TB/s, a copy
// reaches 5.2; 5 % of it the spans' edges and shares) and 8 us for the sums.  The
// rest is the row norms' chain, y.dq and |y|^2 over a head's lanes before dy of a
// token is there.

#include <algorithm>

#include "gdr_internal.hpp"
#include "gdr_rows.hpp"

namespace rhz {
namespace {

struct ConvBackParams {
    const void *x, *dq, *dk, *dv;
    const float *w, *bias;
    const int* cu;
    const float *init, *dfin;
    const float *beta_logit, *alpha_logit, *a_log;
    const void *dbeta, *dg;
    void* dx;
    float *dinit, *dbl, *dal;
    float* part;   // [spans][5][C]
    float* parta;  // [gate blocks][H]
    int batch, seq_len, total, heads, d_k, d_v, C;
    int ncb, span, conv_blocks, gate_tokens;
    float q_scale;
};

__device__ __forceinline__ void bounds(const ConvBackParams& p, int s, int& s0, int& s1) {
    seq_bounds(p.cu, s, p.seq_len, s0, s1);
}
// The last sequence that starts at or before token t (0 if none does).
__device__ __forceinline__ int seq_of(const ConvBackParams& p, int t) {
    if (!p.cu) return t / p.seq_len;
    int lo = 0, hi = p.batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (min(max(p.cu[mid], 0), p.seq_len) <= t) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// beta's and g's logits for a block of tokens, and its share of da.
template <typename T>
__device__ __forceinline__ void gate_block(const ConvBackParams& p, int b) {
    const int H = p.heads;
    const int t0 = b * p.gate_tokens, t1 = min(t0 + p.gate_tokens, p.total);
    __shared__ float s[256];
    const int hw = min(H, 256), tw = 256 / hw;  // heads and token rows of the block's threads
    for (int h0 = 0; h0 < H; h0 += hw) {
        const int h = h0 + threadIdx.x % hw, tr = threadIdx.x / hw;
        float da = 0.f;
        if (h < H && tr < tw) {
            const float a = p.a_log[h], spa = softplus_f(a);
            for (int t = t0 + tr; t < t1; t += tw) {
                if (p.cu) {  // tokens of no sequence keep their gradients' memory
                    int s0, s1;
                    bounds(p, seq_of(p, t), s0, s1);
                    if (t < s0 || t >= s1) continue;
                }
                const long i = (long)t * H + h;
                const float sb = sigmoid_f(p.beta_logit[i]), l = p.alpha_logit[i];
                const float dg = Elem<T>::load(static_cast<const T*>(p.dg), i);
                p.dbl[i] = Elem<T>::load(static_cast<const T*>(p.dbeta), i) * sb * (1.f - sb);
                p.dal[i] = -dg * spa * sigmoid_f(l);
                da -= dg * softplus_f(l);
            }
            da *= sigmoid_f(a);
        }
        s[threadIdx.x] = da;
        __syncthreads();
        if (int(threadIdx.x) < hw && h < H) {
            float x = 0.f;
            for (int i = 0; i < tw; ++i) x += s[i * hw + threadIdx.x];
            p.parta[(long)b * H + h] = x;
        }
        __syncthreads();
    }
}

template <typename T, int G>
__global__ __launch_bounds__(256) void conv_backward_kernel(ConvBackParams p) {
    using V = Vec<T, true>;
    constexpr int N = V::N;
    if (int(blockIdx.x) >= p.conv_blocks) {
        gate_block<T>(p, blockIdx.x - p.conv_blocks);
        return;
    }
    const int span = blockIdx.x / p.ncb;
    const int c = ((blockIdx.x % p.ncb) * 256 + threadIdx.x) * N;
    if (c >= p.C) return;
    const long C = p.C;
    const int qk = p.heads * p.d_k;
    const bool isq = c < qk, isv = c >= 2 * qk;
    const T* __restrict__ x = static_cast<const T*>(p.x) + c;
    // the gradient of this thread's channels: row stride and first column
    const long dl = isv ? (long)p.heads * p.d_v : qk;
    const T* __restrict__ dp = isv   ? static_cast<const T*>(p.dv) + (c - 2 * qk)
                               : isq ? static_cast<const T*>(p.dq) + c
                                     : static_cast<const T*>(p.dk) + (c - qk);
    T* __restrict__ dx = static_cast<T*>(p.dx) + c;
    float w[N][4], b[N], dw[N][4], db[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[e][j] = p.w[4 * (c + e) + j];
            dw[e][j] = 0.f;
        }
        b[e] = p.bias ? p.bias[c + e] : 0.f;
        db[e] = 0.f;
    }
    const int t0 = span * p.span, t1 = min(t0 + p.span, p.total);
    const float scale = isq ? p.q_scale : 1.f;

    for (int s = seq_of(p, t0); s < p.batch; ++s) {
        int s0, s1;
        bounds(p, s, s0, s1);
        if (s0 >= t1) break;
        if (s1 <= t0 || s1 <= s0) continue;
        // the tokens whose dy this span needs: its own and three after them
        const int a0 = max(s0, t0), a1 = min(s1, t1 + 3);
        const bool owns_start = s0 >= t0;
        float a[3][N], o[3][N];  // x_{t-3} .. x_{t-1}; the open dx_{t-3} .. dx_{t-1}
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            const int pos = a0 - 3 + j;
            if (pos >= s0) {
                V::load(x + pos * C, a[j]);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    a[j][e] = p.init ? p.init[((long)s * C + c + e) * 3 + (3 + pos - s0)] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < N; ++e) o[j][e] = 0.f;
        }
        // dx_pos is complete: a token of this span, or a carried sample
        auto emit = [&](int pos, const float (&y)[N]) {
            if (pos >= s0) {
                if (pos >= t0 && pos < t1) V::template store<true>(dx + pos * C, y);
            } else if (owns_start && p.dinit) {
#pragma unroll
                for (int e = 0; e < N; ++e) p.dinit[((long)s * C + c + e) * 3 + (3 + pos - s0)] = y[e];
            }
        };
        auto token = [&](int t, const typename V::Raw& rx, const typename V::Raw& rd) {
            float xt[N], d[N], dy[N];
            V::unpack(rx, xt);
            V::unpack(rd, d);
            if (isv) {
#pragma unroll
                for (int e = 0; e < N; ++e) dy[e] = d[e];
            } else {
                float y[N], ss = 0.f, yd = 0.f;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    y[e] = w[e][0] * a[0][e] + w[e][1] * a[1][e] + w[e][2] * a[2][e] + w[e][3] * xt[e] + b[e];
                    ss += y[e] * y[e];
                    yd += y[e] * d[e];
                }
                ss = row_sum<G>(ss);
                yd = row_sum<G>(yd);
                // |y| below 1e-12 is taken as 1e-12 by the forward pass, a constant
                const float r = __builtin_amdgcn_rsqf(fmaxf(ss, 1e-24f)), f = scale * r;
                const float m = ss > 1e-24f ? yd * r * r : 0.f;
#pragma unroll
                for (int e = 0; e < N; ++e) dy[e] = f * (d[e] - y[e] * m);
            }
            float done[N];
            const bool mine = t < t1;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                done[e] = o[0][e] + w[e][0] * dy[e];
                o[0][e] = o[1][e] + w[e][1] * dy[e];
                o[1][e] = o[2][e] + w[e][2] * dy[e];
                o[2][e] = w[e][3] * dy[e];
                const float u = mine ? dy[e] : 0.f;
                dw[e][0] += u * a[0][e];
                dw[e][1] += u * a[1][e];
                dw[e][2] += u * a[2][e];
                dw[e][3] += u * xt[e];
                db[e] += u;
                a[0][e] = a[1][e];
                a[1][e] = a[2][e];
                a[2][e] = xt[e];
            }
            emit(t - 3, done);
        };
        // four tokens at a time, the next four's inputs read ahead
        constexpr int U = 4;
        typename V::Raw rx[U], rd[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const long t = min(a0 + i, a1 - 1);
            rx[i] = V::load_raw(x + t * C);
            rd[i] = V::load_raw(dp + t * dl);
        }
        for (int t = a0; t < a1; t += U) {
            typename V::Raw nx[U], nd[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const long n = min(t + U + i, a1 - 1);
                nx[i] = V::load_raw(x + n * C);
                nd[i] = V::load_raw(dp + n * dl);
            }
#pragma unroll
            for (int i = 0; i < U; ++i)
                if (t + i < a1) token(t + i, rx[i], rd[i]);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                rx[i] = nx[i];
                rd[i] = nd[i];
            }
        }
        if (a1 == s1) {  // the sequence's end: the last three inputs are the carried state too
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                if (p.dfin)
#pragma unroll
                    for (int e = 0; e < N; ++e) o[j][e] += p.dfin[((long)s * C + c + e) * 3 + j];
                emit(s1 - 3 + j, o[j]);
            }
        }
    }
    float* part = p.part + (long)span * 5 * C + c;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) part[j * C + e] = dw[e][j];
#pragma unroll
    for (int e = 0; e < N; ++e) part[4 * C + e] = db[e];
}

// The carried state of an empty sequence passes through.
__global__ __launch_bounds__(256) void conv_backward_empty_kernel(ConvBackParams p) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.C) return;
    for (int s = blockIdx.y; s < p.batch; s += gridDim.y) {
        int s0, s1;
        bounds(p, s, s0, s1);
        if (s1 > s0) continue;
        const long o = ((long)s * p.C + c) * 3;
#pragma unroll
        for (int k = 0; k < 3; ++k) p.dinit[o + k] = p.dfin ? p.dfin[o + k] : 0.f;
    }
}

// dw [C, 4], dbias [C] and da_log [H] from the blocks' shares, in a fixed
// order: 64 columns (of the 5 C, then of the H) and 16 slices of the shares to
// a workgroup.
__global__ __launch_bounds__(1024) void conv_backward_sums_kernel(ConvBackParams p, int spans, int gates, float* dw,
                                                                  float* db, float* da) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
    const long wide = 5L * p.C, nw = (wide + 63) / 64;
    const bool gate = blockIdx.x >= nw;
    const long c = (gate ? blockIdx.x - nw : blockIdx.x) * 64 + lane, cols = gate ? p.heads : wide;
    const float* part = gate ? p.parta : p.part;
    const int n = gate ? gates : spans;
    float x = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int b = slice; b < n; b += 16) x += part[b * cols + c];
    }
    s[slice][lane] = x;
    __syncthreads();
    if (slice || c >= cols) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) x += s[i][lane];
    if (gate) {
        da[c] = x;
    } else if (c >= 4L * p.C) {
        if (db) db[c - 4L * p.C] = x;
    } else {
        dw[(c % p.C) * 4 + c / p.C] = x;
    }
}

// Spans and gate blocks of a call.
struct ConvBackShape {
    int total, n, ncb, span, spans, gate_tokens, gates;
};
// About kBlocks blocks of 256 threads (four per CU): fewer leave HBM waiting,
// more write more shares of dw (20 bytes per channel and span).  16384 tokens of
// 6144 channels in bf16, whole call: 174 us with 256 blocks, 159 with 512, 148
// with 1024, 158 with 1536, 166 with 2048.  Spans are 8 tokens at least: six more
// are read at their edges.  64 tokens, waited for: 43 us, 48 with spans of 16; 1080
// tokens of 1536 channels in fp32 29.3 and 28.8 us.
constexpr int kBlocks = 1024, kMinSpan = 8;
ConvBackShape conv_back_shape(const rhz_gdr_conv_prepare_backward_args& a) {
    ConvBackShape s{};
    s.total = a.cu_seqlens ? a.seq_len : a.batch * a.seq_len;
    s.n = a.dtype == RHZ_F32 ? 4 : 8;
    const int C = a.heads * (2 * a.d_k + a.d_v);
    s.ncb = (C / s.n + 255) / 256;
    const int want = std::max(1, kBlocks / s.ncb);
    s.span = std::max(kMinSpan, (s.total + want - 1) / want);
    s.spans = (s.total + s.span - 1) / s.span;
    const int rows = std::max(1, 256 / std::min(a.heads, 256));  // tokens of a gate block at once
    s.gate_tokens = std::max(rows, (s.total + 255) / 256);
    s.gates = (s.total + s.gate_tokens - 1) / s.gate_tokens;
    return s;
}

}  // namespace

size_t conv_prepare_backward_workspace_bytes(const rhz_gdr_conv_prepare_backward_args& a) {
    const ConvBackShape s = conv_back_shape(a);
    const size_t C = (size_t)a.heads * (2 * a.d_k + a.d_v);
    return (size_t)s.spans * 5 * C * 4 + (size_t)s.gates * a.heads * 4;
}

hipError_t launch_conv_prepare_backward(const rhz_gdr_conv_prepare_backward_args& a, hipStream_t st) {
    const ConvBackShape s = conv_back_shape(a);
    const int C = a.heads * (2 * a.d_k + a.d_v);
    ConvBackParams p{};
    p.x = a.x;
    p.dq = a.grad_q;
    p.dk = a.grad_k;
    p.dv = a.grad_v;
    p.w = a.weight;
    p.bias = a.bias;
    p.cu = a.cu_seqlens;
    p.init = a.initial_state;
    p.dfin = a.grad_final_state;
    p.beta_logit = a.beta_logit;
    p.alpha_logit = a.alpha_logit;
    p.a_log = a.a_log;
    p.dbeta = a.grad_beta;
    p.dg = a.grad_g;
    p.dx = a.grad_x;
    p.dinit = a.grad_initial_state;
    p.dbl = a.grad_beta_logit;
    p.dal = a.grad_alpha_logit;
    p.part = static_cast<float*>(a.workspace);
    p.parta = p.part + (size_t)s.spans * 5 * C;
    p.batch = a.batch;
    p.seq_len = a.seq_len;
    p.total = s.total;
    p.heads = a.heads;
    p.d_k = a.d_k;
    p.d_v = a.d_v;
    p.C = C;
    p.ncb = s.ncb;
    p.span = s.span;
    p.conv_blocks = s.spans * s.ncb;
    p.gate_tokens = s.gate_tokens;
    p.q_scale = a.q_scale;
    if (s.total > 0) {
        const int64_t blocks = (int64_t)p.conv_blocks + s.gates;
        if (const hipError_t e = check_grid(blocks, 256); e != hipSuccess) return e;
        const dim3 grid((unsigned)blocks);
#define RHZ_CONV_BACK(T, G) hipLaunchKernelGGL((conv_backward_kernel<T, G>), grid, dim3(256), 0, st, p)
#define RHZ_CONV_BACK_G(T) \
    switch (a.d_k / s.n) { \
        case 1: RHZ_CONV_BACK(T, 1); break; \
        case 2: RHZ_CONV_BACK(T, 2); break; \
        case 4: RHZ_CONV_BACK(T, 4); break; \
        case 8: RHZ_CONV_BACK(T, 8); break; \
        case 16: RHZ_CONV_BACK(T, 16); break; \
        case 32: RHZ_CONV_BACK(T, 32); break; \
        default: RHZ_CONV_BACK(T, 64); break; \
    }
        if (a.dtype == RHZ_F32) {
            RHZ_CONV_BACK_G(float)
        } else {
            RHZ_CONV_BACK_G(uint16_t)
        }
#undef RHZ_CONV_BACK_G
#undef RHZ_CONV_BACK
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    const int64_t sums = (5LL * C + 63) / 64 + (a.heads + 63) / 64;
    if (const hipError_t e = check_grid(sums, 1024); e != hipSuccess) return e;
    hipLaunchKernelGGL(conv_backward_sums_kernel, dim3((unsigned)sums), dim3(1024), 0, st, p, s.spans, s.gates,
                       a.grad_weight, a.grad_bias, a.grad_a_log);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (a.grad_initial_state && (a.cu_seqlens || a.seq_len == 0)) {
        hipLaunchKernelGGL(conv_backward_empty_kernel, dim3((C + 255) / 256, std::min(a.batch, 65535)), dim3(256), 0, st,
                           p);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace rhz
