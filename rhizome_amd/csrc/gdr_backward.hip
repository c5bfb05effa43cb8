// gdr_backward.hip -- backward pass of the gated delta-rule prefill, gfx950.
//
// The forward recurrence in chunks of 64 tokens (S0 the state before the
// chunk, G the running log-decay from the chunk's start, gamma = e^G, tail_s =
// e^{G_c - G_s}, D_rs = e^{G_r - G_s} for s <= r):
//
//   L_rs = D_rs k_r.k_s (s < r),  P_rs = D_rs q_r.k_s (s <= r),
//   T = (I + L diag(beta))^{-1},
//   W = T (V - diag(gamma) K S0^T)         (beta_s w_s is what token s writes)
//   O = diag(gamma) Q S0^T + P diag(beta) W
//   S1 = gamma_c S0 + sum_s beta_s tail_s w_s k_s^T
//
// and its adjoint, dS1 being the gradient of the state after the chunk:
//
//   dX = T^T diag(beta) (P^T dO + diag(tail) K dS1^T)                  (= dV)
//   dS0 = gamma_c dS1 + dO^T diag(gamma) Q - dX^T diag(gamma) K
//   N1 = (dO W^T) o D diag(beta) (s <= r),  N2 = (dX W^T) o D diag(beta) (s < r)
//   dQ = diag(gamma) dO S0 + N1 K
//   dK = diag(beta tail) W dS1 - diag(gamma) dX S0 + N1^T Q - (N2 + N2^T) K
//   dbeta_s = tail_s k_s.(W dS1)_s + sum_r (P o dO W^T - L o dX W^T)_rs
//   dg_t = gamma_c <dS1, S0> + sum_{r >= t} a_r + sum_{s < t} b_s
//          + sum_{r >= t > s} M_rs,
//     a_r = gamma_r (q_r.(dO S0)_r - k_r.(dX S0)_r),
//     b_s = beta_s tail_s k_s.(W dS1)_s,  M = N1 o (Q K^T) - N2 o (K K^T).
//
// dg is summed over exactly the pairs (r, s) whose decay holds alpha_t, so
// nothing cancels and dalpha_t = dg_t / alpha_t keeps its accuracy for small
// alpha_t; below kTinyAlpha the sum is formed without alpha_t's factor.
//
// Kernels: bwd_prep_kernel forms what depends on one chunk's inputs alone
// (T and the products with it) for every (chunk, head) at once;
// bwd_scan_kernel carries S and dS along the chunks, the two directions at
// the same time since neither needs the other; bwd_grad_kernel forms the
// gradients of every (chunk, head) at once from S0 and dS1.
//
// bf16 tensors are multiplied as fp16 (11 significant bits) on MFMA with fp32
// accumulation: each fp16 operand is scaled by a power of two of its own, from
// the largest magnitude of the tile it is rounded in, so that the magnitude of
// the inputs (a loss's gradient of 1e-8, say) does not matter.  S, dS and every
// sum are fp32.  fp32 tensors are multiplied in fp32 throughout.

#include <algorithm>
#include <type_traits>

#include "gdr_device.hpp"
#include "gdr_internal.hpp"

namespace rhz {
namespace {

constexpr int C64 = kChunk;           // tokens of a chunk
constexpr double kMinLog = -1000.0;   // log-decays below it decay to 0 in fp32 all the same
constexpr float kTinyAlpha = 1e-18f;  // below: dalpha is formed without dividing by alpha

// ------------------------------------------------------------- operands
// An MFMA operand is held in "units" of 16 bytes per lane.  Lane (g, m), g =
// lane / 16, m = lane % 16, holds for row m of a 16-row tile the contraction
// indices 16 b + 4 g .. + 3 of one (fp32) or two (fp16) blocks b.  An
// accumulator tile holds rows 4 g .. 4 g + 3 of column m, so accumulators are
// the units of the next product's right operand as they stand.
struct OpF16 {
    using Elt = _Float16;
    using Unit = f16x8;
    static constexpr int kBlocks = 2;  // 16-index blocks of a unit
    static constexpr bool kScaled = true;
    static __device__ __forceinline__ f32x4 mma(const Unit& a, const Unit& b, const f32x4& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    // the unit of two accumulator tiles, times s
    static __device__ __forceinline__ Unit pack(const f32x4* t, float s) {
        Unit u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = (_Float16)(t[0][i] * s);
            u[4 + i] = (_Float16)(t[1][i] * s);
        }
        return u;
    }
    static __device__ __forceinline__ void unpack(const Unit& u, f32x4* t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            t[0][i] = (float)u[i];
            t[1][i] = (float)u[4 + i];
        }
    }
};
struct OpF32 {
    using Elt = float;
    using Unit = f32x4;
    static constexpr int kBlocks = 1;
    static constexpr bool kScaled = false;
    static __device__ __forceinline__ f32x4 mma(const Unit& a, const Unit& b, f32x4 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Unit pack(const f32x4* t, float s) {
        Unit u;
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = t[0][i] * s;
        return u;
    }
    static __device__ __forceinline__ void unpack(const Unit& u, f32x4* t) { t[0] = u; }
};

// A matrix of units in LDS, NKU units along the contraction per 16-row tile.
// A wave reads one unit of a tile at once, 1 KiB; within it the row is XORed
// so that the staging writes, which run along tiles, units and g, spread over
// the banks.
template <class Op, int NKU>
struct LdsMat {
    using Unit = typename Op::Unit;
    using Elt = typename Op::Elt;
    static constexpr int kTileBytes = NKU * 1024;
    char* p;
    static __device__ __forceinline__ int slot(int mt, int ku, int g, int m) {
        return g * 16 + (m ^ (((g << 2) ^ (ku & 3) ^ (mt & 3)) & 15));
    }
    __device__ __forceinline__ Unit unit(int mt, int ku, int lane) const {
        return *reinterpret_cast<const Unit*>(p + (mt * NKU + ku) * 1024 + slot(mt, ku, lane >> 4, lane & 15) * 16);
    }
    __device__ __forceinline__ void put_unit(int mt, int ku, int lane, const Unit& u) const {
        *reinterpret_cast<Unit*>(p + (mt * NKU + ku) * 1024 + slot(mt, ku, lane >> 4, lane & 15) * 16) = u;
    }
    // the four contraction indices k .. k + 3 (k a multiple of 4) of a row
    static __device__ __forceinline__ int offset4(int row, int k) {
        const int b = k >> 4, ku = b / Op::kBlocks, half = b % Op::kBlocks;
        return ((row >> 4) * NKU + ku) * 1024 + slot(row >> 4, ku, (k >> 2) & 3, row & 15) * 16 + half * 8;
    }
    __device__ __forceinline__ void put4(int row, int k, float a, float b, float c, float d) const {
        if constexpr (Op::kScaled) {
            uint2 u = {pack_f16x2(a, b), pack_f16x2(c, d)};
            *reinterpret_cast<uint2*>(p + offset4(row, k)) = u;
        } else {
            *reinterpret_cast<f32x4*>(p + offset4(row, k)) = f32x4{a, b, c, d};
        }
    }
    __device__ __forceinline__ void put4(int row, int k, uint2 u) const {
        *reinterpret_cast<uint2*>(p + offset4(row, k)) = u;
    }
    __device__ __forceinline__ f32x4 get4(int row, int k) const {
        if constexpr (Op::kScaled) {
            typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
            const f16x4 h = *reinterpret_cast<const f16x4*>(p + offset4(row, k));
            return f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
        } else {
            return *reinterpret_cast<const f32x4*>(p + offset4(row, k));
        }
    }
};

// 64 x 64 fp32 in LDS, 16-byte groups of a row XORed by the row.
__device__ __forceinline__ int sq_at(int r, int c) { return r * 64 + ((((c >> 2) ^ r) & 15) << 2) + (c & 3); }

__device__ __forceinline__ int bits_abs(float x) { return int(__float_as_uint(x) & 0x7fffffffu); }
// Maximum over the wave of non-negative ints (magnitude bits: a NaN's are the largest).
__device__ __forceinline__ int wave_max_bits(int x) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x = max(x, __shfl_xor(x, off, kWave));
    return __builtin_amdgcn_readfirstlane(x);
}
// The power of two that a tile of largest magnitude `bits` is divided by, so
// that its largest value lands in [2^to, 2^(to+1)).
__device__ __forceinline__ int tile_exp(int bits, int to) { return max(min((bits >> 23) - 127, 100), -100) - to; }

// Four consecutive elements of a row, zero from `n` on.
template <typename T>
__device__ __forceinline__ float4 row4(const T* p, int n, bool vec) {
    if (vec && n >= 4) return load4(p);
    float4 r;
    r.x = n > 0 ? Elem<T>::load(p, 0) : 0.f;
    r.y = n > 1 ? Elem<T>::load(p, 1) : 0.f;
    r.z = n > 2 ? Elem<T>::load(p, 2) : 0.f;
    r.w = n > 3 ? Elem<T>::load(p, 3) : 0.f;
    return r;
}
template <typename T>
__device__ __forceinline__ void put_row4(T* p, int n, bool vec, float a, float b, float c, float d) {
    if (vec && n >= 4) {
        if constexpr (sizeof(T) == 4)
            *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d};
        else
            *reinterpret_cast<uint2*>(p) = uint2{pack_bf16x2(a, b), pack_bf16x2(c, d)};
        return;
    }
    if (n > 0) Elem<T>::store(p, 0, a);
    if (n > 1) Elem<T>::store(p, 1, b);
    if (n > 2) Elem<T>::store(p, 2, c);
    if (n > 3) Elem<T>::store(p, 3, d);
}

// ------------------------------------------------------------ workspace
// One record per (chunk, head): unit matrices for DK = d_k padded to 32, 64
// or 128 and d_v padded to 16-row tiles (an even number of them).
struct RecLayout {
    size_t wk, kt, kd, qt, wt, ot, dot, s0, ds1, vec, bytes;
};
__host__ __device__ inline RecLayout rec_layout(int DK, int dvt, int es) {
    RecLayout l{};
    const size_t tk = (size_t)64 * DK * es, tv = (size_t)64 * dvt * 16 * es, st = (size_t)DK * dvt * 16 * es;
    size_t at = 0;
    l.wk = at; at += tk;    // T diag(gamma) K          (token; d_k)
    l.kt = at; at += tk;    // K                        (d_k; token)
    l.kd = at; at += tk;    // T^T diag(beta tail) K    (token; d_k)
    l.qt = at; at += tk;    // Q                        (d_k; token)
    l.wt = at; at += tv;    // T V, then W              (d_v; token)
    l.ot = at; at += tv;    // T^T diag(beta) P^T dO, then dX  (d_v; token)
    l.dot = at; at += tv;   // dO                       (d_v; token)
    l.s0 = at; at += st;    // S0                       (d_v; d_k)
    l.ds1 = at; at += st;   // dS1                      (d_v; d_k)
    l.vec = at;             // Vec, then the tiles' exponents
    at += 256 * 4 + 6 * 64 * 4;
    l.bytes = (at + 255) & ~(size_t)255;
    return l;
}
// the record's small values: gamma [64], beta tail [64], gamma_c, exponents of K and Q
enum { kVecGamma = 0, kVecWrite = 64, kVecGc = 128, kVecEK = 129, kVecEQ = 130, kVecBad = 131 };
// exponents by d_v tile, from float 256 on
enum { kExpV = 256, kExpO = 320, kExpW = 384, kExpX = 448, kExpS = 512, kExpD = 576 };

struct BwdParams {
    const void *q, *k, *v, *dout;
    const float *gate, *beta, *init, *dfinal;
    const int *cu, *chunk_base;  // packed: chunk_base[n] chunks precede sequence n
    void *dq, *dk, *dv, *dgate, *dbeta;
    float* dinit;
    char* ws;
    RecLayout rec;
    int batch, seq_len, heads, d_k, d_v, dvt, gate_is_alpha;
    bool vec_k, vec_v;  // rows of q, k (of v, dO) are loaded and stored four elements at a time
    bool vec_s;         // rows of the states, 16 bytes at a time
};

// The chunk `ci` of the launch: its sequence, first token and number of
// tokens; false beyond the last chunk.
struct ChunkAt {
    int seq, t0, n;
};
__device__ __forceinline__ bool find_chunk(const BwdParams& p, int ci, ChunkAt& at) {
    if (!p.cu) {
        const int nc = (p.seq_len + C64 - 1) / C64;
        at.seq = ci / nc;
        const int c = ci - at.seq * nc;
        at.t0 = at.seq * p.seq_len + c * C64;
        at.n = min(C64, p.seq_len - c * C64);
        return true;
    }
    if (ci >= p.chunk_base[p.batch]) return false;
    int lo = 0, hi = p.batch - 1;  // the last sequence with chunk_base <= ci
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.chunk_base[mid] <= ci) lo = mid; else hi = mid - 1;
    }
    int a, b;
    seq_bounds(p.cu, lo, p.seq_len, a, b);
    at.seq = lo;
    at.t0 = a + (ci - p.chunk_base[lo]) * C64;
    at.n = min(C64, b - at.t0);
    return true;
}

// Running log-decays and factors of a chunk, by the first wave.
struct Gates {
    double G[64];
    float gamma[64], tail[64], beta[64], gate[64];
};
__device__ __forceinline__ bool load_gates(const BwdParams& p, const ChunkAt& at, int h, Gates& gs, int lane) {
    const bool in = lane < at.n;
    const long r = (long)(at.t0 + (in ? lane : 0)) * p.heads + h;
    const float gate = in ? p.gate[r] : (p.gate_is_alpha ? 1.f : 0.f);
    const float beta = in ? p.beta[r] : 0.f;
    double g = p.gate_is_alpha ? log((double)gate) : (double)gate;
    const bool bad = !(g <= 0.0) || !(beta >= 0.f && beta <= 1.f);
    if (g < kMinLog) g = kMinLog;
    double G = g;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(G, off, kWave);
        if (lane >= off) G += o;
    }
    const double Gc = __shfl(G, 63, kWave);
    gs.G[lane] = G;
    gs.gamma[lane] = expf((float)G);
    gs.tail[lane] = expf((float)(Gc - G));
    gs.beta[lane] = beta;
    gs.gate[lane] = gate;
    return bad;
}
__device__ __forceinline__ float decay(const Gates& gs, int r, int s) { return expf((float)(gs.G[r] - gs.G[s])); }

// A 64-token block of q or k: thread blocks of 4 tokens x 4 columns.
template <typename T, int DK>
struct Block64 {
    static constexpr int NB = (16 * (DK / 4) + 255) / 256;
    float4 x[NB][4];
    __device__ __forceinline__ int load(const T* base, long ld, int n, int d, bool vec) {
        int m = 0;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int id = threadIdx.x + 256 * i, cb = id % (DK / 4), rb = id / (DK / 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = 4 * rb + j;
                x[i][j] = t < n && rb < 16 ? row4<T>(base + t * ld + 4 * cb, d - 4 * cb, vec) : float4{0, 0, 0, 0};
                m = max(m, max(max(bits_abs(x[i][j].x), bits_abs(x[i][j].y)),
                               max(bits_abs(x[i][j].z), bits_abs(x[i][j].w))));
            }
        }
        return m;
    }
    // rows (token; column) and / or columns (column; token) as units, times s
    template <class Op>
    __device__ __forceinline__ void put_rows(const LdsMat<Op, DK / (16 * Op::kBlocks)>& a, float s) const {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int id = threadIdx.x + 256 * i, cb = id % (DK / 4), rb = id / (DK / 4);
            if (rb >= 16) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4& y = x[i][j];
                a.put4(4 * rb + j, 4 * cb, y.x * s, y.y * s, y.z * s, y.w * s);
            }
        }
    }
    template <class Op>
    __device__ __forceinline__ void put_cols(const LdsMat<Op, 64 / (16 * Op::kBlocks)>& a, float s) const {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int id = threadIdx.x + 256 * i, cb = id % (DK / 4), rb = id / (DK / 4);
            if (rb >= 16) break;
            const float4 *y = x[i];
            a.put4(4 * cb + 0, 4 * rb, y[0].x * s, y[1].x * s, y[2].x * s, y[3].x * s);
            a.put4(4 * cb + 1, 4 * rb, y[0].y * s, y[1].y * s, y[2].y * s, y[3].y * s);
            a.put4(4 * cb + 2, 4 * rb, y[0].z * s, y[1].z * s, y[2].z * s, y[3].z * s);
            a.put4(4 * cb + 3, 4 * rb, y[0].w * s, y[1].w * s, y[2].w * s, y[3].w * s);
        }
    }
};

// ----------------------------------------------------------------- prep
// One (chunk, head) per workgroup of four waves.  LDS: K by rows (then T in
// fp32), K by columns, Q by rows (then by columns), L diag(beta) in fp32 (then
// T^T diag(beta) P^T), P (then each wave's tile of V or dO).
template <class Op, int DK>
struct PrepLds {
    static constexpr int kRow = 64 * DK * int(sizeof(typename Op::Elt));
    static constexpr int kSq = 64 * 64 * 4;
    static constexpr int kKr = 0;
    static constexpr int kKt = kKr + (kRow > kSq ? kRow : kSq);  // T lies where K's rows were
    static constexpr int kQr = kKt + kRow;
    static constexpr int kA = kQr + kRow;
    static constexpr int kP = kA + kSq;
    static constexpr int kGates = kP + 64 * 64 * int(sizeof(typename Op::Elt));
    static constexpr int kMisc = kGates + int(sizeof(Gates));
    static constexpr int kBytes = kMisc + 64;
};

template <class Op, typename T, int DK>
__device__ __forceinline__ void prep_chunk(const BwdParams& p, const ChunkAt& at, int h, char* rec, char* lds) {
    using Unit = typename Op::Unit;
    using L = PrepLds<Op, DK>;
    constexpr int NT = DK / 16, NKK = NT / Op::kBlocks, NKT = 4 / Op::kBlocks, NBK = Op::kBlocks;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, m = lane & 15;
    const LdsMat<Op, NKK> Kr{lds + L::kKr}, Qr{lds + L::kQr};
    const LdsMat<Op, NKT> Kt{lds + L::kKt}, Qt{lds + L::kQr}, Pm{lds + L::kP}, Bo{lds + L::kA};
    float* Af = reinterpret_cast<float*>(lds + L::kA);
    float* Tf = reinterpret_cast<float*>(lds + L::kKr);
    Gates& gs = *reinterpret_cast<Gates*>(lds + L::kGates);
    int* misc = reinterpret_cast<int*>(lds + L::kMisc);  // maxima of K, Q by wave; [8] outside the domain
    float* vec = reinterpret_cast<float*>(rec + p.rec.vec);
    int* exps = reinterpret_cast<int*>(vec);

    const long ldk = (long)p.heads * p.d_k, ldv = (long)p.heads * p.d_v;
    const T* kp = static_cast<const T*>(p.k) + at.t0 * ldk + (long)h * p.d_k;
    const T* qp = static_cast<const T*>(p.q) + at.t0 * ldk + (long)h * p.d_k;
    Block64<T, DK> kb, qb;
    const int mk = kb.load(kp, ldk, at.n, p.d_k, p.vec_k), mq = qb.load(qp, ldk, at.n, p.d_k, p.vec_k);
    bool bad = false;
    if (wave == 0) bad = load_gates(p, at, h, gs, lane);
    int ek = 0, eq = 0;
    if constexpr (Op::kScaled) {
        const int wk = wave_max_bits(mk), wq = wave_max_bits(mq);
        if (lane == 0) {
            misc[wave] = wk;
            misc[4 + wave] = wq;
        }
        if (tid == 0) misc[8] = 0;
    }
    __syncthreads();
    if constexpr (Op::kScaled) {
        const int bk = max(max(misc[0], misc[1]), max(misc[2], misc[3]));
        const int bq = max(max(misc[4], misc[5]), max(misc[6], misc[7]));
        ek = tile_exp(bk, 0);
        eq = tile_exp(bq, 0);
        bad = bad || bk >= 0x7f800000 || bq >= 0x7f800000;
    }
    const float sk = exp2i(-ek), sq = exp2i(-eq);
    kb.template put_rows<Op>(Kr, sk);
    kb.template put_cols<Op>(Kt, sk);
    qb.template put_rows<Op>(Qr, sq);
    if (tid < 64) {
        vec[kVecGamma + tid] = gs.gamma[tid];
        vec[kVecWrite + tid] = gs.beta[tid] * gs.tail[tid];
    }
    if (tid == 0) {
        vec[kVecGc] = gs.gamma[63];
        exps[kVecEK] = ek;
        exps[kVecEQ] = eq;
    }
    __syncthreads();

    // L diag(beta) (fp32) and P (scaled as K and Q are): tile pairs over the waves
    const float kk2 = exp2i(2 * ek);
#pragma unroll 1
    for (int id = wave; id < 16; id += 4) {
        const int mt = id >> 2, nt = id & 3;  // rows, columns
        if (nt <= mt) {
            f32x4 c = {0, 0, 0, 0};
#pragma unroll
            for (int ku = 0; ku < NKK; ++ku) c = Op::mma(Kr.unit(mt, ku, lane), Kr.unit(nt, ku, lane), c);
            const int s = 16 * nt + m;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * mt + 4 * g + i;
                const float kk = c[i] * kk2;
                if (Op::kScaled && r == s && !(kk <= 1.03125f)) bad = true;
                Af[sq_at(r, s)] = s < r ? kk * decay(gs, r, s) * gs.beta[s] : 0.f;
            }
        }
        // P by rows s of q, contraction over rows j of k: tile (j = mt, s = nt)
        f32x4 c = {0, 0, 0, 0};
        if (mt <= nt) {
#pragma unroll
            for (int ku = 0; ku < NKK; ++ku) c = Op::mma(Kr.unit(mt, ku, lane), Qr.unit(nt, ku, lane), c);
        }
        const int s = 16 * nt + m;
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = 16 * mt + 4 * g + i;
            x[i] = j <= s ? c[i] * decay(gs, s, j) : 0.f;
        }
        Pm.put4(s, 16 * mt + 4 * g, x[0], x[1], x[2], x[3]);
    }
    if constexpr (Op::kScaled)
        if (bad) misc[8] = 1;
    __syncthreads();

    // T's diagonal blocks by forward substitution, column m of block `wave`
    // in lane (., m); Q by columns meanwhile
    f32x4 tc[4];  // block column `wave` of T as accumulator tiles
    {
        float t[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float x = i == m ? 1.f : 0.f;
#pragma unroll
            for (int s4 = 0; s4 < (i + 3) / 4; ++s4) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(Af + sq_at(16 * wave + i, 16 * wave + 4 * s4));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (4 * s4 + e < i) x -= a[e] * t[4 * s4 + e];
            }
            t[i] = x;
        }
        f32x4 d;
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = g == 0 ? t[i] : g == 1 ? t[4 + i] : g == 2 ? t[8 + i] : t[12 + i];
#pragma unroll
        for (int b = 0; b < 4; ++b) tc[b] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < 4; ++b)
            if (b == wave) tc[b] = d;
        // T overwrites K's rows, whose last readers passed the barrier
#pragma unroll
        for (int b = 0; b < 4; ++b)
            if (b <= wave)  // the blocks above the diagonal are zero
#pragma unroll
                for (int i = 0; i < 4; ++i) Tf[sq_at(16 * b + 4 * g + i, 16 * wave + m)] = tc[b][i];
    }
    qb.template put_cols<Op>(Qt, sq);
    __syncthreads();
    // T_iw = -T_ii sum_{w <= b < i} A_ib T_bw down block column w, in fp32
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        if (i > wave) {
            f32x4 y = {0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < i; ++b)
                if (b >= wave)
                    y = OpF32::mma(*reinterpret_cast<const f32x4*>(Af + sq_at(16 * i + m, 16 * b + 4 * g)), tc[b], y);
            f32x4 z = {0, 0, 0, 0};
            z = OpF32::mma(*reinterpret_cast<const f32x4*>(Tf + sq_at(16 * i + m, 16 * i + 4 * g)), y, z);
            tc[i] = -z;
        }
    }
#pragma unroll
    for (int i = 1; i < 4; ++i)
        if (i > wave)
#pragma unroll
            for (int e = 0; e < 4; ++e) Tf[sq_at(16 * i + 4 * g + e, 16 * wave + m)] = tc[i][e];
    __syncthreads();

    // right operands of token tile `wave`: T's rows times gamma, T's columns
    // times beta (and tail)
    {
        Unit ub[NKT];
        const int r = 16 * wave + m;
#pragma unroll
        for (int ku = 0; ku < NKT; ++ku) {
            f32x4 t[NBK];
#pragma unroll
            for (int b = 0; b < NBK; ++b) {
                const int s = 16 * (ku * NBK + b) + 4 * g;
                t[b] = *reinterpret_cast<const f32x4*>(Tf + sq_at(r, s));
#pragma unroll
                for (int e = 0; e < 4; ++e) t[b][e] *= gs.gamma[s + e];
            }
            ub[ku] = Op::pack(t, 1.f);
        }
        Unit* out = reinterpret_cast<Unit*>(rec + p.rec.wk);
        auto times_k = [&] {
#pragma unroll
            for (int u = 0; u < NKK; ++u) {
                f32x4 c[NBK];
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
                    c[b] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int ku = 0; ku < NKT; ++ku) c[b] = Op::mma(Kt.unit(u * NBK + b, ku, lane), ub[ku], c[b]);
                }
                out[(wave * NKK + u) * 64 + lane] = Op::pack(c, 1.f);
            }
        };
        times_k();
        Unit uo[NKT];
#pragma unroll
        for (int ku = 0; ku < NKT; ++ku) {
            f32x4 t[NBK], o[NBK];
#pragma unroll
            for (int b = 0; b < NBK; ++b) {
                const int j = 16 * (ku * NBK + b) + 4 * g;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[b][e] = Tf[sq_at(j + e, r)] * gs.beta[j + e];
                    t[b][e] = o[b][e] * gs.tail[j + e];
                }
            }
            ub[ku] = Op::pack(t, 1.f);
            uo[ku] = Op::pack(o, 1.f);
        }
        out = reinterpret_cast<Unit*>(rec + p.rec.kd);
        times_k();
        // T^T diag(beta) P^T, rows of tile `wave`
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            f32x4 c = {0, 0, 0, 0};
#pragma unroll
            for (int ku = 0; ku < NKT; ++ku) c = Op::mma(Pm.unit(mt, ku, lane), uo[ku], c);
            Bo.put4(r, 16 * mt + 4 * g, c[0], c[1], c[2], c[3]);
        }
        Unit* okt = reinterpret_cast<Unit*>(rec + p.rec.kt);
        Unit* oqt = reinterpret_cast<Unit*>(rec + p.rec.qt);
        for (int mt = wave; mt < NT; mt += 4)
#pragma unroll
            for (int ku = 0; ku < NKT; ++ku) {
                okt[(mt * NKT + ku) * 64 + lane] = Kt.unit(mt, ku, lane);
                oqt[(mt * NKT + ku) * 64 + lane] = Qt.unit(mt, ku, lane);
            }
    }
    Unit ta[4][NKT];  // T by rows, left operand
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int ku = 0; ku < NKT; ++ku) {
            f32x4 t[NBK];
#pragma unroll
            for (int b = 0; b < NBK; ++b)
                t[b] = *reinterpret_cast<const f32x4*>(Tf + sq_at(16 * mt + m, 16 * (ku * NBK + b) + 4 * g));
            ta[mt][ku] = Op::pack(t, 1.f);
        }
    __syncthreads();

    // T V and T^T diag(beta) P^T dO by 16-column tiles of d_v, one wave each
    const LdsMat<Op, NKT> st{lds + L::kP + wave * (NKT * 1024)};
    const T* vp = static_cast<const T*>(p.v) + at.t0 * ldv + (long)h * p.d_v;
    const T* op = static_cast<const T*>(p.dout) + at.t0 * ldv + (long)h * p.d_v;
    const int rb = lane >> 2, cb = lane & 3;
    bool bad_v = false;
    for (int tile = wave; tile < p.dvt; tile += 4) {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const T* src = which ? op : vp;
            float4 y[4];
            int mx = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = 4 * rb + j, c = 16 * tile + 4 * cb;
                y[j] = t < at.n ? row4<T>(src + t * ldv + c, p.d_v - c, p.vec_v) : float4{0, 0, 0, 0};
                mx = max(mx, max(max(bits_abs(y[j].x), bits_abs(y[j].y)), max(bits_abs(y[j].z), bits_abs(y[j].w))));
            }
            float s = 1.f;
            if constexpr (Op::kScaled) {
                const int bits = wave_max_bits(mx), e = tile_exp(bits, -2);
                bad_v = bad_v || bits >= 0x7f800000;
                s = exp2i(-e);
                if (lane == 0) exps[(which ? kExpO : kExpV) + tile] = e;
            }
            st.put4(4 * cb + 0, 4 * rb, y[0].x * s, y[1].x * s, y[2].x * s, y[3].x * s);
            st.put4(4 * cb + 1, 4 * rb, y[0].y * s, y[1].y * s, y[2].y * s, y[3].y * s);
            st.put4(4 * cb + 2, 4 * rb, y[0].z * s, y[1].z * s, y[2].z * s, y[3].z * s);
            st.put4(4 * cb + 3, 4 * rb, y[0].w * s, y[1].w * s, y[2].w * s, y[3].w * s);
            __builtin_amdgcn_wave_barrier();
            Unit ub[NKT];
#pragma unroll
            for (int ku = 0; ku < NKT; ++ku) ub[ku] = st.unit(0, ku, lane);
            __builtin_amdgcn_wave_barrier();
            Unit* o = reinterpret_cast<Unit*>(rec + (which ? p.rec.ot : p.rec.wt)) + (long)tile * NKT * 64;
#pragma unroll
            for (int u = 0; u < NKT; ++u) {
                f32x4 c[NBK];
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
                    const int mt = u * NBK + b;
                    c[b] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int ku = 0; ku < NKT; ++ku)
                        c[b] = Op::mma(which ? Bo.unit(mt, ku, lane) : ta[mt][ku], ub[ku], c[b]);
                }
                o[u * 64 + lane] = Op::pack(c, 1.f);
            }
            if (which) {
                Unit* od = reinterpret_cast<Unit*>(rec + p.rec.dot) + (long)tile * NKT * 64;
#pragma unroll
                for (int ku = 0; ku < NKT; ++ku) od[ku * 64 + lane] = ub[ku];
            }
        }
    }
    if constexpr (Op::kScaled) {
        if (bad_v) misc[8] = 1;
        __syncthreads();
        if (tid == 0) exps[kVecBad] = misc[8];
    }
}

template <class Op, typename T, int DK>
__global__ __launch_bounds__(256) void bwd_prep_kernel(BwdParams p) {
    __shared__ __align__(16) char lds[PrepLds<Op, DK>::kBytes];
    const int ci = blockIdx.x / p.heads, h = blockIdx.x - ci * p.heads;
    ChunkAt at;
    if (!find_chunk(p, ci, at)) return;
    prep_chunk<Op, T, DK>(p, at, h, p.ws + (size_t)blockIdx.x * p.rec.bytes, lds);
}

// ----------------------------------------------------------------- scan
// One wave carries 16 rows of S (or of dS) along a sequence's chunks in
// accumulators: tile b holds d_k indices 16 b + 4 g .. + 3 of row m.  The
// operands come straight from the record's units, each 1 KiB read by a wave at
// once, and the state's own operands from its accumulators, so a wave needs no
// LDS and waits for no other.  A unit of the next chunk is read as soon as the
// present chunk's has been used.
template <class Op, int DK>
struct State {
    static constexpr int NT = DK / 16, NBK = Op::kBlocks, NU = NT / NBK;
    f32x4 s[NT];
    int e = 0;  // the state is s * 2^e

    __device__ __forceinline__ void load(const BwdParams& p, const float* base, int row, int g) {
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const int c = 16 * b + 4 * g;
            float4 x = {0, 0, 0, 0};
            if (base && row < p.d_v) x = row4<float>(base + (long)row * p.d_k + c, p.d_k - c, p.vec_s);
            s[b] = f32x4{x.x, x.y, x.z, x.w};
        }
    }
    __device__ __forceinline__ void store(const BwdParams& p, float* base, int row, int g) const {
        if (row >= p.d_v) return;
        const float f = exp2i(e);
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const int c = 16 * b + 4 * g;
            put_row4<float>(base + (long)row * p.d_k + c, p.d_k - c, p.vec_s, s[b][0] * f, s[b][1] * f, s[b][2] * f,
                            s[b][3] * f);
        }
    }
    // operand units of the state divided by 2^f; returns f, and through `top`
    // the exponent of its largest value
    __device__ __forceinline__ int operands(typename Op::Unit (&u)[NU], int& top) const {
        int f = 0;
        top = 0;
        float sc = 1.f;
        if constexpr (Op::kScaled) {
            float mx = 0.f;
#pragma unroll
            for (int b = 0; b < NT; ++b)
                mx = fmaxf(fmaxf(fmaxf(mx, fabsf(s[b][0])), fabsf(s[b][1])), fmaxf(fabsf(s[b][2]), fabsf(s[b][3])));
            top = tile_exp(bits_abs(wave_max(mx)), 0) + e;
            f = top - 11;
            sc = exp2i(e - f);
        }
#pragma unroll
        for (int i = 0; i < NU; ++i) u[i] = Op::pack(&s[i * NBK], sc);
        return f;
    }
};

template <class Op>
__device__ __forceinline__ int tokens_exp(const f32x4 (&w)[4], int to) {
    if constexpr (!Op::kScaled) return 0;
    float mx = 0.f;
#pragma unroll
    for (int b = 0; b < 4; ++b)
        mx = fmaxf(fmaxf(fmaxf(mx, fabsf(w[b][0])), fabsf(w[b][1])), fmaxf(fabsf(w[b][2]), fabsf(w[b][3])));
    return tile_exp(bits_abs(wave_max(mx)), to);
}

template <class Op, int NMT, int NKU>
__device__ __forceinline__ void load_units(typename Op::Unit (&u)[NMT][NKU], const char* base, int lane) {
    const typename Op::Unit* b = reinterpret_cast<const typename Op::Unit*>(base) + lane;
#pragma unroll
    for (int i = 0; i < NMT; ++i)
#pragma unroll
        for (int k = 0; k < NKU; ++k) u[i][k] = b[(i * NKU + k) * 64];
}

// a vector of 64 by tokens, as the accumulators' rows hold them
__device__ __forceinline__ void load_tokens(f32x4 (&x)[4], const float* v, int g) {
#pragma unroll
    for (int b = 0; b < 4; ++b) x[b] = *reinterpret_cast<const f32x4*>(v + 16 * b + 4 * g);
}

// what a scan reads of a chunk once for the whole wave: gamma_c and the
// exponents of K, Q and of the wave's tile
struct ChunkScalars {
    float gc;
    int ek, eq, et;
};
template <class Op>
__device__ __forceinline__ ChunkScalars chunk_scalars(const BwdParams& p, const char* rec, int at) {
    const float* vec = reinterpret_cast<const float*>(rec + p.rec.vec);
    const int* exps = reinterpret_cast<const int*>(vec);
    if constexpr (Op::kScaled) return {vec[kVecGc], exps[kVecEK], exps[kVecEQ], exps[at]};
    return {vec[kVecGc], 0, 0, 0};
}

// W and the next state: W = T V - (T diag(gamma) K) S0^T, S1 = gamma_c S0 + (beta tail W)^T K.
template <class Op, int DK>
__device__ __forceinline__ void scan_forward(const BwdParams& p, State<Op, DK>& S, char* rec, size_t stride, int nc,
                                             int tile, int lane) {
    using Unit = typename Op::Unit;
    constexpr int NT = DK / 16, NBK = Op::kBlocks, NU = NT / NBK, NKT = 4 / NBK;
    const int g = lane >> 4;
    if (nc == 0) return;
    Unit wk[4][NU], kt[NT][NKT], wt[1][NKT];
    f32x4 wr[4];
    load_units<Op>(wk, rec + p.rec.wk, lane);
    load_units<Op>(wt, rec + p.rec.wt + (size_t)tile * NKT * 1024, lane);
    load_tokens(wr, reinterpret_cast<const float*>(rec + p.rec.vec) + kVecWrite, g);
    if constexpr (Op::kScaled) load_units<Op>(kt, rec + p.rec.kt, lane);
    ChunkScalars sc = chunk_scalars<Op>(p, rec, kExpV + tile);
    for (int c = 0; c < nc; ++c) {
        char* next = rec + (c + 1 < nc ? stride : 0);  // the last chunk reads its own again
        const float gc = sc.gc;
        const int ek = sc.ek, ev = sc.et;
        sc = chunk_scalars<Op>(p, next, kExpV + tile);
        if constexpr (!Op::kScaled) load_units<Op>(kt, rec + p.rec.kt, lane);
        Unit su[NU];
        int top;
        const int f = S.operands(su, top);
        Unit* os = reinterpret_cast<Unit*>(rec + p.rec.s0) + (size_t)tile * NU * 64 + lane;
#pragma unroll
        for (int i = 0; i < NU; ++i) os[i * 64] = su[i];
        f32x4 x[4], w[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) x[b] = Op::mma(wk[b][i], su[i], x[b]);
#pragma unroll
        for (int u = 0; u < NKT; ++u) Op::unpack(wt[0][u], &w[u * NBK]);
        const float sv = exp2i(ev), sx = exp2i(f + ek);
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[b][i] = w[b][i] * sv - x[b][i] * sx;
        load_units<Op>(wk, next + p.rec.wk, lane);
        load_units<Op>(wt, next + p.rec.wt + (size_t)tile * NKT * 1024, lane);
        const int ew = tokens_exp<Op>(w, 3);
        const float si = exp2i(-ew);
        Unit* ow = reinterpret_cast<Unit*>(rec + p.rec.wt) + (size_t)tile * NKT * 64 + lane;
#pragma unroll
        for (int u = 0; u < NKT; ++u) ow[u * 64] = Op::pack(&w[u * NBK], si);
        if (Op::kScaled && lane == 0) {
            int* oe = reinterpret_cast<int*>(rec + p.rec.vec);
            oe[kExpW + tile] = ew;
            oe[kExpS + tile] = f;
        }
        // the next state in units of 2^e: those of the larger of what stays
        // (gamma_c S0) and what is written; the operand's largest value stays
        // below 2^12
        int e = 0;
        if constexpr (Op::kScaled) e = max(ew + 3 + ek, top + tile_exp(bits_abs(gc), 0)) - 11;
        const float sw = exp2i(ek - e), sg = gc * exp2i(S.e - e);
        S.e = e;
        Unit wu[NKT];
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[b][i] *= wr[b][i];
#pragma unroll
        for (int u = 0; u < NKT; ++u) wu[u] = Op::pack(&w[u * NBK], sw);
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) S.s[b][i] *= sg;
#pragma unroll
        for (int u = 0; u < NKT; ++u)
#pragma unroll
            for (int b = 0; b < NT; ++b) S.s[b] = Op::mma(kt[b][u], wu[u], S.s[b]);
        if constexpr (Op::kScaled) load_units<Op>(kt, next + p.rec.kt, lane);
        load_tokens(wr, reinterpret_cast<const float*>(next + p.rec.vec) + kVecWrite, g);
        rec = next;
    }
}

// dX and the previous state's gradient: dX = T^T diag(beta) (P^T dO + diag(tail)
// K dS1^T), dS0 = gamma_c dS1 + (gamma dO)^T Q - (gamma dX)^T K.
template <class Op, int DK>
__device__ __forceinline__ void scan_backward(const BwdParams& p, State<Op, DK>& S, char* rec, size_t stride, int nc,
                                              int tile, int lane) {
    using Unit = typename Op::Unit;
    constexpr int NT = DK / 16, NBK = Op::kBlocks, NU = NT / NBK, NKT = 4 / NBK;
    const int g = lane >> 4;
    if (nc == 0) return;
    rec += (size_t)(nc - 1) * stride;
    Unit kd[4][NU], kt[NT][NKT], qt[NT][NKT], ot[1][NKT], dt[1][NKT];
    f32x4 ga[4];
    load_units<Op>(kd, rec + p.rec.kd, lane);
    load_units<Op>(ot, rec + p.rec.ot + (size_t)tile * NKT * 1024, lane);
    load_units<Op>(dt, rec + p.rec.dot + (size_t)tile * NKT * 1024, lane);
    load_tokens(ga, reinterpret_cast<const float*>(rec + p.rec.vec) + kVecGamma, g);
    if constexpr (Op::kScaled) {
        load_units<Op>(kt, rec + p.rec.kt, lane);
        load_units<Op>(qt, rec + p.rec.qt, lane);
    }
    ChunkScalars sc = chunk_scalars<Op>(p, rec, kExpO + tile);
    for (int c = nc - 1; c >= 0; --c) {
        char* next = rec - (c > 0 ? stride : 0);
        const float gc = sc.gc;
        const int ek = sc.ek, eq = sc.eq, eo = sc.et;
        sc = chunk_scalars<Op>(p, next, kExpO + tile);
        Unit su[NU];
        int top;
        const int f = S.operands(su, top);
        Unit* os = reinterpret_cast<Unit*>(rec + p.rec.ds1) + (size_t)tile * NU * 64 + lane;
#pragma unroll
        for (int i = 0; i < NU; ++i) os[i * 64] = su[i];
        f32x4 x[4], w[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) x[b] = Op::mma(kd[b][i], su[i], x[b]);
#pragma unroll
        for (int u = 0; u < NKT; ++u) Op::unpack(ot[0][u], &w[u * NBK]);
        const float so = exp2i(eo + ek + eq), sx = exp2i(f + ek);
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[b][i] = w[b][i] * so + x[b][i] * sx;
        load_units<Op>(kd, next + p.rec.kd, lane);
        load_units<Op>(ot, next + p.rec.ot + (size_t)tile * NKT * 1024, lane);
        const int ew = tokens_exp<Op>(w, -2);
        const float si = exp2i(-ew);
        Unit* ow = reinterpret_cast<Unit*>(rec + p.rec.ot) + (size_t)tile * NKT * 64 + lane;
#pragma unroll
        for (int u = 0; u < NKT; ++u) ow[u * 64] = Op::pack(&w[u * NBK], si);
        if (Op::kScaled && lane == 0) {
            int* oe = reinterpret_cast<int*>(rec + p.rec.vec);
            oe[kExpX + tile] = ew;
            oe[kExpD + tile] = f;
        }
        int e = 0;
        if constexpr (Op::kScaled)
            e = max(max(ew - 2 + ek, eo - 2 + eq), top + tile_exp(bits_abs(gc), 0)) - 11;
        const float sw = -exp2i(ek - e), sd = exp2i(eo + eq - e), sg = gc * exp2i(S.e - e);
        S.e = e;
        Unit wu[NKT], du[NKT];
#pragma unroll
        for (int u = 0; u < NKT; ++u) {
            f32x4 d[NBK];
            Op::unpack(dt[0][u], d);
#pragma unroll
            for (int b = 0; b < NBK; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    d[b][i] *= ga[u * NBK + b][i];
                    w[u * NBK + b][i] *= ga[u * NBK + b][i];
                }
            wu[u] = Op::pack(&w[u * NBK], sw);
            du[u] = Op::pack(d, sd);
        }
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) S.s[b][i] *= sg;
        if constexpr (!Op::kScaled) load_units<Op>(qt, rec + p.rec.qt, lane);
#pragma unroll
        for (int u = 0; u < NKT; ++u)
#pragma unroll
            for (int b = 0; b < NT; ++b) S.s[b] = Op::mma(qt[b][u], du[u], S.s[b]);
        if constexpr (!Op::kScaled) load_units<Op>(kt, rec + p.rec.kt, lane);
#pragma unroll
        for (int u = 0; u < NKT; ++u)
#pragma unroll
            for (int b = 0; b < NT; ++b) S.s[b] = Op::mma(kt[b][u], wu[u], S.s[b]);
        if constexpr (Op::kScaled) {
            load_units<Op>(kt, next + p.rec.kt, lane);
            load_units<Op>(qt, next + p.rec.qt, lane);
        }
        load_units<Op>(dt, next + p.rec.dot + (size_t)tile * NKT * 1024, lane);
        load_tokens(ga, reinterpret_cast<const float*>(next + p.rec.vec) + kVecGamma, g);
        rec = next;
    }
}

// Waves over (direction, d_v tile) of a (sequence, head); four to a workgroup.
template <class Op, int DK>
__global__ __launch_bounds__(256, 1) void bwd_scan_kernel(BwdParams p, int splits) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int id = blockIdx.x;
    const int part = id % splits;
    id /= splits;
    const bool back = id & 1;
    id >>= 1;
    const int seq = id / p.heads, h = id - seq * p.heads;
    const int tile = part * 4 + wave;
    if (tile >= p.dvt) return;
    int ci, nc;
    if (p.cu) {
        ci = p.chunk_base[seq];
        nc = p.chunk_base[seq + 1] - ci;
    } else {
        nc = (p.seq_len + C64 - 1) / C64;
        ci = seq * nc;
    }
    char* rec = p.ws + ((size_t)ci * p.heads + h) * p.rec.bytes;
    const size_t stride = (size_t)p.heads * p.rec.bytes;
    const long st = ((long)seq * p.heads + h) * p.d_v * p.d_k;
    const int row = 16 * tile + (lane & 15);
    State<Op, DK> S;
    if (!back) {
        S.load(p, p.init ? p.init + st : nullptr, row, lane >> 4);
        scan_forward<Op, DK>(p, S, rec, stride, nc, tile, lane);
    } else {
        S.load(p, p.dfinal ? p.dfinal + st : nullptr, row, lane >> 4);
        scan_backward<Op, DK>(p, S, rec, stride, nc, tile, lane);
        if (p.dinit) S.store(p, p.dinit + st, row, lane >> 4);
    }
}

// ----------------------------------------------------------------- grad
// One (chunk, head) per workgroup of four waves; wave w owns token tile w of
// every product.  Tiles of d_v (64 rows of S as fp16, 32 as fp32) pass through
// LDS, where S0, dS1, W and dX are turned so that d_v runs along the
// contraction; the products over d_v stay in accumulators (dO S0, dX S0, W dS1
// by d_k, dO W^T and dX W^T both ways round).  Then K and Q take the tiles'
// place and the 64 x 64 products follow, right operands from the accumulators.
template <class Op, int DK>
struct GradLds {
    static constexpr int kE = int(sizeof(typename Op::Elt));
    static constexpr int kTdv = 32 * Op::kBlocks;  // rows of S in a tile: two units along the contraction
    static constexpr int kSt = DK * kTdv * kE, kTok = 64 * kTdv * kE;
    static constexpr int kS0 = 0, kDs = kSt, kW = 2 * kSt, kX = kW + kTok, kO = kX + kTok, kTileEnd = kO + kTok;
    static constexpr int kRow = 64 * DK * kE, kSq = 64 * 64 * 4;
    static constexpr int kKr = 0, kQr = kRow;
    static constexpr int kKt = 2 * kRow > kSq ? 2 * kRow : kSq;  // the pair sums lie where K's and Q's rows were
    static constexpr int kQt = kKt + kRow, kKqEnd = kQt + kRow;
    static constexpr int kGates = kTileEnd > kKqEnd ? kTileEnd : kKqEnd;
    static constexpr int kVecs = kGates + int(sizeof(Gates));  // a [64], kw [64], partial sums [3][256], reductions [16]
    static constexpr int kBytes = kVecs + (128 + 768 + 16) * 4;
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float unit_dot(const f16x8& a, const f16x8& b) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        s = __builtin_amdgcn_fdot2(f16x2{a[2 * i], a[2 * i + 1]}, f16x2{b[2 * i], b[2 * i + 1]}, s, false);
    return s;
}
__device__ __forceinline__ float unit_dot(const f32x4& a, const f32x4& b) {
    return a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
}

// Four units of rows 4 mq .. 4 mq + 3 of a (row; column) tile written to LDS as (column; row).
template <class Op, int NKU>
__device__ __forceinline__ void put_turned(const LdsMat<Op, NKU>& a, const typename Op::Unit (&u)[4], int col, int row,
                                           float s) {
    if constexpr (Op::kScaled) {
        f16x8 x[4];
        const _Float16 f = (_Float16)s;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = u[j] * f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const f16x4 y = {x[0][e], x[1][e], x[2][e], x[3][e]};
            a.put4(col + (e >> 2) * 16 + (e & 3), row, __builtin_bit_cast(uint2, y));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) a.put4(col + e, row, u[0][e], u[1][e], u[2][e], u[3][e]);
    }
}

template <class Op, typename T, int DK>
__device__ __forceinline__ void grad_chunk(const BwdParams& p, const ChunkAt& at, int h, const char* rec,
                                           const char* s0, const char* ds1, char* lds) {
    using Unit = typename Op::Unit;
    using L = GradLds<Op, DK>;
    constexpr int NT = DK / 16, NBK = Op::kBlocks, NU = NT / NBK, NKT = 4 / NBK, NKD = 2, NDT = L::kTdv / 16;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, m = lane & 15;
    const LdsMat<Op, NKD> S0{lds + L::kS0}, Ds{lds + L::kDs}, W{lds + L::kW}, X{lds + L::kX}, O{lds + L::kO};
    const LdsMat<Op, NU> Kr{lds + L::kKr}, Qr{lds + L::kQr};
    const LdsMat<Op, NKT> Kt{lds + L::kKt}, Qt{lds + L::kQt};
    Gates& gs = *reinterpret_cast<Gates*>(lds + L::kGates);
    float* va = reinterpret_cast<float*>(lds + L::kVecs);  // a
    float* vk = va + 64;                                   // tail k.(W dS1)
    float* part = va + 128;                                // [3][256]
    float* red = part + 768;                               // [16]
    const int* exps = reinterpret_cast<const int*>(rec + p.rec.vec);

    const long ldk = (long)p.heads * p.d_k, ldv = (long)p.heads * p.d_v;
    const long ok = at.t0 * ldk + (long)h * p.d_k, ov = at.t0 * ldv + (long)h * p.d_v;
    if (wave == 0) load_gates(p, at, h, gs, lane);

    // one exponent for each matrix: its tiles' largest
    int eo = 0, ew = 0, ex = 0, es = 0, ed = 0, ek = 0, eq = 0;
    if constexpr (Op::kScaled) {
        auto top = [&](int a) {
            int x = lane < p.dvt ? exps[a + lane] : -1000;
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) x = max(x, __shfl_xor(x, off, kWave));
            return __builtin_amdgcn_readfirstlane(x);
        };
        eo = top(kExpO), ew = top(kExpW), ex = top(kExpX), es = top(kExpS), ed = top(kExpD);
        ek = exps[kVecEK], eq = exps[kVecEQ];
    }

    f32x4 zq[NT], zk[NT], zw[NT], e1a[4], e2a[4], e1b[4], e2b[4];
#pragma unroll
    for (int b = 0; b < NT; ++b) zq[b] = zk[b] = zw[b] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < 4; ++b) e1a[b] = e2a[b] = e1b[b] = e2b[b] = f32x4{0, 0, 0, 0};
    float ip = 0.f;  // <dS1, S0>

    const T* op = static_cast<const T*>(p.dout) + ov;
    T* dvp = static_cast<T*>(p.dv) + ov;
    const float so = exp2i(-eo), sx = exp2i(ex);
    for (int d0 = 0; d0 < p.dvt; d0 += NDT) {
        const int nd = min(NDT, p.dvt - d0);
        // S0 and dS1: quads of units, NDT tiles x NU units x 16 quads
#pragma unroll
        for (int i = 0; i < (NDT * NU * 16 + 255) / 256; ++i) {
            const int id = tid + 256 * i;
            if (id >= NDT * NU * 16) break;
            const int mt = id / (NU * 16), ku = (id >> 4) % NU, gg = (id >> 2) & 3, mq = id & 3;
            Unit a[4], b[4];
            float fa = 0.f, fb = 0.f;
            if (mt < nd) {
                const long at4 = ((long)(d0 + mt) * NU + ku) * 64 + gg * 16 + 4 * mq;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    a[j] = reinterpret_cast<const Unit*>(s0)[at4 + j];
                    b[j] = reinterpret_cast<const Unit*>(ds1)[at4 + j];
                }
                int xa = 0, xb = 0;
                if constexpr (Op::kScaled) xa = exps[kExpS + d0 + mt], xb = exps[kExpD + d0 + mt];
                float dot = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) dot += unit_dot(a[j], b[j]);
                ip += dot * exp2i(xa) * exp2i(xb);
                fa = exp2i(xa - es), fb = exp2i(xb - ed);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] = b[j] = Unit{};
            }
            const int col = 16 * ku * NBK + 4 * gg, row = 16 * mt + 4 * mq;
            put_turned<Op, NKD>(S0, a, col, row, fa);
            put_turned<Op, NKD>(Ds, b, col, row, fb);
        }
        // W and dX: NDT tiles x NKT units x 16 quads each
#pragma unroll
        for (int i = 0; i < (2 * NDT * NKT * 16 + 255) / 256; ++i) {
            const int id = tid + 256 * i;
            if (id >= 2 * NDT * NKT * 16) break;
            const bool isx = id >= NDT * NKT * 16;
            const int q = isx ? id - NDT * NKT * 16 : id;
            const int mt = q / (NKT * 16), ku = (q >> 4) % NKT, gg = (q >> 2) & 3, mq = q & 3;
            Unit a[4];
            float f = 0.f;
            if (mt < nd) {
                const long at4 = ((long)(d0 + mt) * NKT + ku) * 64 + gg * 16 + 4 * mq;
                const Unit* src = reinterpret_cast<const Unit*>(rec + (isx ? p.rec.ot : p.rec.wt));
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] = src[at4 + j];
                f = 1.f;
                if constexpr (Op::kScaled) f = exp2i(exps[(isx ? kExpX : kExpW) + d0 + mt] - (isx ? ex : ew));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] = Unit{};
            }
            put_turned<Op, NKD>(isx ? X : W, a, 16 * ku * NBK + 4 * gg, 16 * mt + 4 * mq, f);
        }
        // dO by rows
#pragma unroll
        for (int i = 0; i < 64 * (L::kTdv / 4) / 256; ++i) {
            const int id = tid + 256 * i, cb = id % (L::kTdv / 4), t = id / (L::kTdv / 4);
            const int c = 16 * d0 + 4 * cb;
            const float4 y = t < at.n ? row4<T>(op + t * ldv + c, p.d_v - c, p.vec_v) : float4{0, 0, 0, 0};
            O.put4(t, 4 * cb, y.x * so, y.y * so, y.z * so, y.w * so);
        }
        __syncthreads();
        // dV = dX
#pragma unroll
        for (int i = 0; i < 64 * (L::kTdv / 4) / 256; ++i) {
            const int id = tid + 256 * i, cb = id % (L::kTdv / 4), t = id / (L::kTdv / 4);
            const int c = 16 * d0 + 4 * cb;
            const f32x4 y = X.get4(t, 4 * cb);
            if (t < at.n)
                put_row4<T>(dvp + t * ldv + c, p.d_v - c, p.vec_v, y[0] * sx, y[1] * sx, y[2] * sx, y[3] * sx);
        }
#pragma unroll
        for (int ku = 0; ku < NKD; ++ku) {
            const Unit bo = O.unit(wave, ku, lane), bx = X.unit(wave, ku, lane), bw = W.unit(wave, ku, lane);
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                const Unit a = S0.unit(b, ku, lane);
                zq[b] = Op::mma(a, bo, zq[b]);
                zk[b] = Op::mma(a, bx, zk[b]);
                zw[b] = Op::mma(Ds.unit(b, ku, lane), bw, zw[b]);
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (b <= wave) {
                    const Unit a = W.unit(b, ku, lane);
                    e1a[b] = Op::mma(a, bo, e1a[b]);
                    e2a[b] = Op::mma(a, bx, e2a[b]);
                }
                if (b >= wave) {
                    e1b[b] = Op::mma(O.unit(b, ku, lane), bw, e1b[b]);
                    e2b[b] = Op::mma(X.unit(b, ku, lane), bw, e2b[b]);
                }
            }
        }
        __syncthreads();
    }

    // K and Q in both orders
    {
        Block64<T, DK> x;
        const float sk = exp2i(-ek), sq = exp2i(-eq);
        x.load(static_cast<const T*>(p.k) + ok, ldk, at.n, p.d_k, p.vec_k);
        x.template put_rows<Op>(Kr, sk);
        x.template put_cols<Op>(Kt, sk);
        x.load(static_cast<const T*>(p.q) + ok, ldk, at.n, p.d_k, p.vec_k);
        x.template put_rows<Op>(Qr, sq);
        x.template put_cols<Op>(Qt, sq);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) ip += __shfl_xor(ip, off, kWave);
    if (lane == 0) red[wave] = ip;
    __syncthreads();

    const int tok = 16 * wave + m;  // this lane's token as a column of the products
    const float gam = gs.gamma[tok], tail = gs.tail[tok], bet = gs.beta[tok];
    // q.(dO S0), k.(dX S0), k.(W dS1) of the lane's token; q.k and k.k with the tokens up to it
    float qz = 0.f, kz = 0.f, kwz = 0.f;
    f32x4 mh[4];  // rows r of tile b, column s = tok: dO_s.W_r q_s.k_r - dX_s.W_r k_s.k_r
    const float s1 = exp2i(eo + ew), s2 = exp2i(ex + ew);
    {
        Unit uk[NU], uq[NU];
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            uk[i] = Kr.unit(wave, i, lane);
            uq[i] = Qr.unit(wave, i, lane);
            f32x4 k[NBK], q[NBK];
            Op::unpack(uk[i], k);
            Op::unpack(uq[i], q);
#pragma unroll
            for (int b = 0; b < NBK; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    qz += q[b][j] * zq[i * NBK + b][j];
                    kz += k[b][j] * zk[i * NBK + b][j];
                    kwz += k[b][j] * zw[i * NBK + b][j];
                }
        }
        qz += __shfl_xor(qz, 16, kWave);
        kz += __shfl_xor(kz, 16, kWave);
        kwz += __shfl_xor(kwz, 16, kWave);
        qz += __shfl_xor(qz, 32, kWave);
        kz += __shfl_xor(kz, 32, kWave);
        kwz += __shfl_xor(kwz, 32, kWave);
        const float sqk = exp2i(eq + ek) * s1, skk = exp2i(2 * ek) * s2;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            f32x4 qk = {0, 0, 0, 0}, kk = {0, 0, 0, 0};
            if (b <= wave) {
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    const Unit a = Kr.unit(b, i, lane);
                    qk = Op::mma(a, uq[i], qk);
                    kk = Op::mma(a, uk[i], kk);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 16 * b + 4 * g + j;
                const float x1 = e1a[b][j] * qk[j] * sqk, x2 = e2a[b][j] * kk[j] * skk;
                mh[b][j] = r < tok ? x1 - x2 : r == tok ? x1 : 0.f;
            }
        }
    }
    const float ah = qz * exp2i(eo + es + eq) - kz * exp2i(ex + es + ek);  // a without gamma
    const float kwh = kwz * exp2i(ew + ed + ek);                          // k.(W dS1)
    if (g == 0) {
        va[tok] = gam * ah;
        vk[tok] = tail * kwh;
    }
    __syncthreads();  // K's and Q's rows are done with

    float* M = reinterpret_cast<float*>(lds + L::kKr);
    Unit n1[NKT], n2[NKT];
    {
        f32x4 x1[4], x2[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            f32x4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 16 * b + 4 * g + j;
                const float d = r <= tok ? decay(gs, tok, r) : 0.f;
                x1[b][j] = e1a[b][j] * d * gs.beta[r];
                x2[b][j] = r < tok ? e2a[b][j] * d * gs.beta[r] : 0.f;
                y[j] = mh[b][j] * d;
            }
            *reinterpret_cast<f32x4*>(M + sq_at(tok, 16 * b + 4 * g)) = y;
        }
#pragma unroll
        for (int u = 0; u < NKT; ++u) {
            n1[u] = Op::pack(&x1[u * NBK], 1.f);
            n2[u] = Op::pack(&x2[u * NBK], 1.f);
        }
    }
    // dQ = diag(gamma) dO S0 + N1 K;  K's share of dK: -N2 K - N2^T K
    const long orow = ok + tok * ldk;
    f32x4 ak[NT];
    {
        const float f1 = gam * exp2i(eo + es), f2 = s1 * exp2i(ek);
        T* dq = static_cast<T*>(p.dq) + orow;
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            f32x4 c = {0, 0, 0, 0};
            ak[b] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < NKT; ++u) {
                const Unit a = Kt.unit(b, u, lane);
                c = Op::mma(a, n1[u], c);
                ak[b] = Op::mma(a, n2[u], ak[b]);
            }
            const int col = 16 * b + 4 * g;
            if (tok < at.n)
                put_row4<T>(dq + col, p.d_k - col, p.vec_k, zq[b][0] * f1 + c[0] * f2, zq[b][1] * f1 + c[1] * f2,
                            zq[b][2] * f1 + c[2] * f2, zq[b][3] * f1 + c[3] * f2);
        }
    }
    {
        f32x4 x1[4], x2[4];  // rows s of tile b, column r = tok
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int s = 16 * b + 4 * g + j;
                const float d = s >= tok ? decay(gs, s, tok) * bet : 0.f;
                x1[b][j] = e1b[b][j] * d;
                x2[b][j] = s > tok ? e2b[b][j] * d : 0.f;
            }
#pragma unroll
        for (int u = 0; u < NKT; ++u) {
            n1[u] = Op::pack(&x1[u * NBK], 1.f);
            n2[u] = Op::pack(&x2[u * NBK], 1.f);
        }
        const float fk = -gam * exp2i(ex + es), fw = bet * tail * exp2i(ew + ed), fq = s1 * exp2i(eq),
                    fn = -s2 * exp2i(ek);
        T* dk = static_cast<T*>(p.dk) + orow;
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            f32x4 c = {0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < NKT; ++u) {
                c = Op::mma(Qt.unit(b, u, lane), n1[u], c);
                ak[b] = Op::mma(Kt.unit(b, u, lane), n2[u], ak[b]);
            }
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = zk[b][j] * fk + zw[b][j] * fw + c[j] * fq + ak[b][j] * fn;
            const int col = 16 * b + 4 * g;
            if (tok < at.n) put_row4<T>(dk + col, p.d_k - col, p.vec_k, y[0], y[1], y[2], y[3]);
        }
    }
    __syncthreads();

    // gates: column sums of M (dbeta), and for every t the sum of beta_r M_sr
    // over s >= t > r: prefix sums along the rows, then down the columns
    {
        const int t = lane, qu = wave;
        float cs = 0.f, rs = 0.f;
        f32x4 row[4];
#pragma unroll
        for (int i = 0; i < 16; ++i) cs += M[sq_at(16 * qu + i, t)];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            row[i] = *reinterpret_cast<const f32x4*>(M + sq_at(t, 16 * qu + 4 * i));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                row[i][j] *= gs.beta[16 * qu + 4 * i + j];
                rs += row[i][j];
            }
        }
        part[tid] = cs;
        part[256 + tid] = rs;
        __syncthreads();
        float run = 0.f;
#pragma unroll
        for (int w = 0; w < 3; ++w)
            if (w < qu) run += part[256 + 64 * w + t];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = run;
                run += row[i][j];
            }
            *reinterpret_cast<f32x4*>(M + sq_at(t, 16 * qu + 4 * i)) = o;
        }
        __syncthreads();
        float f = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int s = 16 * qu + i;
            const float x = M[sq_at(s, t)];
            f += s >= t ? x : 0.f;
        }
        part[512 + tid] = f;
        __syncthreads();
    }
    const float ipt = red[0] + red[1] + red[2] + red[3];
    T* dgate = static_cast<T*>(p.dgate) + (long)at.t0 * p.heads + h;
    if (tid < 64) {
        float a = va[tid], b = gs.beta[tid] * vk[tid];
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const float x = __shfl_down(a, off, kWave), y = __shfl_up(b, off, kWave);
            if (tid + off < 64) a += x;
            if (tid >= off) b += y;
        }
        b = __shfl_up(b, 1, kWave);  // over s < t, without t's own
        if (tid == 0) b = 0.f;
        const float* f = part + 512;
        float dg = gs.gamma[63] * ipt + a + b + (f[tid] + f[64 + tid] + f[128 + tid] + f[192 + tid]);
        const float db = vk[tid] + part[tid] + part[64 + tid] + part[128 + tid] + part[192 + tid];
        if (tid < at.n) {
            if (p.gate_is_alpha) dg /= gs.gate[tid];
            if (!(p.gate_is_alpha && gs.gate[tid] < kTinyAlpha)) Elem<T>::store(dgate, (long)tid * p.heads, dg);
            Elem<T>::store(static_cast<T*>(p.dbeta) + (long)at.t0 * p.heads + h, (long)tid * p.heads, db);
        }
    }
    if (!p.gate_is_alpha) return;
    // dalpha_t where alpha_t is zero or tiny: the same sum with alpha_t's factor left out
    for (int t = 0; t < at.n; ++t) {
        if (!(gs.gate[t] < kTinyAlpha)) continue;  // uniform
        const double gt = t ? gs.G[t - 1] - gs.G[t] : -gs.G[0];  // -ln alpha_t
        float x = 0.f;
        if (tok >= t) {
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 16 * b + 4 * g + j;
                    if (r < t) x += mh[b][j] * gs.beta[r] * expf((float)(gs.G[tok] - gs.G[r] + gt));
                }
            if (g == 0) x += ah * expf((float)(gs.G[tok] + gt));
        } else if (g == 0) {
            x += bet * kwh * expf((float)(gs.G[63] - gs.G[tok] + gt));
        }
        if (tid == 0) x += ipt * expf((float)(gs.G[63] + gt));
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, kWave);
        if (lane == 0) red[4 + wave] = x;
        __syncthreads();
        if (tid == 0) Elem<T>::store(dgate, (long)t * p.heads, red[4] + red[5] + red[6] + red[7]);
        __syncthreads();
    }
}

template <class Op, typename T, int DK>
__global__ __launch_bounds__(256) void bwd_grad_kernel(BwdParams p) {
    __shared__ __align__(16) char lds[GradLds<Op, DK>::kBytes];
    const int ci = blockIdx.x / p.heads, h = blockIdx.x - ci * p.heads;
    ChunkAt at;
    if (!find_chunk(p, ci, at)) return;
    const char* rec = p.ws + (size_t)blockIdx.x * p.rec.bytes;
    grad_chunk<Op, T, DK>(p, at, h, rec, rec + p.rec.s0, rec + p.rec.ds1, lds);
}

// ---------------------------------------------------------------- exact
// bf16 heads whose inputs leave the fp16 path's domain (a key with |k|^2 >
// 1.03125, beta or alpha outside [0, 1], a value that is not finite): the same
// steps in fp32, one workgroup per (sequence, head), after the others.  The
// states before the chunks are kept in fp32 where the records' S0 and dS1 were
// (the same bytes), and everything else of the present chunk in the
// workgroup's own scratch: a record of fp32 units and the state's gradient.
template <class Op, int DK>
__device__ __forceinline__ void load_state(State<Op, DK>& S, const char* base, int tile, int lane) {
    const f32x4* b = reinterpret_cast<const f32x4*>(base) + (size_t)tile * (DK / 16) * 64 + lane;
#pragma unroll
    for (int i = 0; i < DK / 16; ++i) S.s[i] = b[i * 64];
}
template <class Op, int DK>
__device__ __forceinline__ void store_state(const State<Op, DK>& S, char* base, int tile, int lane) {
    f32x4* b = reinterpret_cast<f32x4*>(base) + (size_t)tile * (DK / 16) * 64 + lane;
#pragma unroll
    for (int i = 0; i < DK / 16; ++i) b[i * 64] = S.s[i];
}
__host__ __device__ inline size_t exact_scratch(int DK, int dvt) {
    return rec_layout(DK, dvt, 4).bytes + (size_t)DK * dvt * 16 * 4;
}

template <typename T, int DK>
__global__ __launch_bounds__(256, 1) void bwd_exact_kernel(BwdParams p, char* scratch) {
    constexpr int kLds = PrepLds<OpF32, DK>::kBytes > GradLds<OpF32, DK>::kBytes ? PrepLds<OpF32, DK>::kBytes
                                                                                : GradLds<OpF32, DK>::kBytes;
    __shared__ __align__(16) char lds[kLds];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
    BwdParams e = p;
    e.rec = rec_layout(DK, p.dvt, 4);
    char* rec = scratch + blockIdx.x * exact_scratch(DK, p.dvt);
    char* carry = rec + e.rec.bytes;
    const size_t stride = (size_t)p.heads * p.rec.bytes;
    for (int unit = blockIdx.x; unit < p.batch * p.heads; unit += gridDim.x) {
        const int seq = unit / p.heads, h = unit - seq * p.heads;
        int ci, nc, t0, t1;
        seq_bounds(p.cu, seq, p.seq_len, t0, t1);
        if (p.cu) {
            ci = p.chunk_base[seq];
            nc = p.chunk_base[seq + 1] - ci;
        } else {
            nc = (p.seq_len + C64 - 1) / C64;
            ci = seq * nc;
        }
        char* first = p.ws + ((size_t)ci * p.heads + h) * p.rec.bytes;
        int bad = 0;
        for (int c = threadIdx.x; c < nc; c += 256)
            bad |= reinterpret_cast<const int*>(first + c * stride + p.rec.vec)[kVecBad];
        if (!__syncthreads_or(bad)) continue;
        const long st = (long)unit * p.d_v * p.d_k;
        auto chunk = [&](int c) {
            ChunkAt at;
            at.seq = seq;
            at.t0 = t0 + c * C64;
            at.n = min(C64, t1 - at.t0);
            return at;
        };
        for (int c = 0; c < nc; ++c) {
            prep_chunk<OpF32, T, DK>(e, chunk(c), h, rec, lds);
            __syncthreads();
            for (int tile = wave; tile < p.dvt; tile += 4) {
                char* kept = first + c * stride + p.rec.s0;
                State<OpF32, DK> S;
                if (c == 0) {
                    S.load(p, p.init ? p.init + st : nullptr, 16 * tile + row, g);
                    store_state(S, kept, tile, lane);
                } else {
                    load_state(S, kept, tile, lane);
                }
                if (c + 1 < nc) {
                    scan_forward<OpF32, DK>(e, S, rec, 0, 1, tile, lane);
                    store_state(S, kept + stride, tile, lane);
                }
            }
            __syncthreads();
        }
        for (int tile = wave; tile < p.dvt; tile += 4) {
            State<OpF32, DK> S;
            S.load(p, p.dfinal ? p.dfinal + st : nullptr, 16 * tile + row, g);
            store_state(S, carry, tile, lane);
        }
        for (int c = nc - 1; c >= 0; --c) {
            const char* kept = first + c * stride + p.rec.s0;
            prep_chunk<OpF32, T, DK>(e, chunk(c), h, rec, lds);
            __syncthreads();
            for (int tile = wave; tile < p.dvt; tile += 4) {
                State<OpF32, DK> S;
                load_state(S, kept, tile, lane);
                scan_forward<OpF32, DK>(e, S, rec, 0, 1, tile, lane);
                load_state(S, carry, tile, lane);
                scan_backward<OpF32, DK>(e, S, rec, 0, 1, tile, lane);
                store_state(S, carry, tile, lane);
            }
            __syncthreads();
            grad_chunk<OpF32, T, DK>(e, chunk(c), h, rec, rec + e.rec.s0, rec + e.rec.ds1, lds);
            __syncthreads();
        }
        if (p.dinit)
            for (int tile = wave; tile < p.dvt; tile += 4) {
                State<OpF32, DK> S;
                load_state(S, carry, tile, lane);
                S.store(p, p.dinit + st, 16 * tile + row, g);
            }
    }
}

// Chunks before each sequence of a pack: base[n] for n = 0 .. batch, at most
// `most` in all (overlapping sequences, from offsets that decrease, are cut).
__global__ __launch_bounds__(1024) void bwd_chunks_kernel(const int* cu, int batch, int seq_len, int most, int* base) {
    __shared__ long tops[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    long carry = 0;
    for (int n0 = 0; n0 < batch; n0 += 1024) {
        int x = 0;
        if (n0 + tid < batch) {
            int a, b;
            seq_bounds(cu, n0 + tid, seq_len, a, b);
            x = (b - a + C64 - 1) / C64;
        }
        long run = x;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const long y = __shfl_up(run, off, kWave);
            if (lane >= off) run += y;
        }
        if (lane == 63) tops[wave] = run;
        __syncthreads();
        long before = carry;
        for (int w = 0; w < wave; ++w) before += tops[w];
        long all = carry;
        for (int w = 0; w < 16; ++w) all += tops[w];
        if (n0 + tid < batch) base[n0 + tid + 1] = int(min(before + run, (long)most));
        carry = all;
        __syncthreads();
    }
    if (tid == 0) base[0] = 0;
}

// d_k padded to 32, 64 or 128
int padded_dk(int d_k) { return d_k <= 32 ? 32 : d_k <= 64 ? 64 : 128; }
int64_t chunks_of(const rhz_gdr_prefill_backward_args& a) {
    if (a.cu_seqlens) return (int64_t)a.seq_len / C64 + a.batch;
    return (int64_t)a.batch * (((int64_t)a.seq_len + C64 - 1) / C64);
}
int exact_blocks(const rhz_gdr_prefill_backward_args& a) {
    return int(std::min<int64_t>((int64_t)a.batch * a.heads, 256));
}
size_t base_bytes(const rhz_gdr_prefill_backward_args& a) {
    return a.cu_seqlens ? (((size_t)a.batch + 1) * 4 + 255) & ~(size_t)255 : 0;
}

template <class Op, typename T, int DK>
hipError_t go(const BwdParams& p, int64_t chunks, char* scratch, int blocks, hipStream_t st) {
    hipError_t e;
    const int64_t grid = chunks * p.heads;
    const int splits = (p.dvt + 3) / 4;
    const int64_t scans = (int64_t)p.batch * p.heads * 2 * splits;
    if ((e = check_grid(grid, 256)) != hipSuccess) return e;
    if ((e = check_grid(scans, 256)) != hipSuccess) return e;
    if (grid > 0) {
        hipLaunchKernelGGL((bwd_prep_kernel<Op, T, DK>), dim3((unsigned)grid), dim3(256), 0, st, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (grid > 0 || p.dinit) {
        hipLaunchKernelGGL((bwd_scan_kernel<Op, DK>), dim3((unsigned)scans), dim3(256), 0, st, p, splits);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (grid > 0) {
        hipLaunchKernelGGL((bwd_grad_kernel<Op, T, DK>), dim3((unsigned)grid), dim3(256), 0, st, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        if constexpr (Op::kScaled) {
            hipLaunchKernelGGL((bwd_exact_kernel<T, DK>), dim3(blocks), dim3(256), 0, st, p, scratch);
            e = hipGetLastError();
        }
    }
    return e;
}

template <class Op, typename T>
hipError_t pick_dk(const BwdParams& p, int64_t chunks, char* scratch, int blocks, hipStream_t st) {
    switch (padded_dk(p.d_k)) {
        case 32: return go<Op, T, 32>(p, chunks, scratch, blocks, st);
        case 64: return go<Op, T, 64>(p, chunks, scratch, blocks, st);
        default: return go<Op, T, 128>(p, chunks, scratch, blocks, st);
    }
}

int tiles_dv(int d_v) { return ((d_v + 31) / 32) * 2; }

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

size_t backward_workspace_bytes(const rhz_gdr_prefill_backward_args& a) {
    const int DK = padded_dk(a.d_k), dvt = tiles_dv(a.d_v), es = a.dtype == RHZ_F32 ? 4 : 2;
    size_t n = base_bytes(a) + (size_t)chunks_of(a) * a.heads * rec_layout(DK, dvt, es).bytes;
    if (a.dtype != RHZ_F32) n += (size_t)exact_blocks(a) * exact_scratch(DK, dvt);
    return n;
}

hipError_t launch_backward(const rhz_gdr_prefill_backward_args& a, hipStream_t st) {
    const int DK = padded_dk(a.d_k), es = a.dtype == RHZ_F32 ? 4 : 2;
    BwdParams p{};
    p.q = a.q;
    p.k = a.k;
    p.v = a.v;
    p.dout = a.grad_o;
    p.gate = a.gate;
    p.beta = a.beta;
    p.init = a.initial_state;
    p.dfinal = a.grad_final_state;
    p.cu = a.cu_seqlens;
    p.dq = a.grad_q;
    p.dk = a.grad_k;
    p.dv = a.grad_v;
    p.dgate = a.grad_gate;
    p.dbeta = a.grad_beta;
    p.dinit = a.grad_initial_state;
    p.batch = a.batch;
    p.seq_len = a.seq_len;
    p.heads = a.heads;
    p.d_k = a.d_k;
    p.d_v = a.d_v;
    p.dvt = tiles_dv(a.d_v);
    p.gate_is_alpha = a.gate_kind == RHZ_GATE_ALPHA;
    p.rec = rec_layout(DK, p.dvt, es);
    const size_t four = 4 * (size_t)es;
    p.vec_k = a.d_k % 4 == 0 && aligned(a.q, four) && aligned(a.k, four) && aligned(a.grad_q, four) &&
              aligned(a.grad_k, four);
    p.vec_v = a.d_v % 4 == 0 && aligned(a.v, four) && aligned(a.grad_o, four) && aligned(a.grad_v, four);
    p.vec_s = a.d_k % 4 == 0 && aligned(a.initial_state, 16) && aligned(a.grad_final_state, 16) &&
              aligned(a.grad_initial_state, 16);
    char* ws = static_cast<char*>(a.workspace);
    const int64_t chunks = chunks_of(a);
    p.ws = ws + base_bytes(a);
    char* scratch = p.ws + (size_t)chunks * a.heads * p.rec.bytes;
    if (a.cu_seqlens) {
        int* base = reinterpret_cast<int*>(ws);
        p.chunk_base = base;
        hipLaunchKernelGGL(bwd_chunks_kernel, dim3(1), dim3(1024), 0, st, a.cu_seqlens, a.batch, a.seq_len, (int)chunks,
                           base);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (a.dtype == RHZ_F32) return pick_dk<OpF32, float>(p, chunks, scratch, exact_blocks(a), st);
    return pick_dk<OpF16, uint16_t>(p, chunks, scratch, exact_blocks(a), st);
}

}  // namespace rhz
