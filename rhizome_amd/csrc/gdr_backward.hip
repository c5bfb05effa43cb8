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
// Kernels: bwd_prep_kernel forms what depends on one chunk's inputs alone (T and
// P) for every (chunk, head) at once; bwd_scan16_kernel (bf16) and
// bwd_scan32_kernel carry S and dS along the chunks, the two directions at the
// same time since neither needs the other; bwd_grad_kernel forms the gradients
// of every (chunk, head) at once from S0, dS1, W and dX.  What passes between
// them lies in the workspace: a chunk's S0 and dS1 are four times its K, and
// keeping them is what lets the last kernel, 3/4 of the products, run on all
// chunks at once.  4 x 4096 tokens, 16 heads, d = 128, bf16: 484 us, 1.9 GB of
// HBM traffic (the inputs and outputs alone: 0.47), 370 us at a copy's rate.
//
// bf16 tensors are multiplied as fp16 (11 significant bits) on MFMA with fp32
// accumulation: each fp16 operand is scaled by a power of two, from the largest
// magnitude of the tile it is rounded in (of V and dO) or of the chunk's factors
// that it is made of, so that the magnitude of the inputs (a loss's gradient of
// 1e-8, say) does not matter.  S, dS and every sum are fp32.  fp32 tensors are
// multiplied in fp32 throughout.

#include <algorithm>
#include <type_traits>

#include "gdr_device.hpp"
#include "gdr_internal.hpp"

namespace rhz {
namespace {

constexpr int C64 = kChunk;           // tokens of a chunk
constexpr double kMinLog = -1000.0;   // log-decays below it decay to 0 in fp32 all the same
constexpr float kTinyAlpha = 1e-18f;  // below: dalpha is formed without dividing by alpha

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// ------------------------------------------------------------- operands
// An MFMA operand is held in "units" of 16 bytes per lane.  Lane (g, m), g =
// lane / 16, m = lane % 16, holds for row m of a 16-row tile the contraction
// indices 16 b + 4 g .. + 3 of one (fp32) or two (fp16) blocks b.  An
// accumulator tile holds rows 4 g .. 4 g + 3 of column m, so accumulators are
// the units of the next product's right operand as they stand.
struct OpF16 {
    using Elt = _Float16;
    using Unit = f16x8;
    using Quad = f16x4;
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
    using Quad = f32x4;
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

template <class Op>
__device__ __forceinline__ typename Op::Unit lds_unit(const char* p, int i, int lane) {
    return reinterpret_cast<const typename Op::Unit*>(p)[i * 64 + lane];
}

// A matrix by rows in LDS.  A unit of it is read along its rows, or along its
// columns (fp16: ds_read_b64_tr_b16, which gives lane l of 16 the l-th column
// of four rows), so that one copy serves products over either index.  The
// 16-byte groups of a row are XORed by the row: of the lanes that LDS serves at
// once, 16 with 16 bytes or 32 with 8, none share a bank, whether they run down
// 16 rows or along eight rows' 32 bytes (padded rows served only one of the
// two: the bwd scan lost 1500 LDS cycles a chunk to the other).
template <class Op, int COLS>
struct RowMat {
    using Elt = typename Op::Elt;
    using Unit = typename Op::Unit;
    static constexpr int kStride = COLS * int(sizeof(Elt));
    static constexpr int bytes(int rows) { return rows * kStride; }
    char* p;
    static __device__ __forceinline__ int swizzle(int row) {  // in bytes
        constexpr int kSpan = kStride >= 256 ? 0 : kStride == 128 ? 1 : kStride == 64 ? 2 : 3;  // log2 rows per 64 banks
        static_assert(kStride >= 32, "");
        if constexpr (Op::kScaled)
            return (((row >> kSpan) & (COLS / 16 - 1)) << 5) | ((row & 8) << 1);
        else
            return ((row >> kSpan) & (COLS / 4 < 16 ? COLS / 4 - 1 : 15)) << 4;
    }
    __device__ __forceinline__ char* at(int row, int col) const {
        return p + row * kStride + ((col * int(sizeof(Elt))) ^ swizzle(row));
    }
    // a unit's 16 bytes of consecutive columns: an order of the contraction
    // that only another operand read this way shares
    __device__ __forceinline__ Unit run(int row0, int ku, int lane) const {
        return *reinterpret_cast<const Unit*>(at(row0 + (lane & 15), (ku * 4 + (lane >> 4)) * (16 / int(sizeof(Elt)))));
    }
    // the columns 16 b + 4 g .. of a unit's blocks, as accumulators hold them
    __device__ __forceinline__ Unit blocks(int row, int ku, int g) const {
        if constexpr (Op::kScaled) {
            const f16x4 a = *reinterpret_cast<const f16x4*>(at(row, 32 * ku + 4 * g));
            const f16x4 b = *reinterpret_cast<const f16x4*>(at(row, 32 * ku + 16 + 4 * g));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *reinterpret_cast<const Unit*>(at(row, 16 * ku + 4 * g));
        }
    }
    // column 16 ct + m, rows 16 rb + 4 g ..
    __device__ __forceinline__ typename Op::Quad col4(int ct, int rb, int lane) const {
        const int g = lane >> 4, m = lane & 15;
        if constexpr (Op::kScaled) {
            const char* a = at(16 * rb + 4 * g + (m >> 2), 16 * ct + 4 * (m & 3));
            return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a)));
        } else {
            f32x4 x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const float*>(at(16 * rb + 4 * g + j, 16 * ct + m));
            return x;
        }
    }
    __device__ __forceinline__ Unit cols(int ct, int ku, int lane) const {
        if constexpr (Op::kScaled)
            return __builtin_shufflevector(col4(ct, 2 * ku, lane), col4(ct, 2 * ku + 1, lane), 0, 1, 2, 3, 4, 5, 6, 7);
        else
            return col4(ct, ku, lane);
    }
    __device__ __forceinline__ void put_unit(int row, int ku, int g, const Unit& u) const {  // the inverse of blocks()
        if constexpr (Op::kScaled) {
            *reinterpret_cast<f16x4*>(at(row, 32 * ku + 4 * g)) = __builtin_shufflevector(u, u, 0, 1, 2, 3);
            *reinterpret_cast<f16x4*>(at(row, 32 * ku + 16 + 4 * g)) = __builtin_shufflevector(u, u, 4, 5, 6, 7);
        } else {
            *reinterpret_cast<Unit*>(at(row, 16 * ku + 4 * g)) = u;
        }
    }
    template <int N>
    __device__ __forceinline__ void put(int row, int col, const float (&x)[N], float s) const {
        if constexpr (Op::kScaled) {
            // bf16 values times a power of two: their 8 bits fit fp16's 11, so the
            // conversion towards zero, two in one instruction, rounds subnormals alone
            typedef uint32_t words __attribute__((ext_vector_type(N / 2)));
            words h;
#pragma unroll
            for (int i = 0; i < N; i += 2)
                h[i / 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[i] * s, x[i + 1] * s));
            *reinterpret_cast<words*>(at(row, col)) = h;
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 4)
                *reinterpret_cast<f32x4*>(at(row, col + i)) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
        }
    }
};

// The thread's index, computed anew: what depends on it does not move out of a
// loop around the call, where the exact kernel's loops over chunks would keep
// all of it in registers (1.8 KiB of spills a lane, and 7 us a launch for them).
__device__ __forceinline__ int thread_index() {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    return tid;
}

// 64 x 64 fp32 in LDS, 16-byte groups of a row XORed by the row.
__device__ __forceinline__ int sq_at(int r, int c) { return r * 64 + ((((c >> 2) ^ r) & 15) << 2) + (c & 3); }

__device__ __forceinline__ int bits_abs(float x) { return int(__float_as_uint(x) & 0x7fffffffu); }
// Maximum over the wave of non-negative ints (magnitude bits: a NaN's are the
// largest), by DPP within rows of 16 and then over the four rows.
template <int CTRL>
__device__ __forceinline__ int dpp_max(int x) {
    return max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ int wave_max_bits(int x) {
    x = dpp_max<0x128>(dpp_max<0x124>(dpp_max<0x4E>(dpp_max<0xB1>(x))));
    return max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
               max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}
// The exponent of magnitude bits, 100 at most either way.
__device__ __forceinline__ int bits_exp(int bits) { return max(min((bits >> 23) - 127, 100), -100); }
// The exponent that K or Q of a chunk is divided by before its rounding to fp16:
// none for values of ordinary size (largest in [2^-8, 16): fp16's steps of 2^-24
// below 2^-14 are then 2^-16 of it at most), else the largest value's.
__device__ __forceinline__ int rows_exp(int bits) {
    const int e = bits_exp(bits);
    return bits == 0 || (e >= -8 && e < 4) ? 0 : e;
}

// A run of 16 bytes of a row of T (8 bf16 or 4 fp32).  VEC: rows are whole runs
// and aligned, and a run outside the matrix (`in` false) is read from zeros
// kept for it: nothing touches the loaded registers before their use, so that
// loads issued ahead stay in flight.
template <typename T>
constexpr int kRun = 16 / int(sizeof(T));
__device__ const u32x4 kZeroRun = {0, 0, 0, 0};
typedef const __attribute__((address_space(1))) u32x4 global_u32x4;
template <typename T, bool VEC>
__device__ __forceinline__ u32x4 load_run(const T* p, bool in, int n) {
    if constexpr (VEC) {
        const u32x4* u = in ? reinterpret_cast<const u32x4*>(p) : &kZeroRun;
        return *(global_u32x4*)(u);
    } else {
        T x[kRun<T>];
#pragma unroll
        for (int i = 0; i < kRun<T>; ++i) x[i] = in && i < n ? p[i] : T(0);
        return __builtin_bit_cast(u32x4, x);
    }
}
// Whole rows of a chunk: 16 bytes at `offset` bytes behind a pointer that the wave shares.
__device__ __forceinline__ u32x4 load_at(const void* p, unsigned offset) {
    return *(global_u32x4*)(reinterpret_cast<const u32x4*>(static_cast<const char*>(p) + offset));
}
template <typename T>
__device__ __forceinline__ void unpack_run(const u32x4& u, float (&x)[kRun<T>]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(w[i]);
        } else {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
// the larger magnitude bits of a pair of 16-bit floats and of those of `m`
__device__ __forceinline__ u16x2 pair_max_bits(u16x2 m, uint32_t x) {
    return __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x & 0x7fff7fffu));
}
template <typename T>
__device__ __forceinline__ int run_max_bits(const u32x4& u) {
    if constexpr (sizeof(T) == 2) {  // as pairs of 15-bit integers
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) m = pair_max_bits(m, u[i]);
        return max(int(m.x), int(m.y)) << 16;
    } else {
        return int(max(max(u.x & 0x7fffffffu, u.y & 0x7fffffffu), max(u.z & 0x7fffffffu, u.w & 0x7fffffffu)));
    }
}
// Two floats as bf16, round to nearest even, by the hardware's conversion.
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}
// N consecutive values of a row of which n lie in the matrix; VEC: all or none do.
template <typename T, bool VEC, int N>
__device__ __forceinline__ void store_run(T* p, int n, const float (&x)[N]) {
    if constexpr (VEC) {
        if (n <= 0) return;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i += 4)
                *reinterpret_cast<f32x4*>(p + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
        } else if constexpr (N == 8) {
            *reinterpret_cast<u32x4*>(p) =
                u32x4{bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4], x[5]), bf16_pair(x[6], x[7])};
        } else {
            *reinterpret_cast<uint2*>(p) = uint2{bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3])};
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) Elem<T>::store(p, i, x[i]);
    }
}

// ------------------------------------------------------------ workspace
// One record per (chunk, head), for DK = d_k padded to 32, 64 or 128 and d_v
// padded to 16-row tiles (an even number of them).
struct RecLayout {
    size_t t, p, w, x, s0, ds1, vec, bytes;
};
__host__ __device__ inline RecLayout rec_layout(int DK, int dvt, int es) {
    RecLayout l{};
    const size_t tt = (size_t)64 * 64 * es, tv = (size_t)64 * dvt * 16 * es, st = (size_t)DK * dvt * 16 * es;
    size_t at = 0;
    l.t = at; at += tt;     // T by rows
    l.p = at; at += tt;     // P by rows, scaled as K and Q are
    l.w = at; at += tv;     // W                              (token; d_v), by units of d_v
    l.x = at; at += tv;     // dX                             (token; d_v), by units of d_v
    l.s0 = at; at += st;    // S0                             (d_k; d_v), by units of d_v
    l.ds1 = at; at += st;   // dS1                            (d_k; d_v), by units of d_v
    l.vec = at;             // small values, then the tiles' exponents
    at += 256 * 4 + 5 * 64 * 4;
    l.bytes = (at + 255) & ~(size_t)255;
    return l;
}
// the record's small values: gamma, beta tail and beta by token, gamma_c,
// exponents of K and Q, whether the chunk leaves the fp16 operands' domain,
// exponents of the largest beta, beta tail and gamma (the first token's) and of gamma_c
enum {
    kVecGamma = 0, kVecWrite = 64, kVecBeta = 128, kVecGc = 192, kVecEK = 193, kVecEQ = 194, kVecBad = 195, kVecEB = 196,
    kVecEW = 197, kVecEG = 198, kVecEGc = 199, kVecs = 200
};
// exponents by d_v tile, from float 256 on
enum { kExpO = 256, kExpW = 320, kExpX = 384, kExpS = 448, kExpD = 512 };

struct BwdParams {
    const void *q, *k, *v, *dout;
    const float *gate, *beta, *init, *dfinal;
    const int *cu, *chunk_base;  // packed: chunk_base[n] chunks precede sequence n
    void *dq, *dk, *dv, *dgate, *dbeta;
    float* dinit;
    char* ws;
    RecLayout rec;
    int batch, seq_len, heads, d_k, d_v, dvt, gate_is_alpha;
    bool short_rows;  // a chunk's rows lie within 2 GiB
    bool vec_s;  // rows of the states, 16 bytes at a time
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

// Running log-decays (to base 2, in fp64, so that a difference of two is exact
// to fp32 whatever came before) and factors of a chunk, by the first wave.
struct Gates {
    double G[64];
    float gamma[64], tail[64], beta[64], gate[64];
};
__device__ __forceinline__ float pow2(double x) { return __builtin_amdgcn_exp2f((float)x); }
__device__ __forceinline__ bool load_gates(const BwdParams& p, const ChunkAt& at, int h, Gates& gs, int lane) {
    const bool in = lane < at.n;
    const long r = (long)(at.t0 + (in ? lane : 0)) * p.heads + h;
    float gate = p.gate[r], beta = p.beta[r];
    gate = in ? gate : (p.gate_is_alpha ? 1.f : 0.f);
    beta = in ? beta : 0.f;
    const float g = p.gate_is_alpha ? logf(gate) : gate;
    const bool bad = !(g <= 0.f) || !(beta >= 0.f && beta <= 1.f);
    double G = (double)(g < kMinLog ? kMinLog : g) * 1.4426950408889634;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(G, off, kWave);
        if (lane >= off) G += o;
    }
    const double Gc = __shfl(G, 63, kWave);
    gs.G[lane] = G;
    gs.gamma[lane] = pow2(G);
    gs.tail[lane] = pow2(Gc - G);
    gs.beta[lane] = beta;
    gs.gate[lane] = gate;
    return bad;
}
__device__ __forceinline__ float decay(const Gates& gs, int r, int s) { return pow2(gs.G[r] - gs.G[s]); }

// ----------------------------------------------------------------- prep
// One (chunk, head) per workgroup of four waves.  LDS: K by rows (then T), Q by
// rows (then P and T's diagonal blocks in fp32), L diag(beta) in fp32.  T and P
// (16 KiB) are handed on rather than T K, T V, P^T dO and their like (80 KiB):
// the scans multiply by them twice instead, which cost less than the traffic
// (prep 152 -> 66 us, the whole call 594 -> 528 us at the size above).  73 us
// for 0.22 GB: bound by the latency of the forward substitution and the products
// down T's block columns, three workgroups a CU.
template <class Op, int DK>
struct PrepLds {
    using T64 = RowMat<Op, 64>;
    static constexpr int kRow = RowMat<Op, DK>::bytes(64), kT64 = T64::bytes(64), kDiag = 4 * 16 * 16 * 4;
    static constexpr int kKr = 0, kT = 0;
    static constexpr int kQr = kRow > kT64 ? kRow : kT64;
    static constexpr int kP = kQr, kTd = kQr + kT64;
    static constexpr int kA = kQr + (kRow > kT64 + kDiag ? kRow : kT64 + kDiag);
    static constexpr int kGates = kA + 64 * 64 * 4;
    static constexpr int kMisc = kGates + int(sizeof(Gates));
    static constexpr int kBytes = kMisc + 64;
};

template <class Op, typename T, int DK, bool VEC>
__device__ __forceinline__ void prep_chunk(const BwdParams& p, const ChunkAt& at, int h, char* rec, char* lds) {
    using Unit = typename Op::Unit;
    using Elt = typename Op::Elt;
    using L = PrepLds<Op, DK>;
    constexpr int NT = DK / 16, NBK = Op::kBlocks, NKK = NT / NBK, NKT = 4 / NBK, R = kRun<T>;
    constexpr int NR = 64 * DK / R / 256;  // runs of K (and of Q) per thread
    const int tid = thread_index(), wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4,
              m = lane & 15;
    const RowMat<Op, DK> Kr{lds + L::kKr}, Qr{lds + L::kQr};
    const RowMat<Op, 64> Th{lds + L::kT}, Ph{lds + L::kP};
    float* Td = reinterpret_cast<float*>(lds + L::kTd);
    float* Af = reinterpret_cast<float*>(lds + L::kA);
    Gates& gs = *reinterpret_cast<Gates*>(lds + L::kGates);
    int* misc = reinterpret_cast<int*>(lds + L::kMisc);  // maxima of K, Q by wave; [8] outside the domain
    float* vec = reinterpret_cast<float*>(rec + p.rec.vec);
    int* exps = reinterpret_cast<int*>(vec);

    const long ldk = (long)p.heads * p.d_k;
    const T* kp = static_cast<const T*>(p.k) + at.t0 * ldk + (long)h * p.d_k;
    const T* qp = static_cast<const T*>(p.q) + at.t0 * ldk + (long)h * p.d_k;
    u32x4 kb[NR], qb[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int id = tid + 256 * i, t = id / (DK / R), c = id % (DK / R) * R;
        const bool in = t < at.n && c < p.d_k;
        kb[i] = load_run<T, VEC>(kp + t * ldk + c, in, p.d_k - c);
        qb[i] = load_run<T, VEC>(qp + t * ldk + c, in, p.d_k - c);
    }
    bool bad = false;
    if (wave == 0) bad = load_gates(p, at, h, gs, lane);
    int ek = 0, eq = 0;
    if constexpr (Op::kScaled) {
        int mk = 0, mq = 0;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            mk = max(mk, run_max_bits<T>(kb[i]));
            mq = max(mq, run_max_bits<T>(qb[i]));
        }
        mk = wave_max_bits(mk);
        mq = wave_max_bits(mq);
        if (lane == 0) {
            misc[wave] = mk;
            misc[4 + wave] = mq;
        }
        if (tid == 0) misc[8] = 0;
        __syncthreads();
        const int bk = max(max(misc[0], misc[1]), max(misc[2], misc[3]));
        const int bq = max(max(misc[4], misc[5]), max(misc[6], misc[7]));
        ek = rows_exp(bk);
        eq = rows_exp(bq);
        bad = bad || bk >= 0x7f800000 || bq >= 0x7f800000;
    }
    {
        const float sk = exp2i(-ek), sq = exp2i(-eq);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int id = tid + 256 * i, t = id / (DK / R), c = id % (DK / R) * R;
            float x[R];
            unpack_run<T>(kb[i], x);
            Kr.put(t, c, x, sk);
            unpack_run<T>(qb[i], x);
            Qr.put(t, c, x, sq);
        }
    }
    __syncthreads();
    if (tid < 64) {
        const float beta = gs.beta[tid], write = beta * gs.tail[tid];
        vec[kVecGamma + tid] = gs.gamma[tid];
        vec[kVecWrite + tid] = write;
        vec[kVecBeta + tid] = beta;
        if constexpr (Op::kScaled) {
            const int eb = bits_exp(wave_max_bits(bits_abs(beta))), ew = bits_exp(wave_max_bits(bits_abs(write)));
            if (tid == 0) {
                exps[kVecEB] = eb;
                exps[kVecEW] = ew;
                exps[kVecEG] = bits_exp(bits_abs(gs.gamma[0]));
                exps[kVecEGc] = bits_exp(bits_abs(gs.gamma[63]));
            }
        }
    }
    if (tid == 0) {
        vec[kVecGc] = gs.gamma[63];
        exps[kVecEK] = ek;
        exps[kVecEQ] = eq;
    }

    // column tile `wave` of L diag(beta) (fp32), row tile `wave` of P (scaled as
    // K and Q are, in registers): five tiles of products each wave
    Unit pu[NKT];
    {
        const float kk2 = exp2i(2 * ek);
        const int s = 16 * wave + m;
        const float bs = gs.beta[s];
        Unit uk[NKK], uq[NKK];
#pragma unroll
        for (int ku = 0; ku < NKK; ++ku) {
            uk[ku] = Kr.run(16 * wave, ku, lane);
            uq[ku] = Qr.run(16 * wave, ku, lane);
        }
        f32x4 pt[4];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            f32x4 ck = {0, 0, 0, 0}, cq = {0, 0, 0, 0};
#pragma unroll
            for (int ku = 0; ku < NKK; ++ku) {
                const Unit a = Kr.run(16 * mt, ku, lane);
                if (mt >= wave) ck = Op::mma(a, uk[ku], ck);
                if (mt <= wave) cq = Op::mma(a, uq[ku], cq);
            }
            pt[mt] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * mt + 4 * g + i;
                if (mt >= wave) {  // row r of L, column s
                    const float kk = ck[i] * kk2;
                    if (Op::kScaled && r == s && !(kk <= 1.03125f)) bad = true;
                    Af[sq_at(r, s)] = s < r ? kk * decay(gs, r, s) * bs : 0.f;
                }
                if (mt <= wave && r <= s) pt[mt][i] = cq[i] * decay(gs, s, r);  // row s of P, column r
            }
        }
#pragma unroll
        for (int u = 0; u < NKT; ++u) pu[u] = Op::pack(&pt[u * NBK], 1.f);
    }
    if constexpr (Op::kScaled)
        if (bad) misc[8] = 1;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NKT; ++u) Ph.put_unit(16 * wave + m, u, g, pu[u]);

    // T's diagonal blocks by forward substitution in fp32, column m of block
    // `wave` in lane (., m); then T_iw = -T_ii sum_{w <= b < i} A_ib T_bw down
    // block column w on fp32 MFMA
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
        // row-major, so that a left operand is one read
#pragma unroll
        for (int i = 0; i < 4; ++i) Td[wave * 256 + (4 * g + i) * 16 + m] = d[i];
        __syncthreads();
        f32x4 tc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            tc[i] = f32x4{0, 0, 0, 0};
            if (i == wave) tc[i] = d;
            if (i > wave) {
                f32x4 y = {0, 0, 0, 0}, z = {0, 0, 0, 0};
#pragma unroll
                for (int b = 0; b < i; ++b)
                    if (b >= wave)
                        y = OpF32::mma(*reinterpret_cast<const f32x4*>(Af + sq_at(16 * i + m, 16 * b + 4 * g)), tc[b], y);
                z = OpF32::mma(*reinterpret_cast<const f32x4*>(Td + i * 256 + m * 16 + 4 * g), y, z);
                tc[i] = -z;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<Elt*>(Th.at(16 * i + 4 * g + e, 16 * wave + m)) = (Elt)tc[i][e];
        }
    }
    __syncthreads();

    constexpr int NP = 64 * int(sizeof(Elt)) / 16;  // 16-byte pieces of a row of T and P
    u32x4* ot = reinterpret_cast<u32x4*>(rec + p.rec.t);
    u32x4* op = reinterpret_cast<u32x4*>(rec + p.rec.p);
#pragma unroll
    for (int i = 0; i < 64 * NP / 256; ++i) {
        const int id = tid + 256 * i;
        ot[id] = *reinterpret_cast<const u32x4*>(Th.at(id / NP, id % NP * (64 / NP)));
        op[id] = *reinterpret_cast<const u32x4*>(Ph.at(id / NP, id % NP * (64 / NP)));
    }
    if (Op::kScaled && tid == 0) exps[kVecBad] = misc[8];
}

template <class Op, typename T, int DK, bool VEC>
__global__ __launch_bounds__(256, Op::kScaled ? 3 : 1) void bwd_prep_kernel(BwdParams p) {
    __shared__ __align__(16) char lds[PrepLds<Op, DK>::kBytes];
    const int ci = blockIdx.x / p.heads, h = blockIdx.x - ci * p.heads;
    ChunkAt at;
    if (!find_chunk(p, ci, at)) return;
    prep_chunk<Op, T, DK, VEC>(p, at, h, p.ws + (size_t)blockIdx.x * p.rec.bytes, lds);
}

// ----------------------------------------------------------------- scan
// A wave carries 16 rows of S (or of dS) along the chunks of a (sequence, head)
// in accumulators: tile b holds d_k indices 16 b + 4 g .. + 3 of row m.  The
// state's own operands come from its accumulators; K, Q, T and P pass through
// LDS once for a workgroup's four such waves and serve as rows and as columns.
// Forward: W = T (V - diag(gamma) K S0^T), S1 = gamma_c S0 + (beta tail W)^T K.
// Back: dX = T^T (diag(beta) P^T dO + diag(beta tail) K dS1^T), dS0 = gamma_c
// dS1 + (gamma dO)^T Q - (gamma dX)^T K.  What the gradients need (S0, W, dS1,
// dX) is turned through LDS into the order that their products take.
template <class Op, int DK>
struct ScanBuf {  // a chunk's shared operands
    static constexpr int kRow = RowMat<Op, DK>::bytes(64), kT64 = RowMat<Op, 64>::bytes(64);
    static constexpr int kK = 0, kT = kRow, kVec = kT + kT64, kQ = kVec + 1024, kP = kQ + kRow;
    static constexpr int kBytes = kP + kT64;
};

// The exponent of the largest value of a wave's tiles (NaNs do not count).
template <int N>
__device__ __forceinline__ int tiles_exp(const f32x4 (&w)[N]) {
    float mx = 0.f;
#pragma unroll
    for (int b = 0; b < N; ++b)
        mx = fmaxf(fmaxf(fmaxf(mx, fabsf(w[b][0])), fabsf(w[b][1])), fmaxf(fabsf(w[b][2]), fabsf(w[b][3])));
    return bits_exp(wave_max_bits(bits_abs(mx)));
}

template <class Op, int DK>
struct State {
    static constexpr int NT = DK / 16, NBK = Op::kBlocks, NU = NT / NBK;
    f32x4 s[NT];
    int e;  // the state is s * 2^e, with |s| below 2^15.1: its fp16 operands are s itself

    __device__ __forceinline__ int top() const { return tiles_exp<NT>(s) + e; }  // the largest value's exponent
    __device__ __forceinline__ void load(const BwdParams& p, const float* base, int row, int c0) {
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const int c = c0 + 16 * b;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[b][i] = 0.f;
            if (base && row < p.d_v && c < p.d_k) {
                const float* r = base + (long)row * p.d_k + c;
                if (p.vec_s) {
                    s[b] = *reinterpret_cast<const f32x4*>(r);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (c + i < p.d_k) s[b][i] = r[i];
                }
            }
        }
        e = 0;
        if constexpr (Op::kScaled) {
            e = top() - 7;
            const float f = exp2i(-e);
#pragma unroll
            for (int b = 0; b < NT; ++b) s[b] *= f;
        }
    }
    __device__ __forceinline__ void store(const BwdParams& p, float* base, int row, int c0) const {
        if (row >= p.d_v) return;
        const float f = exp2i(e);
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const int c = c0 + 16 * b;
            if (c >= p.d_k) continue;
            float* r = base + (long)row * p.d_k + c;
            if (p.vec_s) {
                *reinterpret_cast<f32x4*>(r) = s[b] * f;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c + i < p.d_k) r[i] = s[b][i] * f;
            }
        }
    }
};

// The chunk's tokens of a sequence.
template <typename T>
struct SeqAt {
    const T *k, *q, *vo;  // the sequence's first token of this head: K, Q, and V or dO
    int tokens;
};

// 16 columns of V (or dO) of a chunk, as the rows come from HBM to `THREADS`
// threads; `lane` counts them.
template <typename T, bool VEC, int THREADS = 64>
struct TileRuns {
    static constexpr int R = kRun<T>, RUNS = 64 * 16 / R, N = (RUNS + THREADS - 1) / THREADS, RPR = 16 / R;
    u32x4 r[N];
    __device__ __forceinline__ void load(const BwdParams& p, const SeqAt<T>& at, int c, int tile, int lane) {
        const long ld = (long)p.heads * p.d_v;
        if (VEC && sizeof(T) == 2 && RUNS % THREADS == 0 && p.short_rows && at.tokens - c * C64 >= C64 && 16 * tile + 16 <= p.d_v) {
            const T* base = at.vo + c * C64 * ld + 16 * tile;
            const unsigned off = ((unsigned)(lane / RPR) * (unsigned)ld + lane % RPR * R) * sizeof(T);
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = load_at(base + i * (THREADS / RPR) * ld, off);
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = lane + THREADS * i, t = c * C64 + id / RPR, col = 16 * tile + id % RPR * R;
            r[i] = load_run<T, VEC>(at.vo + t * ld + col, id < RUNS && t < at.tokens && col < p.d_v, p.d_v - col);
        }
    }
    __device__ __forceinline__ int max_bits() const {
        int m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) m = max(m, run_max_bits<T>(r[i]));
        return wave_max_bits(m);
    }
    // through LDS, 16-bit values as they are: rows in, then the tokens 16 b + 4 g .. of column m out
    using Raw = RowMat<typename std::conditional<sizeof(T) == 2, OpF16, OpF32>::type, 16>;
    __device__ __forceinline__ void put(char* corner, int lane) const {
        const Raw tn{corner};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = lane + THREADS * i;
            if (id < RUNS) *reinterpret_cast<u32x4*>(tn.at(id / RPR, id % RPR * R)) = r[i];
        }
    }
    static __device__ __forceinline__ void get(char* corner, f32x4 (&x)[4], int lane) {
        const Raw tn{corner};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if constexpr (sizeof(T) == 2) {
                const s16x4 h = __builtin_bit_cast(s16x4, tn.col4(0, b, lane));
#pragma unroll
                for (int i = 0; i < 4; ++i) x[b][i] = __uint_as_float(uint32_t(uint16_t(h[i])) << 16);
            } else {
                x[b] = tn.col4(0, b, lane);
            }
        }
    }
};

// Rows of two tiles as units with d_v along the contraction: `N` column
// tiles of the turned matrices from `first` on, 1 KiB each.  `top` becomes the
// largest magnitude bits stored.
template <int N, class Mat>
__device__ __forceinline__ void store_turned(const Mat& even, const Mat& odd, char* base, int first, int lane, u16x2& top) {
    char* o = base + first * 1024 + lane * 16;
#pragma unroll
    for (int b = 0; b < N; ++b) {
        const f16x8 u = __builtin_shufflevector(even.col4(first + b, 0, lane), odd.col4(first + b, 0, lane), 0, 1, 2, 3, 4,
                                                5, 6, 7);
        *reinterpret_cast<f16x8*>(o + b * 1024) = u;
        const u32x4 w = __builtin_bit_cast(u32x4, u);
#pragma unroll
        for (int i = 0; i < 4; ++i) top = pair_max_bits(top, w[i]);
    }
}

// A chunk's shared operands on their way from HBM to LDS, by `THREADS` threads.
template <class Op, typename T, int DK, bool VEC, bool BACK, int THREADS = 256>
struct ScanStage {
    static constexpr int R = kRun<T>, RUNS = 64 * DK / R, N = (RUNS + THREADS - 1) / THREADS;
    static constexpr int NP = 64 * int(sizeof(typename Op::Elt)) / 16, NT = 64 * NP / THREADS;
    u32x4 k[N], q[BACK ? N : 1], t[NT], pp[BACK ? NT : 1];
    float vec;
    int ek, eq;
    __device__ __forceinline__ void load(const BwdParams& p, const SeqAt<T>& at, int c, const char* rec, int tid) {
        const long ld = (long)p.heads * p.d_k;
        constexpr int RPR = DK / R;
        if (VEC && sizeof(T) == 2 && RUNS % THREADS == 0 && p.short_rows && at.tokens - c * C64 >= C64 && p.d_k == DK) {
            const unsigned off = ((unsigned)(tid / RPR) * (unsigned)ld + tid % RPR * R) * sizeof(T);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const long from = (c * C64 + i * (THREADS / RPR)) * ld;
                k[i] = load_at(at.k + from, off);
                if constexpr (BACK) q[i] = load_at(at.q + from, off);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int id = tid + THREADS * i, tk = c * C64 + id / RPR, col = id % RPR * R;
                const bool in = id < RUNS && tk < at.tokens && col < p.d_k;
                k[i] = load_run<T, VEC>(at.k + tk * ld + col, in, p.d_k - col);
                if constexpr (BACK) q[i] = load_run<T, VEC>(at.q + tk * ld + col, in, p.d_k - col);
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            t[i] = reinterpret_cast<const u32x4*>(rec + p.rec.t)[tid + THREADS * i];
            if constexpr (BACK) pp[i] = reinterpret_cast<const u32x4*>(rec + p.rec.p)[tid + THREADS * i];
        }
        const float* v = reinterpret_cast<const float*>(rec + p.rec.vec);
        vec = v[min(tid, kVecs - 1)];
        ek = eq = 0;
        if constexpr (Op::kScaled) {
            ek = reinterpret_cast<const int*>(v)[kVecEK];
            eq = reinterpret_cast<const int*>(v)[kVecEQ];
        }
    }
    template <bool SCALE>
    static __device__ __forceinline__ void put_rows_as(char* to, const u32x4* from, int e, int tid) {
        const RowMat<Op, DK> rows{to};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = tid + THREADS * i;
            if (id >= RUNS) break;
            float x[R];
            unpack_run<T>(from[i], x);
            rows.put(id / (DK / R), id % (DK / R) * R, x, SCALE ? exp2i(-e) : 1.f);
        }
    }
    static __device__ __forceinline__ void put_rows(char* to, const u32x4* from, int e, int tid) {
        if (Op::kScaled && __builtin_amdgcn_readfirstlane(e) != 0) put_rows_as<true>(to, from, e, tid);
        else put_rows_as<false>(to, from, e, tid);
    }
    static __device__ __forceinline__ void put_square(char* to, const u32x4* from, int tid) {
        const RowMat<Op, 64> sq{to};
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int id = tid + THREADS * i;
            *reinterpret_cast<u32x4*>(sq.at(id / NP, id % NP * (64 / NP))) = from[i];
        }
    }
    // K, T and the small values, then Q and P (back)
    __device__ __forceinline__ void store(char* buf, int tid) const {
        using L = ScanBuf<Op, DK>;
        put_rows(buf + L::kK, k, ek, tid);
        put_square(buf + L::kT, t, tid);
        if (tid < kVecs) reinterpret_cast<float*>(buf + L::kVec)[tid] = vec;
    }
    __device__ __forceinline__ void store_back(char* buf, int tid) const {
        using L = ScanBuf<Op, DK>;
        if constexpr (BACK) {
            put_rows(buf + L::kQ, q, eq, tid);
            put_square(buf + L::kP, pp, tid);
        }
    }
};

template <typename T>
__device__ __forceinline__ SeqAt<T> seq_at(const BwdParams& p, int seq, int h, bool back) {
    int t0, t1;
    seq_bounds(p.cu, seq, p.seq_len, t0, t1);
    const long rk = ((long)t0 * p.heads + h) * p.d_k, rv = ((long)t0 * p.heads + h) * p.d_v;
    return {static_cast<const T*>(p.k) + rk, static_cast<const T*>(p.q) + rk,
            static_cast<const T*>(back ? p.dout : p.v) + rv, t1 - t0};
}

// The rows that a workgroup of a scan launch carries: the workgroups that share
// a (sequence, head, direction) follow each other on one XCD (blocks go round
// the eight), whose L2 then serves their K, Q, T and P.
struct ScanAt {
    bool back;
    int seq, h, part, nc;
    char* rec;        // the first chunk's record
    size_t stride;    // from chunk to chunk
    long state;       // index of the head's state
};
__device__ __forceinline__ bool scan_at(const BwdParams& p, int splits, ScanAt& a) {
    const int per = 8 * splits, grp = blockIdx.x / per, in = blockIdx.x - grp * per;
    int id = grp * 8 + (in & 7);
    a.part = in >> 3;
    a.back = id & 1;
    id >>= 1;
    if (id >= p.batch * p.heads) return false;
    a.seq = id / p.heads;
    a.h = id - a.seq * p.heads;
    int ci;
    if (p.cu) {
        ci = p.chunk_base[a.seq];
        a.nc = p.chunk_base[a.seq + 1] - ci;
    } else {
        a.nc = (p.seq_len + C64 - 1) / C64;
        ci = a.seq * a.nc;
    }
    a.rec = p.ws + ((size_t)ci * p.heads + a.h) * p.rec.bytes;
    a.stride = (size_t)p.heads * p.rec.bytes;
    a.state = (long)id * p.d_v * p.d_k;
    return true;
}

// bf16 tensors, fp16 operands.  A wave's chunk is one chain of LDS reads and
// products, and a wave issues an instruction every four to five cycles at best,
// so four more waves do what is off the chain: they read K, Q, T, P and the
// carrying waves' columns of V or dO two chunks ahead, convert them to LDS one
// chunk ahead, and turn and store the previous chunk's S0 and W (dS1 and dX).
// Two barriers a chunk: A, the buffers of the chunk are full and its
// predecessor's results lie in LDS; B, these have been read.  What the serving
// waves do is split around B as the chain is.
//
// The chain has no exponent of its own results to wait for: a chunk's values
// are scaled by the larger of the state's and of V's (dO's) largest value and
// those of the factors on their way.  A single term is thereby some 2^10 below
// fp16's range and 2^19 above its subnormals; sums of terms of one sign reach
// 2^10 in W and 2^14 in dX.
// Growth beyond that shows as an infinity or NaN in the state or in the W or dX
// that is handed on (rows of q of some 180 along all of a chunk's keys, say,
// whose state decays before it takes them up), and the head is done again in
// fp32.  The serving waves watch W and dX as they store them, off the chain (no
// difference in time).
//
// 16384 tokens, 16 heads, d_k = 128, d_v = 256: 784 us, some 5900 cycles a chunk,
// of which the chain waits 350; eight serving waves leave it 168 registers: 816.
// 4 x 4096 tokens, d = 128 (a workgroup on every CU): 243 us for 0.85 GB, 67 % of
// a copy's rate.
template <int DK>
struct Scan16Lds {
    using Buf = ScanBuf<OpF16, DK>;
    static constexpr int kTile = RowMat<OpF16, 16>::bytes(64);                    // a wave's columns of V or dO
    static constexpr int kTurnS = RowMat<OpF16, DK>::bytes(16), kTurnW = RowMat<OpF16, 64>::bytes(16);
    static constexpr int kTiles = 2 * Buf::kBytes, kTurn = kTiles + 8 * kTile, kExps = kTurn + 4 * (kTurnS + kTurnW);
    static constexpr int kBytes = kExps + 8 * 4;
};

// two products rounded to a pair of fp16
__device__ __forceinline__ OpF16::Unit pack_products(const f32x4* x, const f32x4* f) {
    const f32x4 t[2] = {x[0] * f[0], x[1] * f[1]};
    return OpF16::pack(t, 1.f);
}

template <typename T, int DK, bool VEC, bool BACK>
__device__ __forceinline__ void scan16_carry(const BwdParams& p, const ScanAt& a, int tile, int wave, int lane, char* lds) {
    using Op = OpF16;
    using Unit = f16x8;
    using L = Scan16Lds<DK>;
    using Buf = typename L::Buf;
    constexpr int NT = DK / 16, NU = NT / 2;
    const int g = lane >> 4, m = lane & 15, row = 16 * tile + m;
    const float* from = BACK ? p.dfinal : p.init;
    State<Op, DK> S;
    S.load(p, from ? from + a.state : nullptr, row, 4 * g);
    const RowMat<Op, DK> ts{lds + L::kTurn + wave * (L::kTurnS + L::kTurnW)};
    const RowMat<Op, 64> tw{lds + L::kTurn + wave * (L::kTurnS + L::kTurnW) + L::kTurnS};
    int* exps = reinterpret_cast<int*>(a.rec + (BACK ? a.nc - 1 : 0) * a.stride + p.rec.vec);
    for (int c = 0; c < a.nc; ++c) {
        // the state's largest value between 2^-4 and 2^10
        int top = tiles_exp<NT>(S.s);
        if (top < -4 || top > 9) {
            const float f = exp2i(5 - top);
#pragma unroll
            for (int b = 0; b < NT; ++b) S.s[b] *= f;
            S.e += top - 5;
            top = 5;
        }
        Unit su[NU];
#pragma unroll
        for (int i = 0; i < NU; ++i) su[i] = Op::pack(&S.s[i * 2], 1.f);
        __syncthreads();  // A
        char* buf = lds + (c & 1) * Buf::kBytes;
        const RowMat<Op, DK> K{buf + Buf::kK}, Q{buf + Buf::kQ};
        const RowMat<Op, 64> Tm{buf + Buf::kT}, P{buf + Buf::kP};
        const float* vec = reinterpret_cast<const float*>(buf + Buf::kVec);
        auto by_token = [&](int v, int b) { return *reinterpret_cast<const f32x4*>(vec + v + 16 * b + 4 * g); };
        const float gc = vec[kVecGc];
        const int ek = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(vec)[kVecEK]);
        const int eq = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(vec)[kVecEQ]);
        const int eb = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(vec)[kVecEB]);
        const int et = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(vec)[kVecEW]);
        const int eg = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(vec)[kVecEG]);
        const int egc = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(vec)[kVecEGc]);
        // of V, or dO: its largest value below 2^ev
        const int ev = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(lds + L::kExps)[(c & 1) * 4 + wave]);
        f32x4 x[4], w[4], vo[4];
        TileRuns<T, VEC>::get(lds + L::kTiles + ((c & 1) * 4 + wave) * L::kTile, vo, lane);
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) x[b] = Op::mma(K.blocks(16 * b + m, i, g), su[i], x[b]);
        // W or dX are kept times 2^-ew, the next state is S times 2^-e: the larger of
        // what the state and V (dO times rows of Q) give, with the largest factors that
        // K, beta and the decays bring, at 2^5 to 2^7.  So small keys or betas leave
        // what they multiply its bits, and a state that is forgotten leaves those of
        // what follows it.
        const int se = S.e, own = top + se - 5, in = ev + (BACK ? eq + 2 : 0) - 5;
        const int ew = BACK ? ek + max(own + et, in + eb) : max(own + ek + eg, in);
        const int e = max(own + egc, BACK ? max(in + eg, ew + ek + eg) : ew + ek + et);
        Unit ru[2];
        if constexpr (!BACK) {
            const float sv = exp2i(-ew), sx = -exp2i(se + ek - ew);
#pragma unroll
            for (int b = 0; b < 4; ++b) w[b] = vo[b] * sv + (by_token(kVecGamma, b) * sx) * x[b];
        } else {
            const int eo = ev + 1;  // dO as an operand: below 1/2
            const float so = exp2i(-eo), sz = exp2i(eo + eq + ek - ew), sx = exp2i(se + ek - ew);
            f32x4 z[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) z[b] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Unit du = Op::pack(&vo[u * 2], so);
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    if (u * 2 + 2 > b) z[b] = Op::mma(P.cols(b, u, lane), du, z[b]);
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) w[b] = (by_token(kVecBeta, b) * sz) * z[b] + (by_token(kVecWrite, b) * sx) * x[b];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) ru[u] = Op::pack(&w[u * 2], 1.f);
#pragma unroll
        for (int b = 0; b < 4; ++b) w[b] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (!BACK && u * 2 <= b) w[b] = Op::mma(Tm.blocks(16 * b + m, u, g), ru[u], w[b]);
                if (BACK && u * 2 + 2 > b) w[b] = Op::mma(Tm.cols(b, u, lane), ru[u], w[b]);
            }
        Unit kc[NT];  // read ahead of the barrier, to be there behind it
#pragma unroll
        for (int b = 0; b < NT; ++b) kc[b] = K.cols(b, 0, lane);
        const float sg = gc * exp2i(se - e);
#pragma unroll
        for (int b = 0; b < NT; ++b) S.s[b] *= sg;
        S.e = e;
        if (lane == 0) {
            exps[(BACK ? kExpX : kExpW) + tile] = ew;
            exps[(BACK ? kExpD : kExpS) + tile] = se;
            if constexpr (BACK) exps[kExpO + tile] = ev + 1;
        }
        exps += (BACK ? -(long)a.stride : (long)a.stride) / 4;
        __syncthreads();  // B
#pragma unroll
        for (int i = 0; i < NU; ++i) ts.put_unit(m, i, g, su[i]);
#pragma unroll
        for (int u = 0; u < 2; ++u) tw.put_unit(m, u, g, Op::pack(&w[u * 2], 1.f));
        const float sd = exp2i(eq - e), sw = exp2i(ew + ek - e);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f32x4 f[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) f[b] = by_token(BACK ? kVecGamma : kVecWrite, u * 2 + b);
            const f32x4 fw[2] = {f[0] * sw, f[1] * sw};
            Unit wu = pack_products(&w[u * 2], fw);
            if constexpr (BACK) wu = -wu;
#pragma unroll
            for (int b = 0; b < NT; ++b) S.s[b] = Op::mma(u ? K.cols(b, u, lane) : kc[b], wu, S.s[b]);
            if constexpr (BACK) {
#pragma unroll
                for (int b = 0; b < 2; ++b) f[b] *= sd;
                const Unit du = pack_products(&vo[u * 2], f);
#pragma unroll
                for (int b = 0; b < NT; ++b) S.s[b] = Op::mma(Q.cols(b, u, lane), du, S.s[b]);
            }
        }
    }
    __syncthreads();  // the last chunk's results lie in LDS
    // a state's operand that is not finite, or one of V or dO, is in the state still
    // (0 times it is NaN): the head is done again
    bool bad = false;
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad = bad || !(fabsf(S.s[b][i]) < INFINITY);
    if (bad && a.nc > 0) reinterpret_cast<int*>(a.rec + p.rec.vec)[kVecBad] = 1;
    if (BACK && p.dinit) S.store(p, p.dinit + a.state, row, 4 * g);
}

// ACTIVE: the tiles it serves carry rows.  The loop's body has no branches around
// loads or stores, so that a wait for loads leaves the later stores in flight;
// beyond the last chunk it stages that one again.
template <typename T, int DK, bool VEC, bool BACK, bool ACTIVE>
__device__ __forceinline__ void scan16_serve(const BwdParams& p, const ScanAt& a, int tid, char* lds) {
    using L = Scan16Lds<DK>;
    constexpr int NT = DK / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    // half the columns of two tiles' results, and V or dO of one of them
    const int pair = wave & 1, half = wave >> 1, mine = 2 * pair + half, tile = a.part * 4 + mine, first = a.part * 2 + pair;
    const SeqAt<T> at = seq_at<T>(p, a.seq, a.h, BACK);
    auto turn = [&](int t) { return lds + L::kTurn + (2 * pair + t) * (L::kTurnS + L::kTurnW); };
    const RowMat<OpF16, DK> ts0{turn(0)}, ts1{turn(1)};
    const RowMat<OpF16, 64> tw0{turn(0) + L::kTurnS}, tw1{turn(1) + L::kTurnS};
    auto chunk = [&](int c) { return BACK ? a.nc - 1 - min(c, a.nc - 1) : min(c, a.nc - 1); };
    ScanStage<OpF16, T, DK, VEC, BACK> st;
    TileRuns<T, VEC> in;
    auto load = [&](int c) {
        st.load(p, at, chunk(c), a.rec + chunk(c) * a.stride, tid);
        if constexpr (ACTIVE) in.load(p, at, chunk(c), tile, lane);
    };
    auto store = [&](int c) { st.store(lds + (c & 1) * L::Buf::kBytes, tid); };
    auto store_rest = [&](int c) {
        st.store_back(lds + (c & 1) * L::Buf::kBytes, tid);
        if constexpr (ACTIVE) {
            const int slot = (c & 1) * 4 + mine;
            in.put(lds + L::kTiles + slot * L::kTile, lane);
            const int e = bits_exp(in.max_bits()) + 1;  // below 2^e
            if (lane == 0) reinterpret_cast<int*>(lds + L::kExps)[slot] = e;
        }
    };
    u16x2 top_w = {0, 0};
    auto results = [&](int c) {
        if constexpr (ACTIVE) {
            char* rec = a.rec + chunk(c) * a.stride;
            u16x2 top_s = {0, 0};  // not needed: the state's operands are in the state
            store_turned<NT / 2>(ts0, ts1, rec + (BACK ? p.rec.ds1 : p.rec.s0) + first * NT * 1024, half * (NT / 2), lane,
                                 top_s);
            store_turned<2>(tw0, tw1, rec + (BACK ? p.rec.x : p.rec.w) + first * 4 * 1024, half * 2, lane, top_w);
        }
    };
    if (a.nc > 0) {
        load(0);
        store(0);
        store_rest(0);
        load(1);
        __syncthreads();  // A
        store(1);
        __syncthreads();  // B
        store_rest(1);
        load(2);
        for (int c = 1; c < a.nc; ++c) {
            __syncthreads();  // A
            results(c - 1);
            store(c + 1);
            __syncthreads();  // B
            store_rest(c + 1);
            load(c + 2);
        }
    }
    __syncthreads();
    if (a.nc > 0) results(a.nc - 1);
    if (max(top_w.x, top_w.y) >= 0x7c00) reinterpret_cast<int*>(a.rec + p.rec.vec)[kVecBad] = 1;  // not finite in fp16
}

template <typename T, int DK, bool VEC>
__global__ __launch_bounds__(512) void bwd_scan16_kernel(BwdParams p, int splits) {
    __shared__ __align__(16) char lds[Scan16Lds<DK>::kBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    ScanAt a;
    if (!scan_at(p, splits, a)) return;
    const int tile = a.part * 4 + wave;
    auto serve = [&](auto back, auto active) {
        scan16_serve<T, DK, VEC, back.value, active.value>(p, a, threadIdx.x - 256, lds);
    };
    if (wave >= 4) {
        const bool active = a.part * 4 + 2 * (wave & 1) < p.dvt;  // dvt is even
        if (a.back) active ? serve(std::true_type{}, std::true_type{}) : serve(std::true_type{}, std::false_type{});
        else active ? serve(std::false_type{}, std::true_type{}) : serve(std::false_type{}, std::false_type{});
    } else if (tile < p.dvt) {
        if (a.back) scan16_carry<T, DK, VEC, true>(p, a, tile, wave, lane, lds);
        else scan16_carry<T, DK, VEC, false>(p, a, tile, wave, lane, lds);
    } else {  // no rows: the barriers alone
        for (int c = 0; c < 2 * a.nc + 1; ++c) __syncthreads();
    }
}

// fp32.  An fp32 product takes its SIMD 16 times as long as an fp16 one, and few
// heads leave most SIMDs idle, so a tile has four waves: each owns a quarter of
// the state's columns (its update, 1/4 of the products) and a block of 16 tokens
// (x, w and y), and they exchange state, w and y through LDS.  2 x 1003 tokens, 8
// heads, d = 64: 53 us, where one wave a tile took 106.
template <int DK, int TILES>
struct Scan32Lds {
    using Buf = ScanBuf<OpF32, DK>;
    static constexpr int kTile = RowMat<OpF32, 16>::bytes(64), kW = RowMat<OpF32, 64>::bytes(16);
    static constexpr int kS = RowMat<OpF32, DK>::bytes(16);
    // by tile: its columns of V or dO, which y overlays, then w and the state
    static constexpr int kWAt = std::max(kTile, kW), kSAt = kWAt + kW, kEach = kSAt + kS;
    static constexpr int kTiles = Buf::kBytes, kBytes = kTiles + TILES * kEach;
};
// d_k columns of the state that one of a tile's four waves carries
template <int DK>
constexpr int kOwn = DK > 64 ? DK / 4 : 16;

// One chunk of a tile, by its four waves (`w`); every wave of the workgroup
// calls it.  The operands, the tile's columns of V or dO and its state lie in
// LDS, behind a barrier.
template <typename T, int DK, int TILES, bool BACK>
__device__ __forceinline__ void scan32_chunk(const BwdParams& p, State<OpF32, kOwn<DK>>& S, char* rec, char* buf,
                                             char* mine, int tile, int w, int lane) {
    using Op = OpF32;
    using L = Scan32Lds<DK, TILES>;
    using Buf = typename L::Buf;
    constexpr int NT = DK / 16, NO = kOwn<DK> / 16;
    const int g = lane >> 4, m = lane & 15;
    const bool own = w * NO < NT;
    const RowMat<Op, DK> K{buf + Buf::kK}, Q{buf + Buf::kQ}, turn_s{mine + L::kSAt};
    const RowMat<Op, 64> Tm{buf + Buf::kT}, P{buf + Buf::kP}, turn_w{mine + L::kWAt}, turn_y{mine};
    const float* vec = reinterpret_cast<const float*>(buf + Buf::kVec);
    auto by_token = [&](int v, int b) { return *reinterpret_cast<const f32x4*>(vec + v + 16 * b + 4 * g); };
    // column tiles of a turned matrix to the record, `n` of them from `first`
    auto keep = [&](const auto& turn, char* base, int tiles, int first, int n) {
        char* o = base + ((size_t)tile * tiles + first) * 1024 + lane * 16;
        for (int b = 0; b < n; ++b) *reinterpret_cast<f32x4*>(o + b * 1024) = turn.col4(first + b, 0, lane);
    };
    f32x4 vo[4], x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    TileRuns<T, true>::get(mine, vo, lane);
#pragma unroll
    for (int i = 0; i < NT; ++i) x = Op::mma(K.blocks(16 * w + m, i, g), turn_s.blocks(m, i, g), x);
    if (own) keep(turn_s, rec + (BACK ? p.rec.ds1 : p.rec.s0), NT, w * NO, NO);
    if constexpr (!BACK) {
        f32x4 v = vo[0];
#pragma unroll
        for (int u = 1; u < 4; ++u) v = w == u ? vo[u] : v;
        x = v - by_token(kVecGamma, w) * x;
    } else {
        f32x4 z = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (u >= w) z = Op::mma(P.cols(w, u, lane), vo[u], z);
        x = by_token(kVecBeta, w) * z + by_token(kVecWrite, w) * x;
    }
    turn_w.put_unit(m, w, g, x);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        if (!BACK && u <= w) y = Op::mma(Tm.blocks(16 * w + m, u, g), turn_w.blocks(m, u, g), y);
        if (BACK && u >= w) y = Op::mma(Tm.cols(w, u, lane), turn_w.blocks(m, u, g), y);
    }
    turn_y.put_unit(m, w, g, y);
    __syncthreads();
    keep(turn_y, rec + (BACK ? p.rec.x : p.rec.w), 4, w, 1);
    if (!own) return;
    const float gc = vec[kVecGc];
#pragma unroll
    for (int b = 0; b < NO; ++b) S.s[b] *= gc;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const f32x4 f = by_token(BACK ? kVecGamma : kVecWrite, u), yu = turn_y.blocks(m, u, g);
        const f32x4 wu = BACK ? -yu * f : yu * f, du = vo[u] * f;
#pragma unroll
        for (int b = 0; b < NO; ++b) S.s[b] = Op::mma(K.cols(w * NO + b, u, lane), wu, S.s[b]);
        if constexpr (BACK) {
#pragma unroll
            for (int b = 0; b < NO; ++b) S.s[b] = Op::mma(Q.cols(w * NO + b, u, lane), du, S.s[b]);
        }
    }
#pragma unroll
    for (int b = 0; b < NO; ++b) turn_s.put_unit(m, w * NO + b, g, S.s[b]);
}

template <typename T, int DK, bool VEC, int TILES, bool BACK>
__device__ __forceinline__ void scan32(const BwdParams& p, const ScanAt& a, char* lds) {
    using L = Scan32Lds<DK, TILES>;
    constexpr int NO = kOwn<DK> / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3, g = lane >> 4;
    const int tile = a.part * TILES + (wave >> 2), row = 16 * tile + (lane & 15), c0 = kOwn<DK> * w + 4 * g;
    const bool own = w * NO < DK / 16;
    const float* from = BACK ? p.dfinal : p.init;
    const SeqAt<T> at = seq_at<T>(p, a.seq, a.h, BACK);
    char* mine = lds + L::kTiles + (wave >> 2) * L::kEach;
    State<OpF32, kOwn<DK>> S;
    S.load(p, from ? from + a.state : nullptr, row, c0);
    const RowMat<OpF32, DK> turn_s{mine + L::kSAt};
    if (own)
#pragma unroll
        for (int b = 0; b < NO; ++b) turn_s.put_unit(lane & 15, w * NO + b, g, S.s[b]);
    auto chunk = [&](int c) { return BACK ? a.nc - 1 - min(c, a.nc - 1) : min(c, a.nc - 1); };
    ScanStage<OpF32, T, DK, VEC, BACK, 256 * TILES> st;
    TileRuns<T, VEC, 256> in;
    if (a.nc > 0) {
        st.load(p, at, chunk(0), a.rec + chunk(0) * a.stride, threadIdx.x);
        in.load(p, at, chunk(0), tile, threadIdx.x & 255);
    }
    for (int c = 0; c < a.nc; ++c) {
        st.store(lds, threadIdx.x);
        st.store_back(lds, threadIdx.x);
        in.put(mine, threadIdx.x & 255);
        __syncthreads();
        st.load(p, at, chunk(c + 1), a.rec + chunk(c + 1) * a.stride, threadIdx.x);
        in.load(p, at, chunk(c + 1), tile, threadIdx.x & 255);
        scan32_chunk<T, DK, TILES, BACK>(p, S, a.rec + chunk(c) * a.stride, lds, mine, tile, w, lane);
        __syncthreads();
    }
    if (BACK && p.dinit && own) S.store(p, p.dinit + a.state, row, c0);
}

template <typename T, int DK, bool VEC, int TILES>
__global__ __launch_bounds__(256 * TILES) void bwd_scan32_kernel(BwdParams p, int splits) {
    __shared__ __align__(16) char lds[Scan32Lds<DK, TILES>::kBytes];
    ScanAt a;
    if (!scan_at(p, splits, a)) return;
    if (a.back) scan32<T, DK, VEC, TILES, true>(p, a, lds);
    else scan32<T, DK, VEC, TILES, false>(p, a, lds);
}

// ----------------------------------------------------------------- grad
// One (chunk, head) per workgroup of four waves; wave w owns token tile w of
// every product.  Tiles of d_v, one unit wide, pass through two buffers of LDS;
// the products over d_v stay in accumulators (dO S0, dX S0, W dS1 by d_k, and
// dO W^T and dX W^T: the tiles up to the diagonal with W's rows as rows, those
// from it on with W's rows as columns).  Then K and Q take the tiles' place and
// the 64 x 64 products follow, right operands from the accumulators.  The
// tiles' exponents differ; right operands are scaled to the largest.
// 202 us for 0.84 GB at 4 x 4096 tokens, 16 heads, d = 128, bf16: 80 % of a
// copy's rate, two workgroups a CU (as first built, with one, 633 us).

template <class Op, int DK>
struct GradLds {
    static constexpr int kTdv = 16 * Op::kBlocks;
    static constexpr int kSt = DK / 16 * 1024, kTok = 4 * 1024;
    static constexpr int kS0 = 0, kDs = kSt, kW = 2 * kSt, kX = kW + kTok, kO = kX + kTok, kBuf = kO + kTok;
    static constexpr int kRow = RowMat<Op, DK>::bytes(64), kSq = 64 * 64 * 4;
    static constexpr int kKr = 0, kQr = kRow, kM = 2 * kRow, kKqEnd = kM + kSq;
    static constexpr int kGates = 2 * kBuf > kKqEnd ? 2 * kBuf : kKqEnd;
    static constexpr int kVecs = kGates + int(sizeof(Gates));  // a [64], kw [64], partial sums [3][256], reductions [16]
    static constexpr int kBytes = kVecs + (128 + 768 + 16) * 4;
};

// the dot products of a unit's blocks
__device__ __forceinline__ void unit_dots(const f16x8& a, const f16x8& b, float (&s)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        s[h] = __builtin_amdgcn_fdot2(f16x2{a[4 * h], a[4 * h + 1]}, f16x2{b[4 * h], b[4 * h + 1]}, 0.f, false);
        s[h] = __builtin_amdgcn_fdot2(f16x2{a[4 * h + 2], a[4 * h + 3]}, f16x2{b[4 * h + 2], b[4 * h + 3]}, s[h], false);
    }
}
__device__ __forceinline__ void unit_dots(const f32x4& a, const f32x4& b, float (&s)[1]) {
    s[0] = a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
}
// The exponent of the largest value of a column of four tiles, whose rows lie in
// the lanes m, 16 + m, 32 + m and 48 + m.
__device__ __forceinline__ int column_exp(const f32x4 (&x)[4]) {
    float mx = 0.f;
#pragma unroll
    for (int b = 0; b < 4; ++b)
        mx = fmaxf(fmaxf(fmaxf(mx, fabsf(x[b][0])), fabsf(x[b][1])), fmaxf(fabsf(x[b][2]), fabsf(x[b][3])));
    mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
    return bits_exp(bits_abs(fmaxf(mx, __shfl_xor(mx, 32, kWave))));
}
// a unit with its two blocks times 2^d0 and 2^d1, d <= 0
__device__ __forceinline__ f16x8 shift_unit(f16x8 u, int d0, int d1) {
    const _Float16 f = (_Float16)exp2i(d0), h = (_Float16)exp2i(d1);
    const f16x8 s = {f, f, f, f, h, h, h, h};
    return u * s;
}
__device__ __forceinline__ f32x4 shift_unit(const f32x4& u, int, int) { return u; }

template <class Op, typename T, int DK, bool VEC>
__device__ __forceinline__ void grad_chunk(const BwdParams& p, const ChunkAt& at, int h, const char* rec, char* lds) {
    using Unit = typename Op::Unit;
    using L = GradLds<Op, DK>;
    constexpr int NT = DK / 16, NBK = Op::kBlocks, NU = NT / NBK, NKT = 4 / NBK, R = kRun<T>;
    constexpr int NS = (NT * 64 + 255) / 256;      // 16-byte pieces of S0's tile per thread
    constexpr int NO = 64 * L::kTdv / R / 256;     // runs of dO's tile per thread
    constexpr int NK = 64 * DK / R / 256;          // runs of K (and of Q) per thread
    const int tid = thread_index(), wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4,
              m = lane & 15;
    const RowMat<Op, DK> Kr{lds + L::kKr}, Qr{lds + L::kQr};
    float* M = reinterpret_cast<float*>(lds + L::kM);
    Gates& gs = *reinterpret_cast<Gates*>(lds + L::kGates);
    float* va = reinterpret_cast<float*>(lds + L::kVecs);  // a
    float* vk = va + 64;                                   // tail k.(W dS1)
    float* part = va + 128;                                // [3][256]
    float* red = part + 768;                               // [16]
    const int* exps = reinterpret_cast<const int*>(rec + p.rec.vec);
    const long ldk = (long)p.heads * p.d_k, ldv = (long)p.heads * p.d_v;
    const long ok = at.t0 * ldk + (long)h * p.d_k, ov = at.t0 * ldv + (long)h * p.d_v;
    const T* op = static_cast<const T*>(p.dout) + ov;
    T* dvp = static_cast<T*>(p.dv) + ov;
    const int tiles = (p.dvt + NBK - 1) / NBK;

    // the tiles of d_v on their way to LDS
    constexpr int NOR = NO > 0 ? NO : 1;
    u32x4 rs[NS], rd[NS], rw, rx, ro[NOR];
    auto load_tile = [&](int t) {
        const u32x4* s0 = reinterpret_cast<const u32x4*>(rec + p.rec.s0) + (long)t * NT * 64;
        const u32x4* d1 = reinterpret_cast<const u32x4*>(rec + p.rec.ds1) + (long)t * NT * 64;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int id = min(tid + 256 * i, NT * 64 - 1);
            rs[i] = s0[id];
            rd[i] = d1[id];
        }
        rw = reinterpret_cast<const u32x4*>(rec + p.rec.w)[(long)t * 256 + tid];
        rx = reinterpret_cast<const u32x4*>(rec + p.rec.x)[(long)t * 256 + tid];
#pragma unroll
        for (int i = 0; i < NOR; ++i) {
            const int id = tid + 256 * i, tk = id / (L::kTdv / R), c = t * L::kTdv + id % (L::kTdv / R) * R;
            ro[i] = load_run<T, VEC>(op + tk * ldv + c, tk < at.n && c < p.d_v, p.d_v - c);
        }
    };
    load_tile(0);
    if (wave == 0) load_gates(p, at, h, gs, lane);

    // exponents: lane t holds those of d_v tile t; e.. the largest of a product's
    int xs = 0, xd = 0, xw = 0, xx = 0, eo = 0, es = 0, ed = 0, exs = 0, ew = 0, exw = 0, ek = 0, eq = 0;
    if constexpr (Op::kScaled) {
        const bool in = lane < p.dvt;
        xs = in ? exps[kExpS + lane] : -1000, xd = in ? exps[kExpD + lane] : -1000;
        xw = in ? exps[kExpW + lane] : -1000, xx = in ? exps[kExpX + lane] : -1000;
        auto top = [](int x) { return wave_max_bits(x + 8192) - 8192; };
        eo = top(in ? exps[kExpO + lane] : -1000);
        es = top(xs), ed = top(xw + xd), exs = top(xx + xs), ew = top(xw), exw = top(xx + xw);
        ek = exps[kVecEK], eq = exps[kVecEQ];
    }
    const float so = exp2i(-eo);

    f32x4 zq[NT], zk[NT], zw[NT], e1[5], e2[5];  // [4]: the diagonal tile with W's rows as columns
#pragma unroll
    for (int b = 0; b < NT; ++b) zq[b] = zk[b] = zw[b] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < 5; ++b) e1[b] = e2[b] = f32x4{0, 0, 0, 0};
    float ip = 0.f;  // <dS1, S0>

    auto tile = [&](int t, auto ahead) {
        char* buf = lds + (t & 1) * L::kBuf;
        int s0e = 0, s1e = 0, d0e = 0, d1e = 0, w0e = 0, w1e = 0, x0e = 0, x1e = 0;
        if constexpr (Op::kScaled) {
            s0e = __builtin_amdgcn_readlane(xs, 2 * t), s1e = __builtin_amdgcn_readlane(xs, 2 * t + 1);
            d0e = __builtin_amdgcn_readlane(xd, 2 * t), d1e = __builtin_amdgcn_readlane(xd, 2 * t + 1);
            w0e = __builtin_amdgcn_readlane(xw, 2 * t), w1e = __builtin_amdgcn_readlane(xw, 2 * t + 1);
            x0e = __builtin_amdgcn_readlane(xx, 2 * t), x1e = __builtin_amdgcn_readlane(xx, 2 * t + 1);
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int id = tid + 256 * i;
            if (NT * 64 % 256 == 0 || id < NT * 64) {
                reinterpret_cast<u32x4*>(buf + L::kS0)[id] = rs[i];
                reinterpret_cast<u32x4*>(buf + L::kDs)[id] = rd[i];
                float d[NBK];
                unit_dots(__builtin_bit_cast(Unit, rs[i]), __builtin_bit_cast(Unit, rd[i]), d);
                ip += d[0] * exp2i(s0e) * exp2i(d0e);
                if constexpr (NBK == 2) ip += d[NBK - 1] * exp2i(s1e) * exp2i(d1e);
            }
        }
        reinterpret_cast<u32x4*>(buf + L::kW)[tid] = rw;
        reinterpret_cast<u32x4*>(buf + L::kX)[tid] = rx;
#pragma unroll
        for (int i = 0; i < NOR; ++i) {
            const int id = tid + 256 * i, tk = id / (L::kTdv / R), c = id % (L::kTdv / R) * R;
            if (NO == 0 && tk >= 64) break;  // half as many runs as threads
            float x[R];
            unpack_run<T>(ro[i], x);
            // unit (token tile; d_v): block c / 16, lanes g = c / 4 % 4 and, of eight columns, the next
            char* o = buf + L::kO + (tk >> 4) * 1024 + ((c >> 2 & 3) * 16 + (tk & 15)) * 16;
            if constexpr (Op::kScaled) {
                o += (c >> 4) * 8;
#pragma unroll
                for (int j = 0; j < R; j += 4) {
                    const f16x4 y = {(_Float16)(x[j] * so), (_Float16)(x[j + 1] * so), (_Float16)(x[j + 2] * so),
                                     (_Float16)(x[j + 3] * so)};
                    *reinterpret_cast<f16x4*>(o + j / 4 * 256) = y;
                }
            } else {
#pragma unroll
                for (int j = 0; j < R; j += 4)
                    *reinterpret_cast<f32x4*>(o + j / 4 * 256) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
            }
        }
        __syncthreads();
        ahead();
        // dV = dX
        {
            constexpr int NP = 64 * L::kTdv / 8;  // pieces of eight columns
            static_assert(NP <= 256, "");
            if (NP == 256 || tid < NP) {
                const int tk = tid / (L::kTdv / 8), c = tid % (L::kTdv / 8) * 8;
                const char* o = buf + L::kX + (tk >> 4) * 1024 + ((c >> 2 & 3) * 16 + (tk & 15)) * 16;
                float x[8];
                if constexpr (Op::kScaled) {
                    const float f = exp2i(c < 16 ? x0e : x1e);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        x[j] = (float)reinterpret_cast<const f16x4*>(o + (c >> 4) * 8 + j / 4 * 256)[0][j & 3] * f;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = reinterpret_cast<const f32x4*>(o + j / 4 * 256)[0][j & 3];
                }
                const int col = t * L::kTdv + c;
                if (tk < at.n) {
                    if constexpr (VEC && sizeof(T) == 4) {  // rows are whole runs of four
                        const float a[4] = {x[0], x[1], x[2], x[3]}, b[4] = {x[4], x[5], x[6], x[7]};
                        store_run<T, true, 4>(dvp + tk * ldv + col, p.d_v - col, a);
                        store_run<T, true, 4>(dvp + tk * ldv + col + 4, p.d_v - col - 4, b);
                    } else {
                        store_run<T, VEC, 8>(dvp + tk * ldv + col, p.d_v - col, x);
                    }
                }
            }
        }
        const Unit bo = lds_unit<Op>(buf + L::kO, wave, lane), bx = lds_unit<Op>(buf + L::kX, wave, lane),
                   bw = lds_unit<Op>(buf + L::kW, wave, lane);
        {
            const Unit b1 = shift_unit(bo, s0e - es, s1e - es);
            const Unit b2 = shift_unit(bx, x0e + s0e - exs, x1e + s1e - exs);
            const Unit b3 = shift_unit(bw, w0e + d0e - ed, w1e + d1e - ed);
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                const Unit a = lds_unit<Op>(buf + L::kS0, b, lane);
                zq[b] = Op::mma(a, b1, zq[b]);
                zk[b] = Op::mma(a, b2, zk[b]);
                zw[b] = Op::mma(lds_unit<Op>(buf + L::kDs, b, lane), b3, zw[b]);
            }
        }
        {
            const Unit b1 = shift_unit(bo, w0e - ew, w1e - ew), b2 = shift_unit(bx, x0e + w0e - exw, x1e + w1e - exw);
            const Unit c1 = shift_unit(bw, w0e - ew, w1e - ew), c2 = shift_unit(bw, x0e + w0e - exw, x1e + w1e - exw);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (b <= wave) {
                    const Unit a = lds_unit<Op>(buf + L::kW, b, lane);
                    e1[b] = Op::mma(a, b1, e1[b]);
                    e2[b] = Op::mma(a, b2, e2[b]);
                } else {
                    e1[b] = Op::mma(lds_unit<Op>(buf + L::kO, b, lane), c1, e1[b]);
                    e2[b] = Op::mma(lds_unit<Op>(buf + L::kX, b, lane), c2, e2[b]);
                }
            }
            e1[4] = Op::mma(bo, c1, e1[4]);
            e2[4] = Op::mma(bx, c2, e2[4]);
        }
    };
    for (int t = 0; t + 1 < tiles; ++t) tile(t, [&] { load_tile(t + 1); });
    // K and Q by rows, where the tiles were
    u32x4 rk[NK], rq[NK];
    tile(tiles - 1, [&] {
        const T* kp = static_cast<const T*>(p.k) + ok;
        const T* qp = static_cast<const T*>(p.q) + ok;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int id = tid + 256 * i, tk = id / (DK / R), c = id % (DK / R) * R;
            const bool in = tk < at.n && c < p.d_k;
            rk[i] = load_run<T, VEC>(kp + tk * ldk + c, in, p.d_k - c);
            rq[i] = load_run<T, VEC>(qp + tk * ldk + c, in, p.d_k - c);
        }
    });
    {
        const float sk = exp2i(-ek), sq = exp2i(-eq);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int id = tid + 256 * i, tk = id / (DK / R), c = id % (DK / R) * R;
            float x[R];
            unpack_run<T>(rk[i], x);
            Kr.put(tk, c, x, sk);
            unpack_run<T>(rq[i], x);
            Qr.put(tk, c, x, sq);
        }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) ip += __shfl_xor(ip, off, kWave);
    if (lane == 0) red[wave] = ip;
    __syncthreads();

    const int tok = 16 * wave + m;  // this lane's token as a column of the products
    const float gam = gs.gamma[tok], tail = gs.tail[tok], bet = gs.beta[tok];
    const float s1 = exp2i(eo + ew), s2 = exp2i(exw);
    // q.(dO S0), k.(dX S0), k.(W dS1) of the lane's token
    float qz = 0.f, kz = 0.f, kwz = 0.f;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        f32x4 k[NBK], q[NBK];
        Op::unpack(Kr.blocks(tok, i, g), k);
        Op::unpack(Qr.blocks(tok, i, g), q);
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
    const float ah = qz * exp2i(eo + es + eq) - kz * exp2i(exs + ek);  // a without gamma
    const float kwh = kwz * exp2i(ed + ek);                            // k.(W dS1)
    if (g == 0) {
        va[tok] = gam * ah;
        vk[tok] = tail * kwh;
    }
    // rows r of tile b, column s = tok: dO_s.W_r q_s.k_r - dX_s.W_r k_s.k_r, and
    // with its decay to M
    f32x4 mh[4];
    Unit n1[NKT], n2[NKT];
    // A column of N1 or N2 is rounded to fp16 by a power of two of its own, which
    // the products' results, columns of the same token, take back: its values are
    // sums over all of d_v, without a bound within fp16's range (ones everywhere,
    // beta = 1/2, d_v = 256: 84000), and proportional to beta, without one from
    // its subnormals either.
    int en1 = 0, en2 = 0;
    auto pack_n = [&](const f32x4 (&x1)[4], const f32x4 (&x2)[4]) {
        if constexpr (Op::kScaled) {
            en1 = column_exp(x1);
            en2 = column_exp(x2);
        }
        const float f1 = exp2i(-en1), f2 = exp2i(-en2);
#pragma unroll
        for (int u = 0; u < NKT; ++u) {
            n1[u] = Op::pack(&x1[u * NBK], f1);
            n2[u] = Op::pack(&x2[u * NBK], f2);
        }
    };
    {
        const float sqk = exp2i(eq + ek) * s1, skk = exp2i(2 * ek) * s2;
        Unit uk[NU], uq[NU];
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            uk[i] = Kr.run(16 * wave, i, lane);
            uq[i] = Qr.run(16 * wave, i, lane);
        }
        f32x4 x1[4], x2[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            mh[b] = x1[b] = x2[b] = f32x4{0, 0, 0, 0};
            f32x4 y = {0, 0, 0, 0};
            if (b <= wave) {
                f32x4 qk = {0, 0, 0, 0}, kk = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    const Unit a = Kr.run(16 * b, i, lane);
                    qk = Op::mma(a, uq[i], qk);
                    kk = Op::mma(a, uk[i], kk);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 16 * b + 4 * g + j;
                    const float d = r <= tok ? decay(gs, tok, r) : 0.f, br = d * gs.beta[r];
                    const float f1 = e1[b][j] * qk[j] * sqk, f2 = e2[b][j] * kk[j] * skk;
                    mh[b][j] = r < tok ? f1 - f2 : r == tok ? f1 : 0.f;
                    y[j] = mh[b][j] * d;
                    x1[b][j] = e1[b][j] * br;
                    x2[b][j] = r < tok ? e2[b][j] * br : 0.f;
                }
            }
            *reinterpret_cast<f32x4*>(M + sq_at(tok, 16 * b + 4 * g)) = y;
        }
        pack_n(x1, x2);
    }
    // dQ = diag(gamma) dO S0 + N1 K;  K's share of dK: -N2 K - N2^T K
    const long orow = ok + tok * ldk;
    f32x4 ak[NT];
    {
        const float f1 = gam * exp2i(eo + es), f2 = exp2i(eo + ew + ek + en1), fn = -exp2i(exw + ek + en2);
        T* dq = static_cast<T*>(p.dq) + orow;
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            f32x4 c = {0, 0, 0, 0};
            ak[b] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < NKT; ++u)
                if (u * NBK <= wave) {
                    const Unit a = Kr.cols(b, u, lane);
                    c = Op::mma(a, n1[u], c);
                    ak[b] = Op::mma(a, n2[u], ak[b]);
                }
            const int col = 16 * b + 4 * g;
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = zq[b][j] * f1 + c[j] * f2;
            if (tok < at.n) store_run<T, VEC, 4>(dq + col, p.d_k - col, y);
            ak[b] *= fn;
        }
    }
    {
        f32x4 x1[4], x2[4];  // rows s of tile b, column r = tok
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            x1[b] = x2[b] = f32x4{0, 0, 0, 0};
            if (b >= wave) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int s = 16 * b + 4 * g + j;
                    const float d = s >= tok ? decay(gs, s, tok) * bet : 0.f;
                    x1[b][j] = (b == wave ? e1[4][j] : e1[b][j]) * d;
                    x2[b][j] = s > tok ? (b == wave ? e2[4][j] : e2[b][j]) * d : 0.f;
                }
            }
        }
        pack_n(x1, x2);
        const float fk = -gam * exp2i(exs), fw = bet * tail * exp2i(ed);
        const float fq = exp2i(eo + ew + eq + en1), fn = -exp2i(exw + ek + en2);
        T* dk = static_cast<T*>(p.dk) + orow;
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            f32x4 c = {0, 0, 0, 0}, n = {0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < NKT; ++u)
                if (u * NBK + NBK > wave) {
                    c = Op::mma(Qr.cols(b, u, lane), n1[u], c);
                    n = Op::mma(Kr.cols(b, u, lane), n2[u], n);
                }
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = zk[b][j] * fk + zw[b][j] * fw + c[j] * fq + (ak[b][j] + n[j] * fn);
            const int col = 16 * b + 4 * g;
            if (tok < at.n) store_run<T, VEC, 4>(dk + col, p.d_k - col, y);
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
        const double gt = t ? gs.G[t - 1] - gs.G[t] : -gs.G[0];  // -log2 alpha_t
        float x = 0.f;
        if (tok >= t) {
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 16 * b + 4 * g + j;
                    if (r < t) x += mh[b][j] * gs.beta[r] * pow2(gs.G[tok] - gs.G[r] + gt);
                }
            if (g == 0) x += ah * pow2(gs.G[tok] + gt);
        } else if (g == 0) {
            x += bet * kwh * pow2(gs.G[63] - gs.G[tok] + gt);
        }
        if (tid == 0) x += ipt * pow2(gs.G[63] + gt);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, kWave);
        if (lane == 0) red[4 + wave] = x;
        __syncthreads();
        if (tid == 0) Elem<T>::store(dgate, (long)t * p.heads, red[4] + red[5] + red[6] + red[7]);
        __syncthreads();
    }
}

template <class Op, typename T, int DK, bool VEC>
__global__ __launch_bounds__(256, Op::kScaled ? 2 : 1) void bwd_grad_kernel(BwdParams p) {
    __shared__ __align__(16) char lds[GradLds<Op, DK>::kBytes];
    const int ci = blockIdx.x / p.heads, h = blockIdx.x - ci * p.heads;
    ChunkAt at;
    if (!find_chunk(p, ci, at)) return;
    grad_chunk<Op, T, DK, VEC>(p, at, h, p.ws + (size_t)blockIdx.x * p.rec.bytes, lds);
}

// ---------------------------------------------------------------- exact
// bf16 heads whose inputs leave the fp16 path's domain (a key with |k|^2 >
// 1.03125, beta or alpha outside [0, 1], a value that is not finite) or whose
// values left fp16's range: the same steps in fp32, one workgroup per (sequence,
// head), after the others.  5 us where no head is flagged, else 2.4 us a token at
// d = 128 (4096 tokens 10 ms) and 3.9 at d_v = 256 (16384 tokens 64 ms).  The
// states before the chunks are kept in fp32 where the records' S0 and dS1 were
// (the same bytes), and everything else of the present chunk in the
// workgroup's own scratch: a record of fp32 units and the state's gradient.
template <int DK>
__device__ __forceinline__ f32x4* kept_state(char* base, int tile, int w, int lane) {
    return reinterpret_cast<f32x4*>(base) + ((size_t)tile * (DK / 16) + w * (kOwn<DK> / 16)) * 64 + lane;
}
__host__ __device__ inline size_t exact_scratch(int DK, int dvt) {
    return rec_layout(DK, dvt, 4).bytes + (size_t)DK * dvt * 16 * 4;
}

template <typename T, int DK, bool VEC>
__global__ __launch_bounds__(256, 1) void bwd_exact_kernel(BwdParams p, char* scratch) {
    using L = Scan32Lds<DK, 1>;
    constexpr int NO = kOwn<DK> / 16;
    constexpr int kPrep = PrepLds<OpF32, DK>::kBytes, kGrad = GradLds<OpF32, DK>::kBytes;
    __shared__ __align__(16) char lds[std::max(std::max(kPrep, kGrad), L::kBytes)];
    struct Thread {
        int tid, w, lane, m, g, c0;
        bool own;
    };
    auto thread = [] {
        const int tid = thread_index(), w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4;
        return Thread{tid, w, lane, lane & 15, g, kOwn<DK> * w + 4 * g, w * NO < DK / 16};
    };
    BwdParams e = p;
    e.rec = rec_layout(DK, p.dvt, 4);
    char* rec = scratch + blockIdx.x * exact_scratch(DK, p.dvt);
    char* carry = rec + e.rec.bytes;
    char* mine = lds + L::kTiles;
    const RowMat<OpF32, DK> turn_s{mine + L::kSAt};
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
        using St = State<OpF32, kOwn<DK>>;
        auto get = [&](const Thread& id, St& S, char* base, int tile) {
            const f32x4* b = kept_state<DK>(base, tile, id.w, id.lane);
            S.e = 0;
            if (id.own)
#pragma unroll
                for (int i = 0; i < NO; ++i) S.s[i] = b[i * 64];
        };
        auto put = [&](const Thread& id, const St& S, char* base, int tile) {
            f32x4* b = kept_state<DK>(base, tile, id.w, id.lane);
            if (id.own)
#pragma unroll
                for (int i = 0; i < NO; ++i) b[i * 64] = S.s[i];
        };
        // chunk c of every tile: forward from the states of `kept` to those of
        // `next`, or back over it on the states' gradients, in place
        auto step = [&](auto back, int c, char* kept, char* next) {
            const Thread id = thread();
            const SeqAt<T> from = seq_at<T>(p, seq, h, back.value);
            __syncthreads();
            ScanStage<OpF32, T, DK, VEC, back.value> sg;
            sg.load(e, from, c, rec, id.tid);
            sg.store(lds, id.tid);
            sg.store_back(lds, id.tid);
            for (int tile = 0; tile < p.dvt; ++tile) {
                St S;
                get(id, S, kept, tile);
                __syncthreads();
                TileRuns<T, VEC, 256> in;
                in.load(e, from, c, tile, id.tid);
                in.put(mine, id.tid);
                if (id.own)
#pragma unroll
                    for (int b = 0; b < NO; ++b) turn_s.put_unit(id.m, id.w * NO + b, id.g, S.s[b]);
                __syncthreads();
                scan32_chunk<T, DK, 1, back.value>(e, S, rec, lds, mine, tile, id.w, id.lane);
                if (next) put(id, S, next, tile);
            }
            __syncthreads();
        };
        // a state's tiles from where the caller has it
        auto begin = [&](const float* from, char* base) {
            const Thread id = thread();
            for (int tile = 0; tile < p.dvt; ++tile) {
                St S;
                S.load(p, from ? from + st : nullptr, 16 * tile + id.m, id.c0);
                put(id, S, base, tile);
            }
        };
        begin(p.init, first + p.rec.s0);
        for (int c = 0; c + 1 < nc; ++c) {
            char* kept = first + c * stride + p.rec.s0;
            prep_chunk<OpF32, T, DK, VEC>(e, chunk(c), h, rec, lds);
            step(std::false_type{}, c, kept, kept + stride);
        }
        begin(p.dfinal, carry);
        for (int c = nc - 1; c >= 0; --c) {
            prep_chunk<OpF32, T, DK, VEC>(e, chunk(c), h, rec, lds);
            step(std::false_type{}, c, first + c * stride + p.rec.s0, nullptr);
            step(std::true_type{}, c, carry, carry);
            grad_chunk<OpF32, T, DK, VEC>(e, chunk(c), h, rec, lds);
            __syncthreads();
        }
        if (p.dinit) {
            const Thread id = thread();
            for (int tile = 0; tile < p.dvt; ++tile) {
                St S;
                get(id, S, carry, tile);
                if (id.own) S.store(p, p.dinit + st, 16 * tile + id.m, id.c0);
            }
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

// 16-row tiles of fp32 scans up to which each has a workgroup of its own; two
// share one, its K, Q, T and P and each SIMD, where the card has more tiles than
// CUs.  d = 128, 1024 tokens, whole call: 256 tiles 140 us with one and 162 with
// two a workgroup, 512 tiles 268 and 221; d = 64: 117 and 134, 227 and 198.
constexpr int64_t kOneTile = 256;

template <class Op, typename T, int DK, bool VEC>
hipError_t go(const BwdParams& p, int64_t chunks, char* scratch, int blocks, hipStream_t st) {
    hipError_t e;
    const int64_t grid = chunks * p.heads;
    const int64_t walks = (int64_t)p.batch * p.heads * 2;
    const int tiles = Op::kScaled ? 4 : walks * p.dvt > kOneTile ? 2 : 1;
    const int splits = (p.dvt + tiles - 1) / tiles;  // dvt is even
    const int64_t scans = (walks + 7) / 8 * 8 * splits;
    if ((e = check_grid(grid, 256)) != hipSuccess) return e;
    if ((e = check_grid(scans, 512)) != hipSuccess) return e;
    if (grid > 0) {
        hipLaunchKernelGGL((bwd_prep_kernel<Op, T, DK, VEC>), dim3((unsigned)grid), dim3(256), 0, st, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (grid > 0 || p.dinit) {
        if constexpr (Op::kScaled)
            hipLaunchKernelGGL((bwd_scan16_kernel<T, DK, VEC>), dim3((unsigned)scans), dim3(512), 0, st, p, splits);
        else if (tiles == 1)
            hipLaunchKernelGGL((bwd_scan32_kernel<T, DK, VEC, 1>), dim3((unsigned)scans), dim3(256), 0, st, p, splits);
        else
            hipLaunchKernelGGL((bwd_scan32_kernel<T, DK, VEC, 2>), dim3((unsigned)scans), dim3(512), 0, st, p, splits);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (grid > 0) {
        hipLaunchKernelGGL((bwd_grad_kernel<Op, T, DK, VEC>), dim3((unsigned)grid), dim3(256), 0, st, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        if constexpr (Op::kScaled) {
            hipLaunchKernelGGL((bwd_exact_kernel<T, DK, VEC>), dim3(blocks), dim3(256), 0, st, p, scratch);
            e = hipGetLastError();
        }
    }
    return e;
}

template <class Op, typename T>
hipError_t pick_dk(const BwdParams& p, bool vec, int64_t chunks, char* scratch, int blocks, hipStream_t st) {
    switch (padded_dk(p.d_k)) {
        case 32:
            return vec ? go<Op, T, 32, true>(p, chunks, scratch, blocks, st)
                       : go<Op, T, 32, false>(p, chunks, scratch, blocks, st);
        case 64:
            return vec ? go<Op, T, 64, true>(p, chunks, scratch, blocks, st)
                       : go<Op, T, 64, false>(p, chunks, scratch, blocks, st);
        default:
            return vec ? go<Op, T, 128, true>(p, chunks, scratch, blocks, st)
                       : go<Op, T, 128, false>(p, chunks, scratch, blocks, st);
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
    p.short_rows = (int64_t)a.heads * std::max(a.d_k, a.d_v) * C64 * es < INT32_MAX;
    // rows of q, k, v, dO and of their gradients as whole runs of 16 bytes
    const int run = 16 / es;
    const bool vec = a.d_k % run == 0 && a.d_v % run == 0 && aligned(a.q, 16) && aligned(a.k, 16) && aligned(a.v, 16) &&
                     aligned(a.grad_o, 16) && aligned(a.grad_q, 16) && aligned(a.grad_k, 16) && aligned(a.grad_v, 16);
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
    if (a.dtype == RHZ_F32) return pick_dk<OpF32, float>(p, vec, chunks, scratch, exact_blocks(a), st);
    return pick_dk<OpF16, uint16_t>(p, vec, chunks, scratch, exact_blocks(a), st);
}

}  // namespace rhz
