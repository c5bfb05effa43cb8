// attn_device.hpp -- tiles and products shared by the latent attention's
// prefill and its backward passes.
//
// All products run on 32x32 matrix instructions in one arrangement: a wave
// holds 32 rows of its own side (queries in the forward pass and for dq, keys
// for dk and dv), one a lane of either half, and meets tiles of 32 rows of the
// other side from LDS.  The scores come out with the lane's row as column and
// the tile's rows in registers, register i of half g holding tile row
// (i & 3) + 8 (i >> 2) + 4 g.  These registers are at once an operand of the
// product that sums over the tile's rows, if that product counts the rows in
// the same order: its other operand, the tile transposed, is read accordingly.
// So weights and their gradients never leave a lane.
#pragma once

#include "gdr_device.hpp"

namespace rhz {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

constexpr float kLog2e = 1.4426950408889634f;

// 16 bytes: 8 bf16 or 4 fp32 values
template <typename T> constexpr int kChunkElems = 16 / int(sizeof(T));

typedef __attribute__((address_space(3))) const char lds_char;
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
    return uint32_t(reinterpret_cast<uintptr_t>((lds_char*)p));
}
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at) {
    return *reinterpret_cast<__attribute__((address_space(3))) const V*>(at);
}

// A tile of ROWS rows of D values in LDS, in panels of 128 bytes of each row.
// Chunk c of a panel's row r lies at place c ^ twist(r): two rows fill the 64
// banks, and the row's next three bits, the lowest first in weight, move its
// chunks apart, so that these all fall on different banks: one chunk of 16
// rows (operands along the row), and the 64 bytes each of 4 rows that half a
// wave reads transposed.  Read with the chunk as a constant, an address is the
// lane's own XOR a constant plus a constant.
__host__ __device__ constexpr int twist(int row) { return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1); }

template <typename T, int D, int ROWS>
struct Tile {
    static constexpr int kPanels = (D * int(sizeof(T)) + 127) / 128, kPanelBytes = ROWS * 128;
    static constexpr int kRows = ROWS;
    u32x4 chunk[kPanels * ROWS * 8];
};

// What a lane reads of tiles: along rows, and transposed.
struct LaneReads {
    uint32_t row, col;  // relative to the tile
};
template <typename T>
__device__ __forceinline__ LaneReads lane_reads(int lane) {
    const int g = lane >> 5, r = lane & 31;
    LaneReads a;
    a.row = r * 128 + ((twist(r) ^ g) << 4);
    if constexpr (sizeof(T) == 2) {
        // lane i of 16 addresses row i / 4, columns 4 (i % 4) ..; twist of row
        // 16 s + 8 part + 4 g + i / 4 is that of 4 g + i / 4, XOR part
        const int i = lane & 15, at = 4 * g + (i >> 2), c = ((lane >> 4) & 1) * 2 + ((i >> 1) & 1);
        a.col = at * 128 + ((c ^ twist(at)) << 4) + (i & 1) * 8;
    } else {
        // row (i & 3) + 8 (i >> 2) + 4 g: twist of 4 g, XOR a constant of i
        a.col = 4 * g * 128 + ((((lane & 31) >> 2) ^ twist(4 * g)) << 4) + (lane & 3) * 4;
    }
    return a;
}
// Chunk 2 i + g of row 32 u + lane % 32.
template <typename TILE>
__device__ __forceinline__ u32x4 read_row(uint32_t tile, const LaneReads& a, int u, int i) {
    return lds_read<u32x4>(((tile + a.row) ^ (((2 * i) & 7) << 4)) + (i >> 2) * TILE::kPanelBytes + u * 32 * 128);
}

// ---- products over a row's values: acc[tile row, lane's row] += A[tile row] . B[lane's row]
// One pair of chunks of either operand, the half g of the wave with chunk 2 c + g.
__device__ __forceinline__ void dot_chunks(f32x16& acc, const u32x4& a, const u32x4& b, uint16_t) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0,
                                                  0);
}
__device__ __forceinline__ void dot_chunks(f32x16& acc, const u32x4& a, const u32x4& b, float) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int t = 0; t < 4; ++t) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[t], y[t], acc, 0, 0, 0);
}

// ---- products over the tile's rows: acc[column d, lane's row] += sum_r tile[r][d] p[r, lane's row]
// p of 32 tile rows as the operand: registers 8 s .. 8 s + 7 are step s.  Where the
// tensors are bf16 the weights (and in the backward pass their gradients) are
// rounded to it: an fp32 product takes sixteen times as long.  The error against 64
// bits grows from 1.6 to 1.8e-3 of a result, its own rounding, to 1.7 to 2.4e-3.
template <typename T> struct Weights;
template <> struct Weights<uint16_t> {
    bf16x8 x[2];
    __device__ __forceinline__ void set(const f32x16& p) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] = (__bf16)p[8 * s + j];
    }
};
template <> struct Weights<float> {
    f32x16 x;
    __device__ __forceinline__ void set(const f32x16& p) { x = p; }
};

// Columns 32 dt .. 32 dt + 31 of tile rows 32 u .. 32 u + 31, transposed, the
// lane with column 32 dt + lane % 32.
template <typename T> struct Columns;
template <> struct Columns<uint16_t> {
    bf16x8 x[2];
    template <typename TILE>
    __device__ __forceinline__ void load(uint32_t tile, const LaneReads& a, int u, int dt) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            s16x4_t h[2];
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const uint32_t at = ((tile + a.col) ^ ((4 * (dt & 1) ^ part) << 4)) + (dt >> 1) * TILE::kPanelBytes +
                                    (32 * u + 16 * s + 8 * part) * 128;
                h[part] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4_t*>(at));
            }
            struct { s16x4_t lo, hi; } both = {h[0], h[1]};
            x[s] = __builtin_bit_cast(bf16x8, both);
        }
    }
};
template <> struct Columns<float> {
    f32x16 x;
    template <typename TILE>
    __device__ __forceinline__ void load(uint32_t tile, const LaneReads& a, int u, int dt) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = (i & 3) + 8 * (i >> 2);
            x[i] = lds_read<float>(((tile + a.col) ^ (twist(r) << 4)) + dt * TILE::kPanelBytes + (32 * u + r) * 128);
        }
    }
};
__device__ __forceinline__ void sum_rows(f32x16& acc, const Columns<uint16_t>& a, const Weights<uint16_t>& p) {
#pragma unroll
    for (int s = 0; s < 2; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.x[s], p.x[s], acc, 0, 0, 0);
}
__device__ __forceinline__ void sum_rows(f32x16& acc, const Columns<float>& a, const Weights<float>& p) {
#pragma unroll
    for (int i = 0; i < 16; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x[i], p.x[i], acc, 0, 0, 0);
}

// ---- global memory
// Where a tile's rows come from: `cols` values of rows `stride` elements apart,
// and `extra` more of a second tensor behind them (the rotary key; cols and
// extra whole chunks unless !VEC).
template <typename T>
struct Rows {
    const T* p;
    const T* extra_p;
    long stride, extra_stride;
    int cols, extra;
};

// One chunk of row row0 + r, zero beyond the columns.  VEC: everything aligned
// to 16 bytes and of whole chunks.  row0 is the same for all lanes; the host has
// checked that 128 rows' offsets stay in 32 bits.
template <typename T, bool VEC>
__device__ __forceinline__ u32x4 load_chunk(const Rows<T>& s, long row0, int r, int chunk) {
    constexpr int E = kChunkElems<T>;
    const int d = chunk * E;
    const T* first = s.p + row0 * s.stride;
    const T* second = s.extra_p + row0 * s.extra_stride;
    if constexpr (VEC) {
        // the address stays in the row where there is no value
        const bool there = d < s.cols + s.extra, behind = there && d >= s.cols;
        const T* p = behind ? second : first;
        const int at = behind ? r * int(s.extra_stride) + (d - s.cols) : r * int(s.stride) + (there ? d : 0);
        const u32x4 v = *reinterpret_cast<const u32x4*>(p + at);
        return there ? v : u32x4{0, 0, 0, 0};
    } else {
        T e[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int c = d + i;
            e[i] = c < s.cols ? first[r * int(s.stride) + c]
                              : c < s.cols + s.extra ? second[r * int(s.extra_stride) + (c - s.cols)] : T(0);
        }
        u32x4 v;
        __builtin_memcpy(&v, e, 16);
        return v;
    }
}

// 16 (or 4) bytes a lane from memory, base + its offset + OFF, to LDS, lane i's
// at lds + 16 i (4 i); base and lds are the same for all lanes (OFF counts in LDS
// too, which is taken back).  Nothing waits for it but landed(): the compiler,
// which would make every later LDS read wait for a load that it knows of, does
// not see these.  Its own waits count them along, which makes them longer, never
// shorter.
template <int OFF>
__device__ __forceinline__ void load_to_lds16(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3" ::"{m0}"(lds - OFF), "v"(off), "s"(base), "n"(OFF)
                 : "memory");
}
__device__ __forceinline__ void load_to_lds4(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, %2" ::"{m0}"(lds), "v"(off), "s"(base) : "memory");
}
// Until every wave's loads into LDS have landed and its LDS reads are done.
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Waits for all but the last N loads of a wave.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// LDS reads and writes done, by all waves; loads on their way stay so.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// A wave's own loads and reads.
__device__ __forceinline__ void wave_landed() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
// A wave's own LDS reads are done: what it read may be written over.
__device__ __forceinline__ void wave_read() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Makes the compiler wait for a value here: a wait that it put off into a loop
// would count the loop's own loads into LDS along, every time.
template <typename V>
__device__ __forceinline__ void settle(V& v) { asm volatile("" : "+v"(v)); }

// Moves tiles of ROWS rows of D values into LDS with NT threads.  Rows beyond
// the valid ones repeat the last: whoever sums over a tile's rows leaves them
// out.  Chunks beyond the columns are zero: clear() once, then never written.
template <typename T, int D, int ROWS, int NT, bool VEC>
struct Mover {
    using TILE = Tile<T, D, ROWS>;
    static constexpr int E = kChunkElems<T>, COUNT = ROWS * 8 / NT, PANELS = TILE::kPanels;
    static_assert(COUNT * NT == ROWS * 8, "whole chunks for every thread");
    Rows<T> s;
    int tid;
    bool whole;                          // every panel is full and of one tensor
    uint32_t off[COUNT], off_behind[COUNT];  // of the thread's chunks of a full tile, from either tensor

    __device__ __forceinline__ Mover(const Rows<T>& rows, int t) : s(rows), tid(t) {
        whole = s.cols % (8 * E) == 0 && s.cols + s.extra == PANELS * 8 * E;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < COUNT; ++i) place(i, ROWS, off[i], off_behind[i]);
        }
    }
    __device__ __forceinline__ void place(int i, int valid, uint32_t& first, uint32_t& behind) const {
        const int r = (i * NT + tid) >> 3, c = (tid & 7) ^ twist(r), rr = min(r, valid - 1);
        first = (rr * int(s.stride) + c * E) * int(sizeof(T));
        behind = (rr * int(s.extra_stride) + c * E) * int(sizeof(T));
    }
    __device__ __forceinline__ void clear(TILE& t) const {
        if (s.cols + s.extra >= PANELS * 8 * E) return;
        for (int at = tid; at < PANELS * ROWS * 8; at += NT) t.chunk[at] = u32x4{0, 0, 0, 0};
    }
    // Panels P .. of the thread's chunk i.
    template <int P>
    __device__ __forceinline__ void panels(int i, const T* first, const T* second, uint32_t at, uint32_t at_behind,
                                           uint32_t lds) const {
        if constexpr (P < PANELS) {
            constexpr int d0 = P * 8 * E;
            const uint32_t to = lds + P * TILE::kPanelBytes;
            if (whole) {
                const bool behind = d0 >= s.cols;
                load_to_lds16<P * 128>(behind ? second : first, behind ? at_behind : at, to);
            } else {
                const int d = d0 + ((tid & 7) ^ twist((i * NT + tid) >> 3)) * E;
                if (d < s.cols) load_to_lds16<P * 128>(first, at, to);
                if (d >= s.cols && d < s.cols + s.extra) load_to_lds16<P * 128>(second, at_behind, to);
            }
            panels<P + 1>(i, first, second, at, at_behind, lds);
        }
    }
    // rows row0 .. of which `valid` (>= 1) are there
    __device__ __forceinline__ void start(long row0, int valid, TILE& t) const {
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const T* first = s.p + row0 * s.stride;
        const T* second = s.extra_p + row0 * s.extra_stride - s.cols;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            if constexpr (VEC) {
                uint32_t at = off[i], at_behind = off_behind[i];
                if (valid < ROWS) place(i, valid, at, at_behind);
                panels<0>(i, first, second, at, at_behind, lds_offset(&t.chunk[0]) + (i * NT + wave * 64) * 16);
            } else {
                const int r = (i * NT + tid) >> 3, c = (tid & 7) ^ twist(r);
#pragma unroll 1
                for (int p = 0; p < PANELS; ++p)
                    t.chunk[p * ROWS * 8 + i * NT + tid] = load_chunk<T, false>(s, row0, min(r, valid - 1), p * 8 + c);
            }
        }
    }
};

// acc[column, lane's row] of 32 columns from d0 to row `out` of D values, times f.
template <typename T>
__device__ __forceinline__ void store_columns(T* out, const f32x16& acc, int d0, int D, float f, bool vec, int lane) {
    const int g = lane >> 5;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int d = d0 + 8 * q + 4 * g;
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = acc[4 * q + j] * f;
        if (vec) {
            if (d < D) {
                if constexpr (sizeof(T) == 4)
                    *reinterpret_cast<f32x4*>(out + d) = f32x4{x[0], x[1], x[2], x[3]};
                else
                    *reinterpret_cast<uint2*>(out + d) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d + j < D) Elem<T>::store(out, d + j, x[j]);
        }
    }
}

// LDS reads some steps ahead of the products that take them, pinned there: left
// to itself the scheduler reads, waits and multiplies by turns, 130 clocks of
// LDS's latency for every 32 of the product.
// acc += sum over i < N of read(i) . own[i]
template <int N, int AHEAD, typename T, typename READ>
__device__ __forceinline__ void dot_ahead(f32x16& acc, const u32x4 (&own)[N], READ read, T) {
    constexpr int A = AHEAD < N ? AHEAD : N;
    u32x4 x[A];
#pragma unroll
    for (int i = 0; i < A; ++i) x[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        dot_chunks(acc, x[i % A], own[i], T());
        if (i + A < N) x[i % A] = read(i + A);
        __builtin_amdgcn_sched_barrier(0);
    }
}
// acc[d] += tile's columns d, transposed, times p, of N column tiles; begin() may
// come long before run().
template <typename T, typename TILE, int N, int AHEAD>
struct SumAhead {
    static constexpr int A = AHEAD < N ? AHEAD : N;
    Columns<T> x[A];
    __device__ __forceinline__ void begin(uint32_t tile, const LaneReads& at, int u) {
#pragma unroll
        for (int d = 0; d < A; ++d) x[d].template load<TILE>(tile, at, u, d);
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void run(f32x16 (&acc)[N], uint32_t tile, const LaneReads& at, int u, const Weights<T>& p) {
#pragma unroll
        for (int d = 0; d < N; ++d) {
            sum_rows(acc[d], x[d % A], p);
            if (d + A < N) x[d % A].template load<TILE>(tile, at, u, d + A);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// The other half's value beside one's own.
__device__ __forceinline__ float2 both_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_of_halves(float x) {
    const float2 v = both_halves(x);
    return fmaxf(v.x, v.y);
}
__device__ __forceinline__ float sum_of_halves(float x) {
    const float2 v = both_halves(x);
    return v.x + v.y;
}

// ---- rows with an infinity or NaN
// Weight 0 does not take a hidden row out of a product if that row holds an
// infinity or NaN: whoever's result is not finite sums again over the rows that
// it sees, in plain fp32, a wave a row.  (Scores are masked one by one, so that
// the maxima, sums and weights are right in any case.)  That takes a time of its
// own for every pair of rows, so it is for rows of which it can say more than NaN:
// those whose own statistic is NaN, which only what they see can make it, are NaN
// in every column as they are, and a sum that is NaN in every column stays so.  4096
// tokens, 16 heads of 128 + 64 channels, bf16, NaN in all queries: prefill 112 ->
// 0.13 ms; in all values 2.0.  An infinity in one value that all later rows see
// takes 113 ms (finite 0.14), in one gradient of o 227 (0.45).
template <int N>
__device__ __forceinline__ uint32_t not_finite_rows(const f32x16 (&acc)[N]) {
    float sum = 0.f;  // 0 * x is NaN where x is not finite, and a sum keeps it
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum = fmaf(acc[d][i], 0.f, sum);
    const unsigned long long b = __ballot(sum != 0.f);
    return uint32_t(b) | uint32_t(b >> 32);
}
// The rows of lanes that have `is`, the same in either half.
__device__ __forceinline__ uint32_t rows_with(bool is) { return uint32_t(__ballot(is)); }
// The last of n for which is(i), -1 for none, by all lanes of a wave together.
template <typename IS>
__device__ __forceinline__ int last_with(int n, int lane, IS is) {
    for (int i0 = (n - 1) / kWave * kWave; i0 >= 0; i0 -= kWave) {
        const unsigned long long b = __ballot(i0 + lane < n && is(i0 + lane));
        if (b) return i0 + 63 - __clzll((long long)b);
    }
    return -1;
}
template <typename T>
__device__ __forceinline__ float value(const Rows<T>& s, long r, int d) {
    const T* p = d < s.cols ? s.p + r * s.stride + d : s.extra_p + (r * s.extra_stride + (d - s.cols));
    return Elem<T>::load(p, 0);
}
// Of one row (a has no second tensor) with another.
template <typename T>
__device__ __forceinline__ float dot_rows(const Rows<T>& a, long ra, const Rows<T>& b, long rb) {
    float sum = 0.f;
    const T *x = a.p + ra * a.stride, *y = b.p + rb * b.stride;
    for (int d = 0; d < b.cols; ++d) sum = fmaf(Elem<T>::load(x, d), Elem<T>::load(y, d), sum);
    x += b.cols;
    y = b.extra_p + rb * b.extra_stride;
    for (int d = 0; d < b.extra; ++d) sum = fmaf(Elem<T>::load(x, d), Elem<T>::load(y, d), sum);
    return sum;
}
// out(d, sum over rows j of [lo, hi) of weight(j) x(j, d)) of at most 64 N
// columns d < cols, all lanes of a wave together.
template <int N, typename WEIGHT, typename X, typename OUT>
__device__ __forceinline__ void sum_row_again(long lo, long hi, int cols, int lane, WEIGHT weight, X x, OUT out) {
    float sum[N] = {};
    for (long j0 = lo; j0 < hi; j0 += kWave) {
        const float p = j0 + lane < hi ? weight(j0 + lane) : 0.f;
        const int n = int(min(hi - j0, long(kWave)));
        for (int i = 0; i < n; ++i) {
            const float pi = __shfl(p, i, kWave);
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (lane + 64 * k < cols) sum[k] = fmaf(pi, x(j0 + i, lane + 64 * k), sum[k]);
        }
        bool nan = true;  // in all of the lane's columns
#pragma unroll
        for (int k = 0; k < N; ++k) nan = nan && (lane + 64 * k >= cols || sum[k] != sum[k]);
        if (__all(nan)) break;
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (lane + 64 * k < cols) out(lane + 64 * k, sum[k]);
}

// Token ranges of sequence `seq` on either side.
struct Range {
    int q0, nq, k0, nk;
};
__device__ __forceinline__ Range seq_range(const int* cu_q, const int* cu_k, int seq, int len_q, int len_k) {
    Range r;
    int q1, k1;
    seq_bounds(cu_q, seq, len_q, r.q0, q1);
    seq_bounds(cu_k, seq, len_k, r.k0, k1);
    r.nq = q1 - r.q0, r.nk = k1 - r.k0;
    return r;
}

// The sequence and its tile of `size` rows that number t stands for, of a pack:
// sequence b's tiles begin at number cu[b] / size + b, which leaves room for
// all of them.  Every lane of a wave takes part.
__device__ __forceinline__ void packed_tile(const int* cu, int batch, int total, int size, int t, int lane, int& seq,
                                            int& tile) {
    int before = 0;  // sequences that begin at or before t
    for (int b0 = 0; b0 < batch; b0 += kWave) {
        const int b = b0 + lane;
        const bool in = b < batch && min(max(cu[min(b, batch - 1)], 0), total) / size + b <= t;
        const int n = __popcll(__ballot(in));
        before += n;
        if (n < kWave) break;
    }
    seq = max(before - 1, 0);
    tile = t - (min(max(cu[seq], 0), total) / size + seq);
    seq = __builtin_amdgcn_readfirstlane(seq);
    tile = __builtin_amdgcn_readfirstlane(tile);
}
// How many numbers these are.
inline int64_t packed_tiles(int64_t total, int batch, int size) { return total / size + batch; }

}  // namespace rhz
