// attn_split.hip -- the latent attention's prefill and backward passes in fp32.
//
// fp32 matrix instructions take sixteen times bf16's time, so that a wave's way
// through a sequence is long and the tiles' traffic small against it.  A
// workgroup therefore has 32 rows only, and its four waves share the other
// side: each has all 32 rows on every fourth tile, with a tile of LDS of its own
// and no barrier, and their sums are added in order at the end.  Against 32 rows
// on each of four waves that share the tiles, as the bf16 kernels have it (2 x 2048
// tokens, 16 heads of 64 + 32 channels): 355 -> 213 us for the prefill, 100 of the
// 154 TFLOP/s of a large matrix product, 1205 -> 718 for the backward pass; and of
// few rows, 513, 1, 190 and 1003 tokens, 8 heads, 103 -> 42 us.
#include <algorithm>

#include "attn_params.hpp"

namespace rhz {
namespace {

using T = float;
constexpr int kThreads = kAttnThreads, kWaves = 4, kRows = 32, kTile = 32, E = 4;

// A wave's two tiles, one behind the other; the four waves' sums lie over them
// at the end, which takes as much.
template <int DA, int DB>
struct WaveTiles {
    Tile<T, DA, kTile> a;
    Tile<T, DB, kTile> b;
};

// acc of column tile d, of all waves, in the memory of their tiles.
template <int D>
struct Sums {
    f32x4* at;
    int lane;
    __device__ __forceinline__ f32x4& of(int wave, int d, int k) const { return at[((wave * D + d) * 4 + k) * kWave + lane]; }
    __device__ __forceinline__ void put(int wave, int d, const f32x16& x) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) of(wave, d, k) = f32x4{x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]};
    }
    __device__ __forceinline__ f32x16 sum(int d) const {
        f32x16 x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            f32x4 s = of(0, d, k);
#pragma unroll
            for (int w = 1; w < kWaves; ++w) s += of(w, d, k);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * k + e] = s[e];
        }
        return x;
    }
};

// --------------------------------------------------------------- the prefill
template <int DQ, int DV, bool VEC>
__global__ __launch_bounds__(kThreads) void latent_prefill_split_kernel(PrefillParams a) {
    constexpr int QC = DQ / (2 * E), VT = DV / 32;
    using TileK = Tile<T, DQ, kTile>;
    using TileV = Tile<T, DV, kTile>;
    __shared__ WaveTiles<DQ, DV> tiles[kWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const LaneReads at = lane_reads<T>(lane);
    int head, seq, tile;
    if (!place<kRows, false>(a, blockIdx.x, lane, head, seq, tile)) return;
    const Range w = seq_range(a.cu_q, a.cu_k, seq, a.len_q, a.len_k);
    if (tile * kRows >= w.nq) return;
    const int first = ((w.nq - 1) / kRows - tile) * kRows;  // the queries with the most keys go first
    const int qi = first + (lane & 31), shift = w.nk - w.nq;
    bool live = qi < w.nq;
    const int end = a.causal ? min(w.nk, min(first + kRows, w.nq) + shift) : w.nk;

    u32x4 q[QC];
    const Rows<T> qrows = {(const T*)a.q + head * a.qh, (const T*)a.q, a.qs, 0, a.d_n + a.d_r, 0};
    const Rows<T> krows = {(const T*)a.k + head * a.kh, (const T*)(a.r ? a.r : a.k), a.ks, a.rs, a.d_n, a.d_r};
    const Rows<T> vrows = {(const T*)a.v + head * a.vh, (const T*)a.v, a.vs, 0, a.d_v, 0};
#pragma unroll
    for (int c = 0; c < QC; ++c) q[c] = load_chunk<T, VEC>(qrows, (long)w.q0 + first, min(qi, w.nq - 1) - first, 2 * c + g);
#pragma unroll
    for (int c = 0; c < QC; ++c) settle(q[c]);
    WaveTiles<DQ, DV>& mine = tiles[wave];
    const Mover<T, DQ, kTile, kWave, VEC> move_a(krows, lane);
    const Mover<T, DV, kTile, kWave, VEC> move_b(vrows, lane);
    move_a.clear(mine.a), move_b.clear(mine.b);
    wave_read();
    const auto start = [&](int k0) {
        move_a.start((long)w.k0 + k0, w.nk - k0, mine.a);
        move_b.start((long)w.k0 + k0, w.nk - k0, mine.b);
    };
    f32x16 o[VT];
#pragma unroll
    for (int d = 0; d < VT; ++d) o[d] = f32x16{};
    const float c = a.scale * kLog2e;
    float m = -INFINITY, l = 0.f;
    const int seen = a.causal ? min(w.nk, qi + shift + 1) : w.nk;
    const uint32_t kt = lds_offset(&mine.a), vt = lds_offset(&mine.b);
    int k0 = wave * kTile;
    if (k0 < end) start(k0);
    for (; k0 < end; k0 += kWaves * kTile) {
        wave_landed();
        f32x16 s = {};
#pragma unroll
        for (int i = 0; i < QC; ++i) dot_chunks(s, read_row<TileK>(kt, at, 0, i), q[i], T());
        if (k0 + kTile > w.nk || (a.causal && k0 + kTile > first + shift + 1)) {
            const int left = seen - k0 - 4 * g;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if ((i & 3) + 8 * (i >> 2) >= left) s[i] = -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        top = max_of_halves(top);
        if (__any((top - m) * c > 8.f)) {
            const float up = fmaxf(m, top);
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - up) * c);
            m = up;
            l *= f;
#pragma unroll
            for (int d = 0; d < VT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -mc));
            l += s[i];
        }
        Weights<T> p;
        p.set(s);
#pragma unroll
        for (int d = 0; d < VT; ++d) {
            Columns<T> x;
            x.template load<TileV>(vt, at, 0, d);
            sum_rows(o[d], x, p);
        }
        wave_read();
        if (k0 + kWaves * kTile < end) start(k0 + kWaves * kTile);
    }
    // the waves' sums at their common maximum, over the tiles' memory
    l = sum_of_halves(l);
    const Sums<VT> sums = {reinterpret_cast<f32x4*>(&tiles[0]), lane};
    float2* stats = reinterpret_cast<float2*>(&sums.at[kWaves * VT * 4 * kWave]);
    static_assert(sizeof(tiles) >= kWaves * (VT * 4096 + kWave * 8), "room for the sums");
    __syncthreads();
    stats[wave * kWave + lane] = make_float2(m, l);
    __syncthreads();
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, stats[i * kWave + lane].x);
    const float tc = top == -INFINITY ? 0.f : top * c;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const float2 v = stats[i * kWave + lane];
        total = fmaf(v.y, __builtin_amdgcn_exp2f(fmaf(v.x, c, -tc)), total);
    }
    const float f = total == 0.f ? 0.f : 1.f / total, own = __builtin_amdgcn_exp2f(fmaf(m, c, -tc));
#pragma unroll
    for (int d = 0; d < VT; ++d) {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= own;
        sums.put(wave, d, o[d]);
    }
    __syncthreads();
    const long row = (long)(w.q0 + min(qi, w.nq - 1)) * a.heads + head;
    if (wave == 0 && g == 0 && live) a.lse[row] = total == 0.f ? -INFINITY : fmaf(top, a.scale, logf(total));
    for (int d = wave; d < VT; d += kWaves) {
        f32x16 x[1] = {sums.sum(d)};
        const uint32_t again = not_finite_rows(x) & rows_with(live && total == total);
        for (uint32_t left = again; left; left &= left - 1) {
            const int r = __ffs(left) - 1;
            const long to = (long)w.q0 + first + r;
            const float mr = __shfl(tc, r, kWave), fr = __shfl(f, r, kWave);
            const int sees = a.causal ? min(w.nk, first + r + shift + 1) : w.nk;
            sum_row_again<1>(
                w.k0, (long)w.k0 + sees, min(32, a.d_v - 32 * d), lane,
                [&](long j) { return __builtin_amdgcn_exp2f(fmaf(dot_rows(qrows, to, krows, j), c, -mr)) * fr; },
                [&](long j, int e) { return value(vrows, j, 32 * d + e); },
                [&](int e, float y) { ((T*)a.o)[(to * a.heads + head) * a.d_v + 32 * d + e] = y; });
        }
        if (live && !(again >> (lane & 31) & 1)) store_columns<T>((T*)a.o + row * a.d_v, x[0], 32 * d, a.d_v, f, VEC, lane);
    }
}

// -------------------------------------------------------------------- dk, dv
template <int DQ, int DV, bool VEC>
__device__ __forceinline__ void dkv(const BackwardParams& a, unsigned block, WaveTiles<DQ, DV> (&tiles)[kWaves]) {
    constexpr int QC = DQ / (2 * E), VC = DV / (2 * E), QT = DQ / 32, VT = DV / 32;
    using TileQ = Tile<T, DQ, kTile>;
    using TileO = Tile<T, DV, kTile>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const LaneReads at = lane_reads<T>(lane);
    int head, seq, tile;
    if (!place<kRows, true>(a, block, lane, head, seq, tile)) return;
    const Range w = seq_range(a.cu_q, a.cu_k, seq, a.len_q, a.len_k);
    const int first = tile * kRows;
    if (first >= w.nk) return;
    const int kj = first + (lane & 31), shift = w.nk - w.nq;
    const bool live = kj < w.nk;

    u32x4 kf[QC], vf[VC];
    const Rows<T> qrows = {(const T*)a.q + head * a.qh, (const T*)a.q, a.qs, 0, a.d_n + a.d_r, 0};
    const Rows<T> orows = {(const T*)a.go + (long)head * a.d_v, (const T*)a.go, (long)a.heads * a.d_v, 0, a.d_v, 0};
    const Rows<T> krows = {(const T*)a.k + head * a.kh, (const T*)(a.r ? a.r : a.k), a.ks, a.rs, a.d_n, a.d_r};
    const Rows<T> vrows = {(const T*)a.v + head * a.vh, (const T*)a.v, a.vs, 0, a.d_v, 0};
    const int r = min(kj, w.nk - 1) - first;
#pragma unroll
    for (int c = 0; c < QC; ++c) kf[c] = load_chunk<T, VEC>(krows, (long)w.k0 + first, r, 2 * c + g);
#pragma unroll
    for (int c = 0; c < VC; ++c) vf[c] = load_chunk<T, VEC>(vrows, (long)w.k0 + first, r, 2 * c + g);
#pragma unroll
    for (int c = 0; c < QC; ++c) settle(kf[c]);
#pragma unroll
    for (int c = 0; c < VC; ++c) settle(vf[c]);
    WaveTiles<DQ, DV>& mine = tiles[wave];
    const Mover<T, DQ, kTile, kWave, VEC> move_a(qrows, lane);
    const Mover<T, DV, kTile, kWave, VEC> move_b(orows, lane);
    move_a.clear(mine.a), move_b.clear(mine.b);
    wave_read();
    const float *lse2 = a.lse2 + head * a.queries + w.q0, *delta = a.delta + head * a.queries + w.q0;
    float lse_r = 0.f, delta_r = 0.f;  // of query lane % 32 of the tile
    const auto start = [&](int q0) {
        const int i = q0 + min(lane & 31, w.nq - q0 - 1);
        lse_r = lse2[i], delta_r = delta[i];
        move_a.start((long)w.q0 + q0, w.nq - q0, mine.a);
        move_b.start((long)w.q0 + q0, w.nq - q0, mine.b);
    };
    f32x16 dk[QT], dv[VT];
#pragma unroll
    for (int d = 0; d < QT; ++d) dk[d] = f32x16{};
#pragma unroll
    for (int d = 0; d < VT; ++d) dv[d] = f32x16{};
    const float c = a.scale * kLog2e;
    const uint32_t qt = lds_offset(&mine.a), ot = lds_offset(&mine.b);
    // the first query that sees the workgroup's first key
    int q0 = (a.causal ? max(0, first - shift) / kTile * kTile : 0) + wave * kTile;
    if (q0 < w.nq) start(q0);
    for (; q0 < w.nq; q0 += kWaves * kTile) {
        wave_landed();
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int i = 0; i < QC; ++i) dot_chunks(s, read_row<TileQ>(qt, at, 0, i), kf[i], T());
#pragma unroll
        for (int i = 0; i < VC; ++i) dot_chunks(dp, read_row<TileO>(ot, at, 0, i), vf[i], T());
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int from = (i & 3) + 8 * (i >> 2) + 4 * g;
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -__shfl(lse_r, from, kWave)));
            dp[i] = s[i] * (dp[i] - __shfl(delta_r, from, kWave));
        }
        if (q0 + kTile > w.nq || (a.causal && first + 31 - shift > q0)) {
            const int least = (a.causal ? kj - shift - q0 : 0) - 4 * g, left = w.nq - q0 - 4 * g;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int e = (i & 3) + 8 * (i >> 2);
                if (e < least || e >= left) s[i] = dp[i] = 0.f;
            }
        }
        Weights<T> p, ds;
        p.set(s);
        ds.set(dp);
#pragma unroll
        for (int d = 0; d < VT; ++d) {
            Columns<T> x;
            x.template load<TileO>(ot, at, 0, d);
            sum_rows(dv[d], x, p);
        }
#pragma unroll
        for (int d = 0; d < QT; ++d) {
            Columns<T> x;
            x.template load<TileQ>(qt, at, 0, d);
            sum_rows(dk[d], x, ds);
        }
        wave_read();
        if (q0 + kWaves * kTile < w.nq) start(q0 + kWaves * kTile);
    }
    const Sums<QT + VT> sums = {reinterpret_cast<f32x4*>(&tiles[0]), lane};
    static_assert(sizeof(tiles) >= kWaves * (QT + VT) * 4096, "room for the sums");
    __syncthreads();
#pragma unroll
    for (int d = 0; d < QT; ++d) sums.put(wave, d, dk[d]);
#pragma unroll
    for (int d = 0; d < VT; ++d) sums.put(wave, QT + d, dv[d]);
    __syncthreads();
    const long token = (long)w.k0 + min(kj, w.nk - 1), row = token * a.heads + head;
    for (int d = wave; d < QT + VT; d += kWaves) {
        const bool is_v = d >= QT;
        const int d0 = 32 * (is_v ? d - QT : d);
        f32x16 x[1] = {sums.sum(d)};
        uint32_t again = not_finite_rows(x) & rows_with(live);
        if (again) {  // but for keys that a query with a NaN sees
            const int last = last_with(w.nq, lane, [&](int i) { return lse2[i] != lse2[i] || (!is_v && delta[i] != delta[i]); });
            again &= rows_with((a.causal ? max(0, kj - shift) : 0) > last);
        }
        const auto put = [&](long to, int e, float y) {  // to column e of a key's row
            if (is_v)
                ((T*)a.dv)[(to * a.heads + head) * a.d_v + e] = y;
            else if (e < a.d_n)
                ((T*)a.dk)[(to * a.heads + head) * a.d_n + e] = y;
            else
                a.dr_part[(head * a.keys + to) * a.d_r + e - a.d_n] = y;
        };
        for (uint32_t left = again; left; left &= left - 1) {
            const int i = __ffs(left) - 1;
            const long to = (long)w.k0 + first + i;
            const int from = a.causal ? max(0, first + i - shift) : 0;
            const Rows<T>& other = is_v ? orows : qrows;
            sum_row_again<1>(
                (long)w.q0 + from, (long)w.q0 + w.nq, min(32, (is_v ? a.d_v : a.d_n + a.d_r) - d0), lane,
                [&](long j) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(dot_rows(qrows, j, krows, to), c, -lse2[j - w.q0]));
                    return is_v ? p : p * (dot_rows(orows, j, vrows, to) - delta[j - w.q0]) * a.scale;
                },
                [&](long j, int e) { return value(other, j, d0 + e); }, [&](int e, float y) { put(to, d0 + e, y); });
        }
        if (!live || again >> (lane & 31) & 1) continue;
        if (is_v) {
            store_columns<T>((T*)a.dv + row * a.d_v, x[0], d0, a.d_v, 1.f, a.vec_out, lane);
        } else if (d0 + 32 <= a.d_n) {
            store_columns<T>((T*)a.dk + row * a.d_n, x[0], d0, a.d_n, a.scale, a.vec_out, lane);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int e = d0 + (i & 3) + 8 * (i >> 2) + 4 * g;
                if (e < a.d_n + a.d_r) put(token, e, x[0][i] * a.scale);
            }
        }
    }
}

// ------------------------------------------------------------------------ dq
template <int DQ, int DV, bool VEC>
__device__ __forceinline__ void dq(const BackwardParams& a, unsigned block, WaveTiles<DQ, DV> (&tiles)[kWaves]) {
    constexpr int QC = DQ / (2 * E), VC = DV / (2 * E), QT = DQ / 32;
    using TileK = Tile<T, DQ, kTile>;
    using TileV = Tile<T, DV, kTile>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const LaneReads at = lane_reads<T>(lane);
    int head, seq, tile;
    if (!place<kRows, false>(a, block, lane, head, seq, tile)) return;
    const Range w = seq_range(a.cu_q, a.cu_k, seq, a.len_q, a.len_k);
    if (tile * kRows >= w.nq) return;
    const int first = ((w.nq - 1) / kRows - tile) * kRows;
    const int qi = first + (lane & 31), shift = w.nk - w.nq, row_in = min(qi, w.nq - 1);
    const bool live = qi < w.nq;
    const int end = a.causal ? min(w.nk, min(first + kRows, w.nq) + shift) : w.nk;

    u32x4 qf[QC], of[VC];
    const Rows<T> qrows = {(const T*)a.q + head * a.qh, (const T*)a.q, a.qs, 0, a.d_n + a.d_r, 0};
    const Rows<T> orows = {(const T*)a.go + (long)head * a.d_v, (const T*)a.go, (long)a.heads * a.d_v, 0, a.d_v, 0};
    const Rows<T> krows = {(const T*)a.k + head * a.kh, (const T*)(a.r ? a.r : a.k), a.ks, a.rs, a.d_n, a.d_r};
    const Rows<T> vrows = {(const T*)a.v + head * a.vh, (const T*)a.v, a.vs, 0, a.d_v, 0};
#pragma unroll
    for (int c = 0; c < QC; ++c) qf[c] = load_chunk<T, VEC>(qrows, (long)w.q0 + first, row_in - first, 2 * c + g);
#pragma unroll
    for (int c = 0; c < VC; ++c) of[c] = load_chunk<T, VEC>(orows, (long)w.q0 + first, row_in - first, 2 * c + g);
    float lse2 = a.lse2[head * a.queries + w.q0 + row_in], delta = a.delta[head * a.queries + w.q0 + row_in];
#pragma unroll
    for (int c = 0; c < QC; ++c) settle(qf[c]);
#pragma unroll
    for (int c = 0; c < VC; ++c) settle(of[c]);
    settle(lse2), settle(delta);
    WaveTiles<DQ, DV>& mine = tiles[wave];
    const Mover<T, DQ, kTile, kWave, VEC> move_a(krows, lane);
    const Mover<T, DV, kTile, kWave, VEC> move_b(vrows, lane);
    move_a.clear(mine.a), move_b.clear(mine.b);
    wave_read();
    const auto start = [&](int k0) {
        move_a.start((long)w.k0 + k0, w.nk - k0, mine.a);
        move_b.start((long)w.k0 + k0, w.nk - k0, mine.b);
    };
    f32x16 dq[QT];
#pragma unroll
    for (int d = 0; d < QT; ++d) dq[d] = f32x16{};
    const float c = a.scale * kLog2e;
    const int seen = a.causal ? min(w.nk, qi + shift + 1) : w.nk;
    const uint32_t kt = lds_offset(&mine.a), vt = lds_offset(&mine.b);
    int k0 = wave * kTile;
    if (k0 < end) start(k0);
    for (; k0 < end; k0 += kWaves * kTile) {
        wave_landed();
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int i = 0; i < QC; ++i) dot_chunks(s, read_row<TileK>(kt, at, 0, i), qf[i], T());
#pragma unroll
        for (int i = 0; i < VC; ++i) dot_chunks(dp, read_row<TileV>(vt, at, 0, i), of[i], T());
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -lse2)) * (dp[i] - delta);
        if (k0 + kTile > w.nk || (a.causal && k0 + kTile > first + shift + 1)) {
            const int left = seen - k0 - 4 * g;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if ((i & 3) + 8 * (i >> 2) >= left) dp[i] = 0.f;
        }
        Weights<T> ds;
        ds.set(dp);
#pragma unroll
        for (int d = 0; d < QT; ++d) {
            Columns<T> x;
            x.template load<TileK>(kt, at, 0, d);
            sum_rows(dq[d], x, ds);
        }
        wave_read();
        if (k0 + kWaves * kTile < end) start(k0 + kWaves * kTile);
    }
    const Sums<QT> sums = {reinterpret_cast<f32x4*>(&tiles[0]), lane};
    __syncthreads();
#pragma unroll
    for (int d = 0; d < QT; ++d) sums.put(wave, d, dq[d]);
    __syncthreads();
    const int cols = a.d_n + a.d_r;
    const bool nan = (lse2 != lse2 || delta != delta) && seen > 0;
    for (int d = wave; d < QT; d += kWaves) {
        f32x16 x[1] = {sums.sum(d)};
        const uint32_t again = not_finite_rows(x) & rows_with(live && !nan);
        for (uint32_t left = again; left; left &= left - 1) {
            const int r = __ffs(left) - 1;
            const long to = (long)w.q0 + first + r;
            const float lr = __shfl(lse2, r, kWave), dr = __shfl(delta, r, kWave);
            const int sees = a.causal ? min(w.nk, first + r + shift + 1) : w.nk;
            sum_row_again<1>(
                w.k0, (long)w.k0 + sees, min(32, cols - 32 * d), lane,
                [&](long j) {
                    return __builtin_amdgcn_exp2f(fmaf(dot_rows(qrows, to, krows, j), c, -lr)) *
                           (dot_rows(orows, to, vrows, j) - dr) * a.scale;
                },
                [&](long j, int e) { return value(krows, j, 32 * d + e); },
                [&](int e, float y) { ((T*)a.dq)[(to * a.heads + head) * cols + 32 * d + e] = y; });
        }
        if (!live || again >> (lane & 31) & 1) continue;
        store_columns<T>((T*)a.dq + ((long)(w.q0 + qi) * a.heads + head) * cols, x[0], 32 * d, cols, a.scale, a.vec_out, lane);
    }
}

// One launch of both, dk and dv first, so that neither ends on a card half empty:
// 64 + 32 channels, 1080 tokens of 8 heads 68 -> 52 us, 2 x 2048 of 16 heads 792
// -> 724, at two workgroups a CU.  Wider ones have the LDS for one only, and each
// kernel then is faster by itself: 128 + 64 channels, 1631 us against 1694 in one.
template <int DQ, int DV, bool VEC>
__global__ __launch_bounds__(kThreads, 2) void attn_backward_split_kernel(BackwardParams a) {
    __shared__ WaveTiles<DQ, DV> tiles[kWaves];
    const unsigned half = gridDim.x / 2;
    if (blockIdx.x < half)
        dkv<DQ, DV, VEC>(a, blockIdx.x, tiles);
    else
        dq<DQ, DV, VEC>(a, blockIdx.x - half, tiles);
}
template <int DQ, int DV, bool VEC>
__global__ __launch_bounds__(kThreads) void attn_dkv_split_kernel(BackwardParams a) {
    __shared__ WaveTiles<DQ, DV> tiles[kWaves];
    dkv<DQ, DV, VEC>(a, blockIdx.x, tiles);
}
template <int DQ, int DV, bool VEC>
__global__ __launch_bounds__(kThreads) void attn_dq_split_kernel(BackwardParams a) {
    __shared__ WaveTiles<DQ, DV> tiles[kWaves];
    dq<DQ, DV, VEC>(a, blockIdx.x, tiles);
}

template <int DQ, int DV, bool VEC>
hipError_t prefill(PrefillParams p, hipStream_t stream) {
    const int64_t queries = p.cu_q ? (int64_t)p.len_q : (int64_t)p.batch * p.len_q;
    const int64_t tiles = attn_tiles(p.cu_q, queries, p.len_q, p.batch, kRows);
    const unsigned blocks = attn_blocks(p.heads, p.batch, p.cu_q, tiles);
    if (!blocks) return hipErrorInvalidConfiguration;
    p.tiles = (int)tiles;
    latent_prefill_split_kernel<DQ, DV, VEC><<<blocks, kThreads, 0, stream>>>(p);
    return hipGetLastError();
}

template <int DQ, int DV, bool VEC>
hipError_t backward(BackwardParams p, hipStream_t stream) {
    const int64_t tq = attn_tiles(p.cu_q, p.queries, p.len_q, p.batch, kRows);
    const int64_t tk = attn_tiles(p.cu_k, p.keys, p.len_k, p.batch, kRows);
    if constexpr (DQ <= 96 && DV <= 64) {
        const unsigned blocks = attn_blocks(p.heads, p.batch, p.cu_q, 2 * std::max(tq, tk));
        if (!blocks) return hipErrorInvalidConfiguration;
        p.tiles = (int)std::max(tq, tk);
        attn_backward_split_kernel<DQ, DV, VEC><<<blocks, kThreads, 0, stream>>>(p);
        return hipGetLastError();
    } else {
        const unsigned dkv = attn_blocks(p.heads, p.batch, p.cu_k, tk), dq = attn_blocks(p.heads, p.batch, p.cu_q, tq);
        if ((p.keys && !dkv) || (p.queries && !dq)) return hipErrorInvalidConfiguration;
        p.tiles = (int)tk;
        if (p.keys) attn_dkv_split_kernel<DQ, DV, VEC><<<dkv, kThreads, 0, stream>>>(p);
        p.tiles = (int)tq;
        if (p.queries) attn_dq_split_kernel<DQ, DV, VEC><<<dq, kThreads, 0, stream>>>(p);
        return hipGetLastError();
    }
}

}  // namespace

// The narrowest kernel that holds the channels: 2 x 4096 tokens, 16 heads, prefill,
// by the kernels for (64, 64), (96, 64), (128, 128) and (192, 128) channels: of 64
// and 64 643 / - / 1703 / 2168 us, of 96 and 64 - / 779 / 1709 / 2172, of 128 and
// 128 - / - / 1495 / 2058.
hipError_t launch_prefill_split(PrefillParams p, bool vec, hipStream_t stream) {
    const int dq = p.d_n + p.d_r;
    if (!vec) return dq <= 64 && p.d_v <= 64 ? prefill<64, 64, false>(p, stream) : prefill<192, 128, false>(p, stream);
    if (p.d_v <= 64 && dq <= 64) return prefill<64, 64, true>(p, stream);
    if (p.d_v <= 64 && dq <= 96) return prefill<96, 64, true>(p, stream);
    if (dq <= 128) return prefill<128, 128, true>(p, stream);
    return prefill<192, 128, true>(p, stream);
}

hipError_t launch_backward_split(BackwardParams p, bool vec, hipStream_t stream) {
    const int dq = p.d_n + p.d_r;
    if (!vec) return dq <= 64 && p.d_v <= 64 ? backward<64, 64, false>(p, stream) : backward<192, 128, false>(p, stream);
    if (p.d_v <= 64 && dq <= 64) return backward<64, 64, true>(p, stream);
    if (p.d_v <= 64 && dq <= 96) return backward<96, 64, true>(p, stream);
    if (dq <= 128) return backward<128, 128, true>(p, stream);
    return backward<192, 128, true>(p, stream);
}

}  // namespace rhz
