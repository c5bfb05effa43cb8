// attn_backward.hip -- backward pass of the latent attention over expanded keys
// and values.
//
// With p_ij = e^(s_ij - lse_i), dp_ij = do_i . v_j and D_i = do_i . o_i - dlse_i,
//     ds = p (dp - D),   dv_j = sum_i p_ij do_i,   dq_i = scale sum_j ds_ij k_j,
//     dk_j = scale sum_i ds_ij q_i,   the rotary part of dk summed over heads.
// The weights are formed again from lse.  One kernel runs over queries and
// holds 128 keys' dk and dv, another runs over keys and holds 128 queries' dq:
// seven products instead of the five that one kernel needs, which would have to
// add its dq from all key tiles in memory, in no fixed order or with waits.
//
// 2 x 4096 tokens, 32 heads of 128 + 64 channels, causal: 1350 to 1420 us by the
// card's clocks.  Of 1394 by one trace of the kernels, D and lse take 31 (134 MB, 4.4
// TB/s), dk and dv 838 (820 TFLOP/s of its four products), dq 511 (1075 of its
// three), the sum over heads 15.  The seven products at the 1152 TFLOP/s of a large
// one: 1074 us, the formula's five 775.
#include "attn_params.hpp"

namespace rhz {
namespace {

constexpr int kThreads = kAttnThreads, kRows = 128;

// ---------------------------------------------------------------- D and lse
// 64 tokens of one head a workgroup, 16 lanes a row.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void attn_delta_kernel(BackwardParams a) {
    constexpr int E = VEC ? kChunkElems<T> : 1;
    const int tid = threadIdx.x, head = blockIdx.x % a.heads, l = tid & 15;
    const long t0 = (long)(blockIdx.x / a.heads) * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long t = t0 + i * 16 + (tid >> 4);
        if (t >= a.queries) continue;
        const long row = t * a.heads + head;
        const T *o = (const T*)a.o + row * a.d_v, *go = (const T*)a.go + row * a.d_v;
        float sum = 0.f;
        for (int d = l * E; d < a.d_v; d += 16 * E) {
            float x[E], y[E];
            Vec<T, VEC>::load(o + d, x);
            Vec<T, VEC>::load(go + d, y);
#pragma unroll
            for (int j = 0; j < E; ++j) sum = fmaf(x[j], y[j], sum);
        }
        sum = lane_group_sum<16>(sum);
        if (l == 0) {
            a.delta[head * a.queries + t] = sum - (a.glse ? a.glse[row] : 0.f);
            a.lse2[head * a.queries + t] = a.lse[row] * kLog2e;
        }
    }
}

// ------------------------------------------------------------------ dk, dv
// Eight waves for 128 keys, two for every 32 of them: the first forms the
// weights p and sums dv = p^T do, the second forms dp, takes p from the first
// through LDS a tile later, and sums dk = ds^T q.  That halves what a wave holds
// (keys or values as operands, and one of the sums), so that each SIMD has one of
// either kind, whose matrix and vector instructions overlap: 1650 -> 1420 us for the
// whole pass of 2 x 4096 tokens, 32 heads, against four waves that each do
// all of it.  Matrix instructions take 37 % of its time and LDS reads 27 %: a tile
// takes the longer of the two kinds' ways through it.  Loads spread over the
// products: 1413 us instead of 1375.
template <int DQ, int DV, bool VEC>
__global__ __launch_bounds__(512, 2) void attn_dkv_kernel(BackwardParams a) {
    using T = uint16_t;
    constexpr int E = kChunkElems<T>, BQ = 32, RING = 4;
    constexpr int QC = DQ / (2 * E), VC = DV / (2 * E), QT = DQ / 32, VT = DV / 32;
    using TileQ = Tile<T, DQ, BQ>;
    using TileO = Tile<T, DV, BQ>;
    __shared__ TileQ qtiles[RING];
    __shared__ TileO otiles[RING];
    __shared__ f32x4 handed[2][4][4][kWave];                 // p: [tile][32 keys][registers by four][lane]
    __shared__ float4 lse_s[RING][16], delta_s[RING][16];  // a wave's 64 floats
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5;
    const int second = wave >> 2, group = wave & 3;
    const LaneReads at = lane_reads<T>(lane);
    int head, seq, tile;
    if (!place<kRows, true>(a, blockIdx.x, lane, head, seq, tile)) return;
    const Range w = seq_range(a.cu_q, a.cu_k, seq, a.len_q, a.len_k);
    const int first = tile * kRows;
    if (first >= w.nk) return;
    const int wk = first + group * 32, kj = wk + (lane & 31);
    const int shift = w.nk - w.nq;
    bool live = kj < w.nk;
    const long token = (long)w.k0 + min(kj, w.nk - 1), row = token * a.heads + head;

    const Rows<T> krows = {(const T*)a.k + head * a.kh, (const T*)(a.r ? a.r : a.k), a.ks, a.rs, a.d_n, a.d_r};
    const Rows<T> vrows = {(const T*)a.v + head * a.vh, (const T*)a.v, a.vs, 0, a.d_v, 0};
    const Rows<T> qrows = {(const T*)a.q + head * a.qh, (const T*)a.q, a.qs, 0, a.d_n + a.d_r, 0};
    const Rows<T> orows = {(const T*)a.go + (long)head * a.d_v, (const T*)a.go, (long)a.heads * a.d_v, 0, a.d_v, 0};
    const float* lse2 = a.lse2 + head * a.queries + w.q0;
    const float* delta = a.delta + head * a.queries + w.q0;
    const float c = a.scale * kLog2e;
    // from the first query that sees the workgroup's first key on
    const int begin = a.causal ? max(0, first - shift) / BQ * BQ : 0;
    const int tiles = w.nq > begin ? (w.nq - begin + BQ - 1) / BQ : 0;

    // The first kind moves q, the second do and what belongs to the queries.
    const Mover<T, DQ, BQ, kThreads, VEC> move_q(qrows, tid & 255);
    const Mover<T, DV, BQ, kThreads, VEC> move_o(orows, tid & 255);
    const auto start = [&](int j) {
        const int q0 = begin + j * BQ, left = w.nq - q0, slot = j % RING;
        if (!second) {
            move_q.start((long)w.q0 + q0, left, qtiles[slot]);
        } else {
            move_o.start((long)w.q0 + q0, left, otiles[slot]);
            const uint32_t off = min(lane, min(BQ, left) - 1) * 4;
            if (group == 0) load_to_lds4(lse2 + q0, off, lds_offset(&lse_s[slot][0]));
            if (group == 1) load_to_lds4(delta + q0, off, lds_offset(&delta_s[slot][0]));
        }
    };
    for (int i = 0; i < RING; ++i) {
        if (!second) move_q.clear(qtiles[i]);
        if (second) move_o.clear(otiles[i]);
    }
    // Tile j is there, for all waves, while j + 1 may be on its way -- if every panel is
    // full and of one tensor: the waits count panels.  Else (64 + 32 channels) j + 1 has
    // to be there too.
    const bool counted = VEC && move_q.whole && move_o.whole;
    const auto wait = [&](int j) {
        if (counted && j + 1 < tiles) {
            if (!second)
                wait_loads<TileQ::kPanels>();
            else if (group < 2)
                wait_loads<TileO::kPanels + 1>();
            else
                wait_loads<TileO::kPanels>();
        } else {
            wait_loads<0>();
        }
        lds_barrier();
    };
    const auto hidden = [&](int j) { return a.causal && begin + j * BQ + BQ - 1 + shift < wk; };  // sees none of the keys
    // p or ds of what is not seen: of the lane's key rows below `least`, and those behind the last query
    const auto clip = [&](int j, f32x16& x) {
        const int qu = begin + j * BQ;
        if (qu + BQ <= w.nq && !(a.causal && wk + 31 - shift > qu)) return;
        const int least = (a.causal ? kj - shift - qu : 0) - 4 * g, left = w.nq - qu - 4 * g;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = (i & 3) + 8 * (i >> 2);
            if (r < least || r >= left) x[i] = 0.f;
        }
    };

    if (!second) {
        u32x4 kf[QC];
#pragma unroll
        for (int i = 0; i < QC; ++i)
            kf[i] = load_chunk<T, VEC>(krows, (long)w.k0 + first, min(kj, w.nk - 1) - first, 2 * i + g);
#pragma unroll
        for (int i = 0; i < QC; ++i) settle(kf[i]);
        f32x16 dv[VT];
#pragma unroll
        for (int d = 0; d < VT; ++d) dv[d] = f32x16{};
        lds_barrier();
        if (tiles > 0) start(0);
        if (tiles > 1) start(1);
        for (int j = 0; j < tiles; ++j) {
            wait(j);
            if (j + 2 < tiles) start(j + 2);
            if (hidden(j)) continue;
            const uint32_t qt = lds_offset(&qtiles[j % RING]), ot = lds_offset(&otiles[j % RING]);
            f32x16 s = {};
            dot_ahead<QC, 6>(s, kf, [&](int i) { return read_row<TileQ>(qt, at, 0, i); }, T());
            SumAhead<T, TileO, VT, 2> sum;
            sum.begin(ot, at, 0);
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const float4 l = lse_s[j % RING][2 * i4 + g];
                s[4 * i4] = __builtin_amdgcn_exp2f(fmaf(s[4 * i4], c, -l.x));
                s[4 * i4 + 1] = __builtin_amdgcn_exp2f(fmaf(s[4 * i4 + 1], c, -l.y));
                s[4 * i4 + 2] = __builtin_amdgcn_exp2f(fmaf(s[4 * i4 + 2], c, -l.z));
                s[4 * i4 + 3] = __builtin_amdgcn_exp2f(fmaf(s[4 * i4 + 3], c, -l.w));
            }
            clip(j, s);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                handed[j & 1][group][k][lane] = f32x4{s[4 * k], s[4 * k + 1], s[4 * k + 2], s[4 * k + 3]};
            Weights<T> p;
            p.set(s);
            sum.run(dv, ot, at, 0, p);
        }
        lds_barrier();  // the last tile's weights are handed on
        uint32_t again = not_finite_rows(dv) & rows_with(live);
        if (again) {  // but for keys that a query with a NaN sees
            const int last = last_with(w.nq, lane, [&](int i) { return lse2[i] != lse2[i]; });
            again &= rows_with((a.causal ? max(0, kj - shift) : 0) > last);
        }
        while (again) {
            const int r = __ffs(again) - 1;
            again &= again - 1;
            const long mine = (long)w.k0 + wk + r;
            const int from = a.causal ? max(0, wk + r - shift) : 0;  // the first query that sees the key
            sum_row_again<2>(
                (long)w.q0 + from, (long)w.q0 + w.nq, a.d_v, lane,
                [&](long i) { return __builtin_amdgcn_exp2f(fmaf(dot_rows(qrows, i, krows, mine), c, -lse2[i - w.q0])); },
                [&](long i, int d) { return value(orows, i, d); },
                [&](int d, float x) { Elem<T>::store((T*)a.dv + (mine * a.heads + head) * a.d_v, d, x); });
            if ((lane & 31) == r) live = false;
        }
        if (!live) return;
#pragma unroll
        for (int d = 0; d < VT; ++d) store_columns<T>((T*)a.dv + row * a.d_v, dv[d], 32 * d, a.d_v, 1.f, a.vec_out, lane);
    } else {
        u32x4 vf[VC];
#pragma unroll
        for (int i = 0; i < VC; ++i)
            vf[i] = load_chunk<T, VEC>(vrows, (long)w.k0 + first, min(kj, w.nk - 1) - first, 2 * i + g);
#pragma unroll
        for (int i = 0; i < VC; ++i) settle(vf[i]);
        f32x16 dk[QT];
#pragma unroll
        for (int d = 0; d < QT; ++d) dk[d] = f32x16{};
        lds_barrier();
        if (tiles > 0) start(0);
        if (tiles > 1) start(1);
        for (int j1 = 0; j1 <= tiles; ++j1) {  // a tile behind the first kind
            if (j1 < tiles)
                wait(j1);
            else
                lds_barrier();
            if (j1 + 2 < tiles) start(j1 + 2);
            const int j = j1 - 1;
            if (j < 0 || hidden(j)) continue;
            const uint32_t qt = lds_offset(&qtiles[j % RING]), ot = lds_offset(&otiles[j % RING]);
            f32x16 dp = {};
            dot_ahead<VC, 6>(dp, vf, [&](int i) { return read_row<TileO>(ot, at, 0, i); }, T());
            SumAhead<T, TileQ, QT, 2> sum;
            sum.begin(qt, at, 0);
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const f32x4 p = handed[j & 1][group][i4][lane];
                const float4 l = delta_s[j % RING][2 * i4 + g];
                dp[4 * i4] = p[0] * (dp[4 * i4] - l.x);
                dp[4 * i4 + 1] = p[1] * (dp[4 * i4 + 1] - l.y);
                dp[4 * i4 + 2] = p[2] * (dp[4 * i4 + 2] - l.z);
                dp[4 * i4 + 3] = p[3] * (dp[4 * i4 + 3] - l.w);
            }
            clip(j, dp);
            Weights<T> ds;
            ds.set(dp);
            sum.run(dk, qt, at, 0, ds);
        }
        uint32_t again = not_finite_rows(dk) & rows_with(live);
        if (again) {
            const int last = last_with(w.nq, lane, [&](int i) { return lse2[i] != lse2[i] || delta[i] != delta[i]; });
            again &= rows_with((a.causal ? max(0, kj - shift) : 0) > last);
        }
        while (again) {
            const int r = __ffs(again) - 1;
            again &= again - 1;
            const long mine = (long)w.k0 + wk + r;
            const int from = a.causal ? max(0, wk + r - shift) : 0;
            sum_row_again<3>(
                (long)w.q0 + from, (long)w.q0 + w.nq, a.d_n + a.d_r, lane,
                [&](long i) {
                    return __builtin_amdgcn_exp2f(fmaf(dot_rows(qrows, i, krows, mine), c, -lse2[i - w.q0])) *
                           (dot_rows(orows, i, vrows, mine) - delta[i - w.q0]) * a.scale;
                },
                [&](long i, int d) { return value(qrows, i, d); },
                [&](int d, float x) {
                    if (d < a.d_n)
                        Elem<T>::store((T*)a.dk + (mine * a.heads + head) * a.d_n, d, x);
                    else
                        a.dr_part[(head * a.keys + mine) * a.d_r + d - a.d_n] = x;
                });
            if ((lane & 31) == r) live = false;
        }
        if (!live) return;
        T* gk = (T*)a.dk + row * a.d_n;
        float* gr = a.dr_part + (head * a.keys + token) * a.d_r;
#pragma unroll
        for (int d = 0; d < QT; ++d) {
            if (32 * d < a.d_n) store_columns<T>(gk, dk[d], 32 * d, a.d_n, a.scale, a.vec_out, lane);
            if (32 * d + 32 > a.d_n) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int e = 32 * d + (i & 3) + 8 * (i >> 2) + 4 * g - a.d_n;
                    if (e >= 0 && e < a.d_r) gr[e] = dk[d][i] * a.scale;
                }
            }
        }
    }
}

// ---------------------------------------------------------------------- dq
// As the prefill, with lse known: p needs no maximum.  32 keys a tile, for the
// registers of two operands and the sum at two workgroups a CU.
template <int DQ, int DV, bool VEC>
__global__ __launch_bounds__(kThreads, 2) void attn_dq_kernel(BackwardParams a) {
    using T = uint16_t;
    constexpr int E = kChunkElems<T>, BN = 32;
    constexpr int QC = DQ / (2 * E), VC = DV / (2 * E), QT = DQ / 32;
    __shared__ Tile<T, DQ, BN> ktiles[2];
    __shared__ Tile<T, DV, BN> vtiles[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5;
    const LaneReads at = lane_reads<T>(lane);
    int head, seq, tile;
    if (!place<kRows, false>(a, blockIdx.x, lane, head, seq, tile)) return;
    const Range w = seq_range(a.cu_q, a.cu_k, seq, a.len_q, a.len_k);
    const int last_tile = (w.nq - 1) / kRows;
    if (w.nq == 0 || tile > last_tile) return;
    const int first = (last_tile - tile) * kRows;  // the queries with the most keys go first
    const int wq = first + wave * 32, qi = wq + (lane & 31);
    const int shift = w.nk - w.nq;
    const int last_q = min(first + kRows, w.nq) - 1;
    const int end = a.causal ? min(w.nk, last_q + shift + 1) : w.nk;

    u32x4 qf[QC], of[VC];
    const int mine = min(qi, w.nq - 1);
    const Rows<T> qrows = {(const T*)a.q + head * a.qh, (const T*)a.q, a.qs, 0, a.d_n + a.d_r, 0};
    const Rows<T> orows = {(const T*)a.go + (long)head * a.d_v, (const T*)a.go, (long)a.heads * a.d_v, 0, a.d_v, 0};
#pragma unroll
    for (int c = 0; c < QC; ++c) qf[c] = load_chunk<T, VEC>(qrows, (long)w.q0 + first, mine - first, 2 * c + g);
#pragma unroll
    for (int c = 0; c < VC; ++c) of[c] = load_chunk<T, VEC>(orows, (long)w.q0 + first, mine - first, 2 * c + g);
    float lse2 = a.lse2[head * a.queries + w.q0 + mine], delta = a.delta[head * a.queries + w.q0 + mine];
    const Rows<T> krows = {(const T*)a.k + head * a.kh, (const T*)(a.r ? a.r : a.k), a.ks, a.rs, a.d_n, a.d_r};
    const Rows<T> vrows = {(const T*)a.v + head * a.vh, (const T*)a.v, a.vs, 0, a.d_v, 0};
#pragma unroll
    for (int c = 0; c < QC; ++c) settle(qf[c]);
#pragma unroll
    for (int c = 0; c < VC; ++c) settle(of[c]);
    settle(lse2), settle(delta);
    f32x16 dq[QT];
#pragma unroll
    for (int d = 0; d < QT; ++d) dq[d] = f32x16{};
    const float c = a.scale * kLog2e;
    const Mover<T, DQ, BN, kThreads, VEC> move_k(krows, tid);
    const Mover<T, DV, BN, kThreads, VEC> move_v(vrows, tid);
    for (int b = 0; b < 2; ++b) move_k.clear(ktiles[b]), move_v.clear(vtiles[b]);
    __syncthreads();
    if (end > 0) {
        move_k.start(w.k0, w.nk, ktiles[0]);
        move_v.start(w.k0, w.nk, vtiles[0]);
    }
    for (int k0 = 0, b = 0; k0 < end; k0 += BN, b ^= 1) {
        landed();
        if (k0 + BN < end) {
            move_k.start((long)w.k0 + k0 + BN, w.nk - k0 - BN, ktiles[b ^ 1]);
            move_v.start((long)w.k0 + k0 + BN, w.nk - k0 - BN, vtiles[b ^ 1]);
        }
        const uint32_t kt = lds_offset(&ktiles[b]);
        const uint32_t vt = lds_offset(&vtiles[b]);
        if (a.causal && k0 > wq + 31 + shift) continue;
        f32x16 s = {}, dp = {};
        dot_ahead<QC, 4>(s, qf, [&](int i) { return read_row<Tile<T, DQ, BN>>(kt, at, 0, i); }, T());
        dot_ahead<VC, 4>(dp, of, [&](int i) { return read_row<Tile<T, DV, BN>>(vt, at, 0, i); }, T());
        SumAhead<T, Tile<T, DQ, BN>, QT, 2> sum;
        sum.begin(kt, at, 0);
        const int seen = a.causal ? min(w.nk, qi + shift + 1) : w.nk;
        const bool masked = k0 + BN > w.nk || (a.causal && k0 + BN > wq + shift + 1);
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -lse2)) * (dp[i] - delta);
        if (masked) {
            const int left = seen - k0 - 4 * g;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if ((i & 3) + 8 * (i >> 2) >= left) dp[i] = 0.f;
        }
        Weights<T> ds;
        ds.set(dp);
        sum.run(dq, kt, at, 0, ds);
    }
    bool live = qi < w.nq;
    const bool nan = (lse2 != lse2 || delta != delta) && (a.causal ? min(w.nk, qi + shift + 1) : w.nk) > 0;
    uint32_t again = not_finite_rows(dq) & rows_with(live && !nan);
    while (again) {
        const int r = __ffs(again) - 1;
        again &= again - 1;
        const long mine = (long)w.q0 + wq + r;
        const float lr = __shfl(lse2, r, kWave), dr = __shfl(delta, r, kWave);
        const int sees = a.causal ? min(w.nk, wq + r + shift + 1) : w.nk;
        sum_row_again<3>(
            w.k0, (long)w.k0 + sees, a.d_n + a.d_r, lane,
            [&](long j) {
                return __builtin_amdgcn_exp2f(fmaf(dot_rows(qrows, mine, krows, j), c, -lr)) *
                       (dot_rows(orows, mine, vrows, j) - dr) * a.scale;
            },
            [&](long j, int d) { return value(krows, j, d); },
            [&](int d, float x) { Elem<T>::store((T*)a.dq + (mine * a.heads + head) * (a.d_n + a.d_r), d, x); });
        if ((lane & 31) == r) live = false;
    }
    if (!live) return;
    T* out = (T*)a.dq + ((long)(w.q0 + qi) * a.heads + head) * (a.d_n + a.d_r);
#pragma unroll
    for (int d = 0; d < QT; ++d) store_columns<T>(out, dq[d], 32 * d, a.d_n + a.d_r, a.scale, a.vec_out, lane);
}

// ------------------------------------------------- the rotary key's gradient
// Sum over the heads of a value's parts, one value a thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void attn_rope_sum_kernel(BackwardParams a) {
    long begin = 0, end = a.keys;
    if (a.cu_k) {
        begin = min(max(a.cu_k[0], 0), a.len_k);
        end = min(max(a.cu_k[a.batch], 0), a.len_k);
    }
    const long at = (long)blockIdx.x * kThreads + threadIdx.x;
    if (at < begin * a.d_r || at >= end * a.d_r) return;
    float sum = 0.f;
#pragma unroll 4
    for (int h = 0; h < a.heads; ++h) sum += a.dr_part[h * a.keys * a.d_r + at];
    Elem<T>::store((T*)a.dr, at, sum);
}

bool too_many(int64_t blocks) { return blocks > INT32_MAX || check_grid(blocks, kThreads) != hipSuccess; }

template <int DQ, int DV, bool VEC>
hipError_t launch(BackwardParams p, hipStream_t stream) {
    const int64_t tq = attn_tiles(p.cu_q, p.queries, p.len_q, p.batch, kRows);
    const int64_t tk = attn_tiles(p.cu_k, p.keys, p.len_k, p.batch, kRows);
    const unsigned dkv = attn_blocks(p.heads, p.batch, p.cu_k, tk, 512), dq = attn_blocks(p.heads, p.batch, p.cu_q, tq);
    if ((p.keys && !dkv) || (p.queries && !dq)) return hipErrorInvalidConfiguration;
    p.tiles = (int)tk;
    if (p.keys) attn_dkv_kernel<DQ, DV, VEC><<<dkv, 512, 0, stream>>>(p);
    p.tiles = (int)tq;
    if (p.queries) attn_dq_kernel<DQ, DV, VEC><<<dq, kThreads, 0, stream>>>(p);
    return hipGetLastError();
}

// The narrowest kernel that holds the channels, as in the prefill: 2 x 4096 tokens,
// 16 heads, of 64 and 64 channels 380 / - / 526 / 602 us, of 96 and 64 - / 444 / 545
// / 617, of 128 and 128 - / - / 561 / 634.
hipError_t pick(const BackwardParams& p, bool vec, hipStream_t stream) {
    const int dq = p.d_n + p.d_r;
    if (!vec) return dq <= 64 && p.d_v <= 64 ? launch<64, 64, false>(p, stream) : launch<192, 128, false>(p, stream);
    if (p.d_v <= 64 && dq <= 64) return launch<64, 64, true>(p, stream);
    if (p.d_v <= 64 && dq <= 96) return launch<96, 64, true>(p, stream);
    if (dq <= 128) return launch<128, 128, true>(p, stream);
    return launch<192, 128, true>(p, stream);
}

template <typename T>
hipError_t launch_all(const BackwardParams& p, bool vec, hipStream_t stream) {
    const int64_t delta = (p.queries + 63) / 64 * p.heads, rope = (p.keys * p.d_r + kThreads - 1) / kThreads;
    if (too_many(delta) || too_many(rope)) return hipErrorInvalidConfiguration;
    if (p.queries && p.vec_delta) attn_delta_kernel<T, true><<<(unsigned)delta, kThreads, 0, stream>>>(p);
    if (p.queries && !p.vec_delta) attn_delta_kernel<T, false><<<(unsigned)delta, kThreads, 0, stream>>>(p);
    const hipError_t e = sizeof(T) == 4 ? launch_backward_split(p, vec, stream) : pick(p, vec, stream);
    if (e != hipSuccess) return e;
    if (rope) attn_rope_sum_kernel<T><<<(unsigned)rope, kThreads, 0, stream>>>(p);
    return hipGetLastError();
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

void counts(const rhz_latent_prefill_args& f, size_t& queries, size_t& keys) {
    queries = f.cu_seqlens ? (size_t)f.seq_len : (size_t)f.batch * f.seq_len;
    keys = f.cu_seqlens ? (size_t)f.seq_len_k : (size_t)f.batch * f.seq_len_k;
}

}  // namespace

size_t latent_prefill_backward_workspace_bytes(const rhz_latent_prefill_backward_args& a) {
    size_t queries, keys;
    counts(a.forward, queries, keys);
    return 2 * up256(queries * a.forward.heads * 4) + up256(keys * a.forward.heads * a.forward.d_r * 4);
}

hipError_t launch_latent_prefill_backward(const rhz_latent_prefill_backward_args& a, hipStream_t stream) {
    const rhz_latent_prefill_args& f = a.forward;
    size_t queries, keys;
    counts(f, queries, keys);
    char* ws = (char*)a.workspace;
    const size_t row = up256(queries * f.heads * 4);
    BackwardParams p = {};
    p.q = f.q, p.k = f.k, p.v = f.v, p.r = f.k_rope, p.go = a.grad_o, p.o = f.o;
    p.cu_q = f.cu_seqlens, p.cu_k = f.cu_seqlens_k ? f.cu_seqlens_k : f.cu_seqlens;
    p.lse = f.lse, p.glse = a.grad_lse;
    p.dq = a.grad_q, p.dk = a.grad_k, p.dv = a.grad_v, p.dr = a.grad_k_rope;
    p.lse2 = (float*)ws, p.delta = (float*)(ws + row), p.dr_part = (float*)(ws + 2 * row);
    p.qs = f.q_token_stride, p.qh = f.q_head_stride, p.ks = f.k_token_stride, p.kh = f.k_head_stride;
    p.vs = f.v_token_stride, p.vh = f.v_head_stride, p.rs = f.k_rope_stride;
    p.queries = (long)queries, p.keys = (long)keys;
    p.batch = f.batch, p.len_q = f.seq_len, p.len_k = f.seq_len_k, p.heads = f.heads;
    p.d_n = f.d_n, p.d_r = f.d_r, p.d_v = f.d_v, p.causal = f.causal, p.scale = f.scale;
    const bool vec = attn_vectors(f) && aligned16(a.grad_o);
    p.vec_delta = f.d_v % (f.dtype == RHZ_F32 ? 4 : 8) == 0 && aligned16(f.o) && aligned16(a.grad_o);
    p.vec_out = vec && aligned16(a.grad_q) && aligned16(a.grad_k) && aligned16(a.grad_v);
    return f.dtype == RHZ_F32 ? launch_all<float>(p, vec, stream) : launch_all<uint16_t>(p, vec, stream);
}

}  // namespace rhz
