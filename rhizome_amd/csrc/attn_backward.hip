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
template <int DQ, int DV, bool VEC>
__global__ __launch_bounds__(kThreads, 1) void attn_dkv_kernel(BackwardParams a) {
    using T = uint16_t;
    constexpr int E = kChunkElems<T>, BQ = 64, SUB = BQ / 32;
    constexpr int QC = DQ / (2 * E), VC = DV / (2 * E), QT = DQ / 32, VT = DV / 32;
    __shared__ Tile<T, DQ, BQ> qtiles[2];
    __shared__ Tile<T, DV, BQ> otiles[2];
    __shared__ float4 lse_s[2][16], delta_s[2][16];  // a wave's 64 floats
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5;
    const LaneReads at = lane_reads<T>(lane);
    int head, seq, tile;
    if (!place(a, a.cu_k, a.len_k, kRows, lane, head, seq, tile)) return;
    const Range w = seq_range(a.cu_q, a.cu_k, seq, a.len_q, a.len_k);
    const int first = tile * kRows;
    if (first >= w.nk) return;
    const int wk = first + wave * 32, kj = wk + (lane & 31);
    const int shift = w.nk - w.nq;

    u32x4 kf[QC], vf[VC];
    const Rows<T> krows = {(const T*)a.k + head * a.kh, (const T*)(a.r ? a.r : a.k), a.ks, a.rs, a.d_n, a.d_r};
    const Rows<T> vrows = {(const T*)a.v + head * a.vh, (const T*)a.v, a.vs, 0, a.d_v, 0};
    {
        const int r = min(kj, w.nk - 1) - first;
#pragma unroll
        for (int c = 0; c < QC; ++c) kf[c] = load_chunk<T, VEC>(krows, (long)w.k0 + first, r, 2 * c + g);
#pragma unroll
        for (int c = 0; c < VC; ++c) vf[c] = load_chunk<T, VEC>(vrows, (long)w.k0 + first, r, 2 * c + g);
    }
    const Rows<T> qrows = {(const T*)a.q + head * a.qh, (const T*)a.q, a.qs, 0, a.d_n + a.d_r, 0};
    const Rows<T> orows = {(const T*)a.go + (long)head * a.d_v, (const T*)a.go, (long)a.heads * a.d_v, 0, a.d_v, 0};
    const float* lse2 = a.lse2 + head * a.queries + w.q0;
    const float* delta = a.delta + head * a.queries + w.q0;
    const Mover<T, DQ, BQ, kThreads, VEC> move_q(qrows, tid);
    const Mover<T, DV, BQ, kThreads, VEC> move_o(orows, tid);
    const auto start = [&](int q0, int b) {
        move_q.start((long)w.q0 + q0, w.nq - q0, qtiles[b]);
        move_o.start((long)w.q0 + q0, w.nq - q0, otiles[b]);
        const uint32_t off = min(lane, min(BQ, w.nq - q0) - 1) * 4;
        if (wave == 0) load_to_lds4(lse2 + q0, off, lds_offset(&lse_s[b][0]));
        if (wave == 1) load_to_lds4(delta + q0, off, lds_offset(&delta_s[b][0]));
    };
#pragma unroll
    for (int c = 0; c < QC; ++c) settle(kf[c]);
#pragma unroll
    for (int c = 0; c < VC; ++c) settle(vf[c]);
    f32x16 dk[QT], dv[VT];
#pragma unroll
    for (int d = 0; d < QT; ++d) dk[d] = f32x16{};
#pragma unroll
    for (int d = 0; d < VT; ++d) dv[d] = f32x16{};
    const float c = a.scale * kLog2e;
    // the first query that sees the workgroup's first key
    const int begin = a.causal ? max(0, first - shift) / BQ * BQ : 0;
    for (int b = 0; b < 2; ++b) move_q.clear(qtiles[b]), move_o.clear(otiles[b]);
    __syncthreads();
    if (begin < w.nq) start(begin, 0);
    for (int q0 = begin, b = 0; q0 < w.nq; q0 += BQ, b ^= 1) {
        landed();
        if (q0 + BQ < w.nq) start(q0 + BQ, b ^ 1);
        const uint32_t qt = lds_offset(&qtiles[b]);
        const uint32_t ot = lds_offset(&otiles[b]);
        if (a.causal && q0 + BQ - 1 + shift < wk) continue;  // sees none of the wave's keys
#pragma unroll 1  // both halves at once take more registers than there are
        for (int u = 0; u < SUB; ++u) {
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int i = 0; i < QC; ++i) dot_chunks(s, read_row<Tile<T, DQ, BQ>>(qt, at, u, i), kf[i], T());
#pragma unroll
            for (int i = 0; i < VC; ++i) dot_chunks(dp, read_row<Tile<T, DV, BQ>>(ot, at, u, i), vf[i], T());
            const int qu = q0 + 32 * u;
            // the lane's key is seen by the tile's queries from number `from` on
            const int from = a.causal ? kj - shift - qu : 0;
            const bool masked = qu + 32 > w.nq || (a.causal && wk + 31 - shift > qu);
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const float4 lq = lse_s[b][8 * u + 2 * i4 + g], dq = delta_s[b][8 * u + 2 * i4 + g];
                const float ls[4] = {lq.x, lq.y, lq.z, lq.w}, ds[4] = {dq.x, dq.y, dq.z, dq.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = 4 * i4 + j;
                    s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -ls[j]));
                    dp[i] = s[i] * (dp[i] - ds[j]);
                }
            }
            if (masked) {
                const int least = from - 4 * g, left = w.nq - qu - 4 * g;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = (i & 3) + 8 * (i >> 2);
                    if (r < least || r >= left) s[i] = dp[i] = 0.f;
                }
            }
            Weights<T> p, ds;
            p.set(s);
            ds.set(dp);
#pragma unroll
            for (int d = 0; d < VT; ++d) {
                Columns<T> x;
                x.template load<Tile<T, DV, BQ>>(ot, at, u, d);
                sum_rows(dv[d], x, p);
            }
#pragma unroll
            for (int d = 0; d < QT; ++d) {
                Columns<T> x;
                x.template load<Tile<T, DQ, BQ>>(qt, at, u, d);
                sum_rows(dk[d], x, ds);
            }
        }
    }
    bool live = kj < w.nk;
    uint32_t again = (not_finite_rows(dv) | not_finite_rows(dk)) & uint32_t(__ballot(live));
    while (again) {
        const int r = __ffs(again) - 1;
        again &= again - 1;
        const long mine = (long)w.k0 + wk + r, row = mine * a.heads + head;
        const int from = a.causal ? max(0, wk + r - shift) : 0;  // the first query that sees the key
        const auto weight = [&](long i) {
            return __builtin_amdgcn_exp2f(fmaf(dot_rows(qrows, i, krows, mine), c, -lse2[i - w.q0]));
        };
        sum_row_again<2>((long)w.q0 + from, (long)w.q0 + w.nq, a.d_v, lane, weight,
                         [&](long i, int d) { return value(orows, i, d); },
                         [&](int d, float x) { Elem<T>::store((T*)a.dv + row * a.d_v, d, x); });
        sum_row_again<3>(
            (long)w.q0 + from, (long)w.q0 + w.nq, a.d_n + a.d_r, lane,
            [&](long i) { return weight(i) * (dot_rows(orows, i, vrows, mine) - delta[i - w.q0]) * a.scale; },
            [&](long i, int d) { return value(qrows, i, d); },
            [&](int d, float x) {
                if (d < a.d_n)
                    Elem<T>::store((T*)a.dk + row * a.d_n, d, x);
                else
                    a.dr_part[(head * a.keys + mine) * a.d_r + d - a.d_n] = x;
            });
        if ((lane & 31) == r) live = false;
    }
    if (!live) return;
    const long token = (long)w.k0 + kj, row = token * a.heads + head;
    T* gv = (T*)a.dv + row * a.d_v;
#pragma unroll
    for (int d = 0; d < VT; ++d) store_columns<T>(gv, dv[d], 32 * d, a.d_v, 1.f, a.vec_out, lane);
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

// ---------------------------------------------------------------------- dq
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
    if (!place(a, a.cu_q, a.len_q, kRows, lane, head, seq, tile)) return;
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
#pragma unroll
        for (int i = 0; i < QC; ++i) dot_chunks(s, read_row<Tile<T, DQ, BN>>(kt, at, 0, i), qf[i], T());
#pragma unroll
        for (int i = 0; i < VC; ++i) dot_chunks(dp, read_row<Tile<T, DV, BN>>(vt, at, 0, i), of[i], T());
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
#pragma unroll
        for (int d = 0; d < QT; ++d) {
            Columns<T> x;
            x.template load<Tile<T, DQ, BN>>(kt, at, 0, d);
            sum_rows(dq[d], x, ds);
        }
    }
    bool live = qi < w.nq;
    uint32_t again = not_finite_rows(dq) & uint32_t(__ballot(live));
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
    if (p.keys) {
        const unsigned blocks = attn_blocks(p.heads, p.batch, p.cu_k, tk);
        if (!blocks) return hipErrorInvalidConfiguration;
        p.tiles = (int)tk;
        attn_dkv_kernel<DQ, DV, VEC><<<blocks, kThreads, 0, stream>>>(p);
    }
    if (p.queries) {
        const unsigned blocks = attn_blocks(p.heads, p.batch, p.cu_q, tq);
        if (!blocks) return hipErrorInvalidConfiguration;
        p.tiles = (int)tq;
        attn_dq_kernel<DQ, DV, VEC><<<blocks, kThreads, 0, stream>>>(p);
    }
    return hipGetLastError();
}

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
