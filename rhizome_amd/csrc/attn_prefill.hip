// attn_prefill.hip -- latent attention over expanded keys and values.
//
// One pass over the keys with the running maximum m and sum l of the softmax:
// a workgroup of four waves has 128 queries of one head, a wave 32 of them, in
// the arrangement of attn_device.hpp, and K and V go by in tiles through LDS.
// Per tile and wave
//     S = K Q^T,   p = 2^(S c - m c),   l += sum p,   O^T += V^T p
// with c = scale log2 e.  The maximum is only raised, and O and l rescaled,
// where a tile's exceeds it by 2^8 or more: p then is at most 2^8, which costs
// neither fp32 sums nor bf16 weights any digits.
//
// Tiles of 64 keys, twice, take 80 KB at 192 + 128 channels, so that two
// workgroups share a CU and one's products run beside the other's softmax.
// 2 x 4096 tokens, 32 heads of 128 + 64 channels, causal: 364 us, 944 TFLOP/s of
// the two products' 344 GF, against 298 us at the 1152 TFLOP/s of a large matrix
// product.  What bounds it: matrix instructions take 42 % of the time and the
// vector unit 36 % (the exponentials above all); without the loads and their
// barriers it would still be 322 us.  Measured at 371 us for this shape and not
// better: S of the next tile ahead of the softmax within a wave 385, eight waves a
// workgroup 382, loads spread over the products 391, tile loads behind S 392.
#include "attn_params.hpp"

namespace rhz {
namespace {

using T = uint16_t;
constexpr int kThreads = kAttnThreads, kQueries = 128;

template <int DQ, int DV, bool VEC>
__global__ __launch_bounds__(kThreads, 2) void latent_prefill_kernel(PrefillParams a) {
    constexpr int E = kChunkElems<T>, BN = 64, SUB = BN / 32;
    constexpr int QC = DQ / (2 * E), VT = DV / 32;
    __shared__ Tile<T, DQ, BN> ktiles[2];
    __shared__ Tile<T, DV, BN> vtiles[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5;
    const LaneReads at = lane_reads<T>(lane);

    int head, seq, tile;
    if (!place<kQueries, false>(a, blockIdx.x, lane, head, seq, tile)) return;
    const Range w = seq_range(a.cu_q, a.cu_k, seq, a.len_q, a.len_k);
    if (tile * kQueries >= w.nq) return;
    const int first = ((w.nq - 1) / kQueries - tile) * kQueries;  // the queries with the most keys go first

    const int wq = first + wave * 32;       // the wave's first query
    const int qi = wq + (lane & 31);        // the lane's
    bool live = qi < w.nq;
    const int shift = w.nk - w.nq;          // query i sees keys 0 .. i + shift
    const int last_q = min(first + kQueries, w.nq) - 1;
    const int end = a.causal ? min(w.nk, last_q + shift + 1) : w.nk;

    u32x4 q[QC];
    const Rows<T> qrows = {(const T*)a.q + head * a.qh, (const T*)a.q, a.qs, 0, a.d_n + a.d_r, 0};
#pragma unroll
    for (int c = 0; c < QC; ++c) q[c] = load_chunk<T, VEC>(qrows, (long)w.q0 + first, min(qi, w.nq - 1) - first, 2 * c + g);
    const Rows<T> krows = {(const T*)a.k + head * a.kh, (const T*)(a.r ? a.r : a.k), a.ks, a.rs, a.d_n, a.d_r};
    const Rows<T> vrows = {(const T*)a.v + head * a.vh, (const T*)a.v, a.vs, 0, a.d_v, 0};
#pragma unroll
    for (int c = 0; c < QC; ++c) settle(q[c]);
    f32x16 o[VT];
#pragma unroll
    for (int d = 0; d < VT; ++d) o[d] = f32x16{};
    const float c = a.scale * kLog2e;
    float m = -INFINITY, l = 0.f;
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
        if (a.causal && k0 > wq + 31 + shift) continue;  // none of the wave's queries sees the tile
        f32x16 s[SUB];
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            s[u] = f32x16{};
            dot_ahead<QC, 6>(s[u], q, [&](int i) { return read_row<Tile<T, DQ, BN>>(kt, at, u, i); }, T());
        }
        const int seen = a.causal ? min(w.nk, qi + shift + 1) : w.nk;  // keys that the lane's query sees
        const bool masked = k0 + BN > w.nk || (a.causal && k0 + BN > wq + shift + 1);
        if (masked) {
            const int left = seen - k0 - 4 * g;
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * u + (i & 3) + 8 * (i >> 2) >= left) s[u][i] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
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
        for (int u = 0; u < SUB; ++u) {
            SumAhead<T, Tile<T, DV, BN>, VT, 2> sum;
            sum.begin(vt, at, u);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[u][i] = __builtin_amdgcn_exp2f(fmaf(s[u][i], c, -mc));
                l += s[u][i];
            }
            Weights<T> p;
            p.set(s[u]);
            sum.run(o, vt, at, u, p);
        }
    }
    l = sum_of_halves(l);
    const float f = l == 0.f ? 0.f : 1.f / l;
    uint32_t again = not_finite_rows(o) & rows_with(live && l == l);
    while (again) {
        const int r = __ffs(again) - 1;
        again &= again - 1;
        const long mine = (long)w.q0 + wq + r;
        const float mr = __shfl(m, r, kWave), fr = __shfl(f, r, kWave);
        const float mc = mr == -INFINITY ? 0.f : mr * c;
        const int sees = a.causal ? min(w.nk, wq + r + shift + 1) : w.nk;
        sum_row_again<2>(
            w.k0, (long)w.k0 + sees, a.d_v, lane,
            [&](long j) { return __builtin_amdgcn_exp2f(fmaf(dot_rows(qrows, mine, krows, j), c, -mc)) * fr; },
            [&](long j, int d) { return value(vrows, j, d); },
            [&](int d, float x) { Elem<T>::store((T*)a.o + (mine * a.heads + head) * a.d_v, d, x); });
        if ((lane & 31) == r) live = false;
    }
    if (g == 0 && qi < w.nq) a.lse[(long)(w.q0 + qi) * a.heads + head] = l == 0.f ? -INFINITY : fmaf(m, a.scale, logf(l));
    if (!live) return;
    const long row = (long)(w.q0 + qi) * a.heads + head;
    T* out = (T*)a.o + row * a.d_v;
#pragma unroll
    for (int d = 0; d < VT; ++d) store_columns<T>(out, o[d], 32 * d, a.d_v, f, VEC, lane);
}

template <int DQ, int DV, bool VEC>
hipError_t launch(PrefillParams p, hipStream_t stream) {
    const int64_t queries = p.cu_q ? (int64_t)p.len_q : (int64_t)p.batch * p.len_q;
    const int64_t tiles = attn_tiles(p.cu_q, queries, p.len_q, p.batch, kQueries);
    const unsigned blocks = attn_blocks(p.heads, p.batch, p.cu_q, tiles);
    if (!blocks) return hipErrorInvalidConfiguration;
    p.tiles = (int)tiles;
    latent_prefill_kernel<DQ, DV, VEC><<<blocks, kThreads, 0, stream>>>(p);
    return hipGetLastError();
}

// The narrowest kernel that holds the channels.  2 x 4096 tokens, 16 heads, by the
// kernels for (64, 64), (96, 64), (128, 128) and (192, 128) channels of keys and
// values: of 64 and 64 104 / - / 164 / 187 us, of 96 and 64 - / 115 / 150 / 169, of
// 128 and 128 - / - / 162 / 184.  Not vec, values are loaded one by one and tiles
// written by the threads: 526 us instead of 115 at 96 and 64.
hipError_t pick(const PrefillParams& p, bool vec, hipStream_t stream) {
    const int dq = p.d_n + p.d_r;
    if (!vec) return dq <= 64 && p.d_v <= 64 ? launch<64, 64, false>(p, stream) : launch<192, 128, false>(p, stream);
    if (p.d_v <= 64 && dq <= 64) return launch<64, 64, true>(p, stream);
    if (p.d_v <= 64 && dq <= 96) return launch<96, 64, true>(p, stream);
    if (dq <= 128) return launch<128, 128, true>(p, stream);
    return launch<192, 128, true>(p, stream);
}

}  // namespace

bool attn_vectors(const rhz_latent_prefill_args& a) {
    const int e = a.dtype == RHZ_F32 ? 4 : 8;
    const bool rope = a.d_r == 0 || (aligned16(a.k_rope) && a.k_rope_stride % e == 0);
    return a.d_n % e == 0 && a.d_r % e == 0 && a.d_v % e == 0 && rope && aligned16(a.q) && aligned16(a.k) &&
           aligned16(a.v) && aligned16(a.o) && a.q_token_stride % e == 0 && a.q_head_stride % e == 0 &&
           a.k_token_stride % e == 0 && a.k_head_stride % e == 0 && a.v_token_stride % e == 0 && a.v_head_stride % e == 0;
}

hipError_t launch_latent_prefill(const rhz_latent_prefill_args& a, hipStream_t stream) {
    const int64_t queries = a.cu_seqlens ? (int64_t)a.seq_len : (int64_t)a.batch * a.seq_len;
    if (queries == 0) return hipSuccess;
    const PrefillParams p = {a.q, a.k, a.v, a.k_rope, a.cu_seqlens, a.cu_seqlens_k ? a.cu_seqlens_k : a.cu_seqlens, a.o, a.lse,
                       a.q_token_stride, a.q_head_stride, a.k_token_stride, a.k_head_stride, a.v_token_stride,
                       a.v_head_stride, a.k_rope_stride, a.batch, a.seq_len, a.seq_len_k, a.heads, a.d_n, a.d_r, a.d_v,
                       a.causal, 0, a.scale};
    const bool vec = attn_vectors(a);
    return a.dtype == RHZ_F32 ? launch_prefill_split(p, vec, stream) : pick(p, vec, stream);
}

}  // namespace rhz
