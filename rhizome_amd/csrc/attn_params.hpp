// attn_params.hpp -- what the latent attention's prefill kernels are given, and
// which rows of which head a workgroup has.
#pragma once

#include "attn_device.hpp"
#include "gdr_internal.hpp"
#include "gdr_rows.hpp"

namespace rhz {

struct PrefillParams {
    const void *q, *k, *v, *r;
    const int *cu_q, *cu_k;
    void* o;
    float* lse;
    long qs, qh, ks, kh, vs, vh, rs;
    int batch, len_q, len_k, heads, d_n, d_r, d_v, causal;
    int tiles;  // of a head's queries, in all sequences of a pack or in one of a dense batch
    float scale;
};

struct BackwardParams {
    const void *q, *k, *v, *r, *go;
    const int *cu_q, *cu_k;
    const float *lse, *glse;
    const void* o;
    void *dq, *dk, *dv, *dr;
    float* lse2;     // [H, queries]: lse log2 e
    float* delta;    // [H, queries]: D
    float* dr_part;  // [H, keys, d_r]
    long qs, qh, ks, kh, vs, vh, rs, queries, keys;
    int batch, len_q, len_k, heads, d_n, d_r, d_v, causal;
    int tiles;  // as above, of queries or of keys
    float scale;
    bool vec_out, vec_delta;
};

constexpr int kAttnThreads = 256;

// Heads (of sequences) whose workgroups are mixed on an XCD.
constexpr int kMixed = 4;

// Number t of a causal pack's tiles of SIZE rows, those with the longest way first;
// false if there are not so many.  One lane a sequence.  The j-th longest of a
// sequence's T tiles sees between top - j and top - j + 1 tiles' worth of the other
// side's rows (queries: top = T + (nk - nq) / SIZE, keys: top = nk / SIZE), so that
// each has one tile at each of T levels: the level of number t is found by
// bisection, then the sequence among those that have it.
template <int SIZE, bool KEYS>
__device__ __forceinline__ bool longest_tile(const int* cu_q, const int* cu_k, int batch, int len_q, int len_k, int t, int lane,
                                             int& seq, int& tile) {
    const Range w = seq_range(cu_q, cu_k, min(lane, batch - 1), len_q, len_k);
    const int rows = KEYS ? w.nk : w.nq, n = lane < batch ? (rows + SIZE - 1) / SIZE : 0;
    const int top = KEYS ? w.nk / SIZE : n + (w.nk - w.nq >= 0 ? (w.nk - w.nq) / SIZE : -((w.nq - w.nk + SIZE - 1) / SIZE));
    const auto above = [&](int level) {  // tiles at this level or above, through scalar registers as in wave_max
        const int x = __builtin_bit_cast(int, lane_group_sum<16>((float)min(max(top - level + 1, 0), n)));
        float sum = 0.f;
#pragma unroll
        for (int row = 0; row < kWave; row += 16) sum += __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, row));
        return __builtin_amdgcn_readfirstlane((int)sum);
    };
    int hi = __builtin_amdgcn_readfirstlane((int)wave_max(n ? (float)top : -1e9f));
    int lo = -__builtin_amdgcn_readfirstlane((int)wave_max(n ? (float)(n - 1 - top) : -1e9f));
    if (lo > hi || above(lo) <= t) return false;
    while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (above(mid) > t)
            lo = mid;
        else
            hi = mid - 1;
    }
    const int rank = t - above(lo + 1);  // by all lanes together
    const bool has = top >= lo && top - lo < n;
    const int before = __popcll(__ballot(has) & ((1ull << lane) - 1));
    const int at = __ffsll((long long)__ballot(has && before == rank)) - 1;
    seq = __builtin_amdgcn_readfirstlane(max(at, 0));
    tile = __builtin_amdgcn_readfirstlane(__shfl(top - lo, seq, kWave));
    return at >= 0;
}
// 12 sequences of 1 to 2222 tokens, 9415 in all, 16 heads of 128 + 64 channels in bf16:
// prefill 125 -> 110 us, backward 431 -> 412.  The fp32 kernels, of 32 rows a
// workgroup, gain nothing (386 us both) and have their tiles sequence by sequence,
// as have packs beyond these sizes: a lane has one sequence, and what is counted
// stays exact in fp32.
constexpr int kMostSorted = kWave, kLongestSorted = 1 << 28;

// Workgroup number -> head, sequence and tile of SIZE rows of the queries or KEYS;
// false if there is none.  A head's workgroups are on one XCD,
// whose L2 keeps what they all read.  There they start in order, by turns on its
// quarters, so that a place stays empty until its turn comes: kMixed heads' tiles
// of one number, which take about as long, follow one another.  2 x 4096 tokens, 32
// heads, by 1, 2, 4 and 8 of them: prefill 411, 386, 374, 375 us, backward 1487,
// 1432, 1402, 1411.
template <int SIZE, bool KEYS, typename PARAMS>
__device__ __forceinline__ bool place(const PARAMS& a, unsigned block, int lane, int& head, int& seq, int& tile) {
    const int* cu = KEYS ? a.cu_k : a.cu_q;
    const int units = a.heads * (cu ? 1 : a.batch);
    const int xcd = block & 7, n = block >> 3;
    const int here = (units - xcd + 7) >> 3;  // units of this XCD
    const int group = n / (kMixed * a.tiles), mixed = min(kMixed, here - group * kMixed);
    if (mixed <= 0) return false;
    const int m = n - group * kMixed * a.tiles;
    if (m >= mixed * a.tiles) return false;
    const int unit = (group * kMixed + m % mixed) * 8 + xcd;
    head = unit % a.heads;
    tile = m / mixed;
    seq = unit / a.heads;
    if (!cu) return true;
    if (SIZE > 32 && a.causal && a.batch > 1 && a.batch <= kMostSorted && a.len_q <= kLongestSorted && a.len_k <= kLongestSorted)
        return longest_tile<SIZE, KEYS>(a.cu_q, a.cu_k, a.batch, a.len_q, a.len_k, tile, lane, seq, tile);
    packed_tile(cu, a.batch, KEYS ? a.len_k : a.len_q, SIZE, tile, lane, seq, tile);
    return true;
}
// Workgroups for `tiles` tiles of every head; 0 if there are too many.
inline unsigned attn_blocks(int heads, int batch, const int* cu, int64_t tiles, int threads = kAttnThreads) {
    const int64_t units = ((int64_t)heads * (cu ? 1 : batch) + 7) / 8 * 8;
    const int64_t blocks = tiles > INT32_MAX ? INT64_MAX / 2 : units * tiles;
    return blocks > INT32_MAX || check_grid(blocks, threads) != hipSuccess ? 0 : (unsigned)blocks;
}
inline int64_t attn_tiles(const int* cu, int64_t total, int len, int batch, int size) {
    return cu ? packed_tiles(total, batch, size) : ((int64_t)len + size - 1) / size;
}

// The fp32 kernels (attn_split.hip); vec: as attn_vectors.
hipError_t launch_prefill_split(PrefillParams p, bool vec, hipStream_t stream);
// dk, dv and the heads' parts of the rotary key's gradient, then dq.
hipError_t launch_backward_split(BackwardParams p, bool vec, hipStream_t stream);

}  // namespace rhz
