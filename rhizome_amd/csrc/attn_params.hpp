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

// Workgroup number -> head, sequence and tile of `size` rows of the side whose
// offsets are `cu`; false if there is none.  A head's workgroups are on one XCD,
// whose L2 keeps what they all read.  There they start in order, by turns on its
// quarters, so that a place stays empty until its turn comes: kMixed heads' tiles
// of one number, which take about as long, follow one another.  2 x 4096 tokens, 32
// heads, by 1, 2, 4 and 8 of them: prefill 411, 386, 374, 375 us, backward 1487,
// 1432, 1402, 1411.
template <typename PARAMS>
__device__ __forceinline__ bool place(const PARAMS& a, unsigned block, const int* cu, int total, int size, int lane, int& head,
                                      int& seq, int& tile) {
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
    if (cu) packed_tile(cu, a.batch, total, size, tile, lane, seq, tile);
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
