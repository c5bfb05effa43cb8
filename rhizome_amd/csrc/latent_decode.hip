// latent_decode.hip -- attention of a sequence's last positions over its paged
// latents, absorbed: the cache's row is the key, its first d_c values the value,
// of all heads.
//
// The rows of q of a sequence, `steps` positions by H heads, meet every cached
// row: 2 (2 d_c + d_r) flops a value pair against (d_c + d_r) e bytes, bound by
// memory up to some 128 rows.  A workgroup takes 32 RT rows of q and one split
// of the sequence, whose cached rows come through LDS in tiles of 32, once for
// the scores (rows of the tile) and once for the sum (its columns).  Of a tile
//   scores: wave w sums q . k over its part of the columns for row tile w % RT;
//           the parts meet in LDS and every wave adds them up and takes the
//           softmax of all rows (cheaper than another exchange);
//   sum:    wave w has the columns from w d_c / 4 on of all rows.
// Splits go to the workspace unnormalised, with their maxima and sums, and are
// joined in order by a second kernel.  Their number depends on the sequence's
// length alone, so that a sequence's result does not depend on its batch.
#include <algorithm>

#include "attn_device.hpp"
#include "gdr_internal.hpp"
#include "gdr_rows.hpp"

namespace rhz {
namespace {

struct DecodeParams {
    const void *q, *cache;
    const int *table, *lengths;
    void* o;
    float* lse;
    float* part;  // [batch, splits, rows, d_c], then their maxima and sums
    float *part_m, *part_l;
    int batch, steps, heads, d_c, D, page, num_pages, max_pages, splits, row_tiles;
    float scale;
};

constexpr int kThreads = 256, kKeys = 32, kTable = 1024;
constexpr int kMaxSplits = 128, kMinSplit = 256;

// Cached rows of a split of a sequence of n rows.
__host__ __device__ inline int split_rows(int n) {
    const int even = (n + kMaxSplits - 1) / kMaxSplits;
    return max(kMinSplit, (even + kKeys - 1) / kKeys * kKeys);
}
__host__ __device__ inline int splits_of(int n) { return n <= 0 ? 1 : (n + split_rows(n) - 1) / split_rows(n); }

__device__ __forceinline__ int rows_of(const DecodeParams& a, int seq) {
    const long room = (long)a.max_pages * a.page;
    return (int)min((long)max(a.lengths[seq], 0), room);
}

// Waits for all but the last n loads of a wave.
template <int N>
__device__ __forceinline__ void landed_but() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
__device__ __forceinline__ void load_to_lds16_from(const void* p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory");
}

template <typename T, int VD, int RT, bool VEC>
__global__ __launch_bounds__(kThreads, 1) void latent_decode_kernel(DecodeParams a) {
    constexpr int E = kChunkElems<T>, KD = VD + 64, BUFS = sizeof(T) == 2 ? 3 : 1;
    constexpr int PARTS = 4 / RT, QP = KD / (2 * E) / PARTS, VTW = VD / 128;  // chunk pairs and column tiles of a wave
    using TILE = Tile<T, KD, kKeys>;
    __shared__ TILE tiles[BUFS];
    __shared__ f32x4 scores[4][4][kWave];  // [part, row tile][registers by four][lane]
    __shared__ int row_at[kTable];
    __shared__ uint32_t there[BUFS];  // a bit for every row of a tile: that its page is in the cache
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5;
    const LaneReads at = lane_reads<T>(lane);

    // the row tiles of a split follow one another on one XCD, whose L2 has the rows
    const int n_unit = blockIdx.x >> 3, unit = n_unit / a.row_tiles * 8 + (blockIdx.x & 7);
    if (unit >= a.batch * a.splits) return;
    const int seq = unit / a.splits, split = unit % a.splits, first_row = n_unit % a.row_tiles * 32 * RT;
    const int n = rows_of(a, seq), splits = splits_of(n);
    if (split >= splits) return;
    const int begin = split * split_rows(n), end = min(n, begin + split_rows(n));
    const int rows = a.steps * a.heads;
    const int length = a.lengths[seq];

    // cache row of position j, -1 where its page is outside the cache
    const auto cache_row = [&](int j) {
        const int page = a.table[(long)seq * a.max_pages + j / a.page];
        return page >= 0 && page < a.num_pages ? page * a.page + j % a.page : -1;
    };
    // positions that row r of q sees, by the length that the caller gave
    const auto sees = [&](int r) { return (int)min((long)n, (long)length - a.steps + r / a.heads + 1); };

    const int part = wave / RT, mine = wave % RT;
    u32x4 q[QP];
    {
        const Rows<T> qrows = {(const T*)a.q, (const T*)a.q, a.D, 0, a.D, 0};
        const int r = min(first_row + 32 * mine + (lane & 31), rows - 1);
#pragma unroll
        for (int i = 0; i < QP; ++i)
            q[i] = load_chunk<T, VEC>(qrows, (long)seq * rows + r, 0, 2 * (part * QP + i) + g);
    }
#pragma unroll
    for (int i = 0; i < QP; ++i) settle(q[i]);
    if (a.D < TILE::kPanels * 8 * E)  // columns that no load writes
        for (int b = 0; b < BUFS; ++b)
            for (int i = tid; i < TILE::kPanels * kKeys * 8; i += kThreads) tiles[b].chunk[i] = u32x4{0, 0, 0, 0};

    const auto fill_table = [&](int j0) {
        for (int i = tid; i < kTable && j0 + i < end + kKeys; i += kThreads) row_at[i] = cache_row(min(j0 + i, end - 1));
    };
    // Tile of positions j0 ..: those beyond the end repeat the last, those whose
    // page is outside the cache take row 0, which costs time if that is not
    // finite (below).
    const auto start = [&](int j0, int b) {
        const int r = tid >> 3, c = (tid & 7) ^ twist(r);
        const int row = row_at[(j0 - begin + r) % kTable];
        const unsigned long long in = __ballot(row >= 0);  // eight lanes a row
        uint32_t bits = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) bits |= uint32_t(in >> (8 * k) & 1) << k;
        if (lane == 0) reinterpret_cast<uint8_t*>(&there[b])[wave] = uint8_t(bits);
        const T* p = (const T*)a.cache + (long)max(row, 0) * a.D;
        const uint32_t lds = lds_offset(&tiles[b].chunk[0]) + wave * 64 * 16;
#pragma unroll
        for (int k = 0; k < TILE::kPanels; ++k) {
            const int d = (k * 8 + c) * E;
            if (k * 8 * E >= a.D) break;
            if constexpr (VEC) {
                if (d < a.D) load_to_lds16_from(p + d, lds + k * TILE::kPanelBytes);
            } else {
                const Rows<T> one = {p, p, 0, 0, a.D, 0};
                tiles[b].chunk[k * kKeys * 8 + tid] = load_chunk<T, false>(one, 0, 0, k * 8 + c);
            }
        }
    };
    f32x16 o[RT][VTW];
    float m[RT], l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        m[t] = -INFINITY, l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < VTW; ++d) o[t][d] = f32x16{};
    }
    const float c = a.scale * kLog2e;
    const int least_seen = sees(first_row);
    fill_table(begin);
    __syncthreads();
    const int tiles_n = (end - begin + kKeys - 1) / kKeys;
    const bool counted = VEC && (a.D + 8 * E - 1) / (8 * E) == TILE::kPanels;  // loads of a tile as the waits count them
    if constexpr (BUFS == 3) {
        if (tiles_n > 0) start(begin, 0);
        if (tiles_n > 1) start(begin + kKeys, 1);
    }
    for (int i = 0; i < tiles_n; ++i) {
        const int j0 = begin + i * kKeys, b = i % BUFS, ahead = i + BUFS - 1;
        if constexpr (BUFS == 3) {
            if (counted && i + 1 < tiles_n)
                landed_but<TILE::kPanels>();
            else
                landed();
        } else {
            landed();
        }
        if (ahead < tiles_n) {
            if (ahead * kKeys % kTable == 0 && ahead > 0) {
                fill_table(begin + ahead * kKeys);
                __syncthreads();
            }
            start(begin + ahead * kKeys, ahead % BUFS);
        }
        if constexpr (BUFS == 1) landed();
        const uint32_t tile = lds_offset(&tiles[b]);
        {
            f32x16 s = {};
#pragma unroll
            for (int k = 0; k < QP; ++k) {
                // chunk pair part * QP + k
                const int pair = part * QP + k;
                const uint32_t p = ((tile + at.row) ^ (((2 * pair) & 7) << 4)) + (pair >> 2) * TILE::kPanelBytes;
                dot_chunks(s, lds_read<u32x4>(p), q[k], T());
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) scores[wave][k][lane] = f32x4{s[4 * k], s[4 * k + 1], s[4 * k + 2], s[4 * k + 3]};
        }
        // LDS alone: the next tiles' loads stay on their way
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const uint32_t in = __builtin_amdgcn_readfirstlane(there[b]);
        const bool masked = j0 + kKeys > min(end, least_seen) || in != ~0u;
        Weights<T> p[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            f32x16 s;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                f32x4 x = scores[t][k][lane];
#pragma unroll
                for (int u = 1; u < PARTS; ++u) x += scores[t + RT * u][k][lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * k + e] = x[e];
            }
            if (masked) {
                const int seen = min(end, sees(min(first_row + 32 * t + (lane & 31), rows - 1)));
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int r = (k & 3) + 8 * (k >> 2) + 4 * g;
                    if (j0 + r >= seen || !(in >> r & 1)) s[k] = -INFINITY;
                }
            }
            float top = s[0];
#pragma unroll
            for (int k = 1; k < 16; ++k) top = fmaxf(top, s[k]);
            top = fmaxf(top, __shfl_xor(top, 32, kWave));
            if (__any((top - m[t]) * c > 8.f)) {
                const float up = fmaxf(m[t], top);
                const float f = m[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[t] - up) * c);
                m[t] = up;
                l[t] *= f;
#pragma unroll
                for (int d = 0; d < VTW; ++d)
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[t][d][k] *= f;
            }
            const float mc = m[t] == -INFINITY ? 0.f : m[t] * c;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                s[k] = __builtin_amdgcn_exp2f(fmaf(s[k], c, -mc));
                l[t] += s[k];
            }
            p[t].set(s);
        }
#pragma unroll
        for (int d = 0; d < VTW; ++d) {
            Columns<T> x;
            const int dt = wave * VTW + d;
            x.template load<TILE>(tile, at, 0, dt);
#pragma unroll
            for (int t = 0; t < RT; ++t) sum_rows(o[t][d], x, p[t]);
        }
    }

    const long slot = (long)seq * a.splits + split;
    const int d0 = wave * VTW * 32, cols = min(a.d_c - d0, VTW * 32);  // the wave's columns
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        l[t] += __shfl_xor(l[t], 32, kWave);
        const int r = first_row + 32 * t + (lane & 31);
        bool live = r < rows;
        const float f = splits > 1 ? 1.f : l[t] == 0.f ? 0.f : 1.f / l[t];
        const auto out = [&](int row, int d, float x) {
            if (splits > 1)
                a.part[(slot * rows + row) * a.d_c + d] = x;
            else
                Elem<T>::store((T*)a.o, ((long)seq * rows + row) * a.d_c + d, x);
        };
        uint32_t again = not_finite_rows(o[t]) & uint32_t(__ballot(live));
        while (again) {  // the row's sum once more over what it sees
            const int i = __ffs(again) - 1, row = first_row + 32 * t + i;
            again &= again - 1;
            const float mr = __shfl(m[t], i, kWave), fr = __shfl(f, i, kWave);
            const float mc = mr == -INFINITY ? 0.f : mr * c;
            const Rows<T> qr = {(const T*)a.q + ((long)seq * rows + row) * a.D, (const T*)a.q, 0, 0, a.D, 0};
            const Rows<T> kr = {(const T*)a.cache, (const T*)a.cache, a.D, 0, a.D, 0};
            sum_row_again<VTW>(
                begin, min(end, sees(row)), cols, lane,
                [&](long j) {
                    const int at = cache_row((int)j);
                    return at < 0 ? 0.f : __builtin_amdgcn_exp2f(fmaf(dot_rows(qr, 0, kr, at), c, -mc)) * fr;
                },
                [&](long j, int d) {
                    const int at = cache_row((int)j);
                    return at < 0 ? 0.f : Elem<T>::load(kr.p, (long)at * a.D + d0 + d);
                },
                [&](int d, float x) { out(row, d0 + d, x); });
            if ((lane & 31) == i) live = false;
        }
        if (wave == 0 && g == 0 && r < rows) {
            if (splits > 1)
                a.part_m[slot * rows + r] = m[t], a.part_l[slot * rows + r] = l[t];
            else if (a.lse)
                a.lse[(long)seq * rows + r] = l[t] == 0.f ? -INFINITY : fmaf(m[t], a.scale, logf(l[t]));
        }
        if (!live) continue;
        const bool vec = a.d_c % 4 == 0 && aligned16(a.o);
#pragma unroll
        for (int d = 0; d < VTW; ++d) {
            if (splits > 1)
                store_columns<float>(a.part + (slot * rows + r) * a.d_c, o[t][d], d0 + 32 * d, a.d_c, 1.f, vec, lane);
            else
                store_columns<T>((T*)a.o + ((long)seq * rows + r) * a.d_c, o[t][d], d0 + 32 * d, a.d_c, f, vec, lane);
        }
    }
}

// One row of q a workgroup: its splits' sums at their common maximum.
constexpr int kJoinThreads = 128;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void latent_join_kernel(DecodeParams a) {
    __shared__ float weight[kMaxSplits];
    const int rows = a.steps * a.heads, seq = blockIdx.x / rows, r = blockIdx.x % rows, tid = threadIdx.x;
    const int splits = splits_of(rows_of(a, seq));
    if (splits == 1) return;
    const float c = a.scale * kLog2e;
    const long first = (long)seq * a.splits * rows + r;  // slot 0's; the next split's is `rows` further
    float top = -INFINITY, sum = 0.f;
    for (int i = 0; i < splits; ++i) top = fmaxf(top, a.part_m[first + (long)i * rows]);
    const float tc = top == -INFINITY ? 0.f : top * c;
    if (tid < splits) weight[tid] = __builtin_amdgcn_exp2f(fmaf(a.part_m[first + (long)tid * rows], c, -tc));
    __syncthreads();
    for (int i = 0; i < splits; ++i) sum = fmaf(weight[i], a.part_l[first + (long)i * rows], sum);
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    const long row = (long)seq * rows + r;
    if (tid == 0 && a.lse) a.lse[row] = sum == 0.f ? -INFINITY : fmaf(top, a.scale, logf(sum));
    const float* p = a.part + first * a.d_c;
    const long step = (long)rows * a.d_c;
    T* out = (T*)a.o + row * a.d_c;
    if (a.d_c % 4 == 0 && aligned16(a.o)) {
        for (int d = tid * 4; d < a.d_c; d += kJoinThreads * 4) {
            f32x4 x = {};
#pragma unroll 8
            for (int i = 0; i < splits; ++i) x += weight[i] * *reinterpret_cast<const f32x4*>(p + i * step + d);
            if constexpr (sizeof(T) == 4)
                *reinterpret_cast<f32x4*>(out + d) = x * f;
            else
                *reinterpret_cast<uint2*>(out + d) = make_uint2(pack_bf16x2(x[0] * f, x[1] * f), pack_bf16x2(x[2] * f, x[3] * f));
        }
    } else {
        for (int d = tid; d < a.d_c; d += kJoinThreads) {
            float x = 0.f;
            for (int i = 0; i < splits; ++i) x = fmaf(weight[i], p[i * step + d], x);
            Elem<T>::store(out, d, x * f);
        }
    }
}

int most_splits(const rhz_latent_decode_args& a) {
    return splits_of((int)std::min<int64_t>((int64_t)a.max_pages * a.page_size, INT32_MAX));
}

template <typename T, int VD, int RT, bool VEC>
hipError_t launch(DecodeParams p, hipStream_t stream) {
    const int rows = p.steps * p.heads;
    p.row_tiles = (rows + 32 * RT - 1) / (32 * RT);
    const int64_t blocks = ((int64_t)p.batch * p.splits + 7) / 8 * 8 * p.row_tiles, joins = (int64_t)p.batch * rows;
    if (blocks > INT32_MAX || joins > INT32_MAX || check_grid(blocks, kThreads) != hipSuccess ||
        check_grid(joins, kJoinThreads) != hipSuccess)
        return hipErrorInvalidConfiguration;
    latent_decode_kernel<T, VD, RT, VEC><<<(unsigned)blocks, kThreads, 0, stream>>>(p);
    if (p.splits > 1) latent_join_kernel<T><<<(unsigned)joins, kJoinThreads, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T, int VD>
hipError_t pick_rows(const DecodeParams& p, bool vec, hipStream_t stream) {
    const int rows = p.steps * p.heads;
    if (!vec) return launch<T, VD, 1, false>(p, stream);
    if (rows <= 32) return launch<T, VD, 1, true>(p, stream);
    if constexpr (sizeof(T) == 2)  // four row tiles' accumulators and queries fill the registers in bf16
        if (rows > 64) return launch<T, VD, 4, true>(p, stream);
    return launch<T, VD, 2, true>(p, stream);
}

template <typename T>
hipError_t pick(const DecodeParams& p, hipStream_t stream) {
    const bool vec = p.D % kChunkElems<T> == 0 && aligned16(p.q) && aligned16(p.cache);
    if (p.d_c <= 128) return pick_rows<T, 128>(p, vec, stream);
    if (p.d_c <= 256) return pick_rows<T, 256>(p, vec, stream);
    return pick_rows<T, 512>(p, vec, stream);
}

size_t part_floats(const rhz_latent_decode_args& a) { return (size_t)a.batch * most_splits(a) * a.steps * a.heads; }

}  // namespace

size_t latent_decode_workspace_bytes(const rhz_latent_decode_args& a) {
    return most_splits(a) == 1 ? 0 : part_floats(a) * (a.d_c + 2) * 4;
}

hipError_t launch_latent_decode(const rhz_latent_decode_args& a, hipStream_t stream) {
    DecodeParams p = {};
    p.q = a.q, p.cache = a.cache, p.table = a.page_table, p.lengths = a.lengths, p.o = a.o, p.lse = a.lse;
    p.batch = a.batch, p.steps = a.steps, p.heads = a.heads, p.d_c = a.d_c, p.D = a.d_c + a.d_r;
    p.page = a.page_size, p.num_pages = a.num_pages, p.max_pages = a.max_pages, p.splits = most_splits(a);
    p.scale = a.scale;
    p.part = (float*)a.workspace;
    p.part_m = p.part + part_floats(a) * a.d_c;
    p.part_l = p.part_m + part_floats(a);
    return a.dtype == RHZ_F32 ? pick<float>(p, stream) : pick<uint16_t>(p, stream);
}

}  // namespace rhz
