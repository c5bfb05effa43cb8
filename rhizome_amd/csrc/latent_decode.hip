// latent_decode.hip -- attention of a sequence's last positions over its paged
// latents, absorbed: the cache's row is the key, its first d_c values the value,
// of all heads.
//
// The rows of q of a sequence, `steps` positions by H heads, meet every cached
// row: 2 (2 d_c + d_r) flops a pair of rows against (d_c + d_r) e bytes a cached
// row, bound by memory up to some 128 rows of q.  A workgroup takes one split of
// the sequence, whose cached rows go through LDS once, there to be read along
// the row for the scores and transposed for the sum.  Splits go to the workspace
// with their maxima and sums, each normalised by its own, since a sum of weights
// times values can leave fp32's range where their mean does not, and are joined in
// order by another kernel.  Their number depends on the sequence's length alone, so that a
// sequence's result does not depend on its batch.
#include <algorithm>

#include "attn_device.hpp"
#include "gdr_internal.hpp"
#include "gdr_rows.hpp"

namespace rhz {
namespace {

constexpr int kTable = 1024;  // cached rows whose places are looked up at once
constexpr int kMaxSplits = 128, kUnit = 32;

// Cached rows of a split of a sequence of n rows: eighths of a short one, for one
// request's latency, of `least` rows at least, but of a long one `best` at most, as
// many as keep the parts' traffic low against the cache's own (at 16 heads a part is
// written and read again for 32 KB each against 1152 bytes a row).
//   bf16, 16 heads, least 64, 128, 256: one sequence of 517 positions 15.1, 15.3, 18.0
// us.  best 256, 512, 1024: one of 16384 - / 25 / 37 us, eight of them - / 38 / 46, 64
// of 2048 to 6084 97 / 87 / 76 (where splits of 512 are a few more than the card has
// places).
//   fp32 takes sixteen times as long for a row: best 128, 256, 512: one of 16384 39 /
// 60 / 107 us, sixteen of 4096 77 / 72 / 115, 32 of them 153 / 139 / 132; least 64,
// 128: one of 517 26 / 32.
struct SplitRule {
    int least, best;
};
template <typename T> constexpr SplitRule kRule = sizeof(T) == 4 ? SplitRule{64, 128} : SplitRule{128, 512};
__device__ __forceinline__ int split_rows(SplitRule r, int n) {
    const int eighth = min(max((n + 7) / 8, r.least), r.best), even = max(eighth, n / kMaxSplits + (n % kMaxSplits != 0));
    return (even + kUnit - 1) / kUnit * kUnit;
}
__device__ __forceinline__ int splits_of(SplitRule r, int n) {
    return n <= 0 ? 1 : (n + split_rows(r, n) - 1) / split_rows(r, n);
}
// No sequence of up to n rows has more.
inline int most_splits_of(SplitRule r, int64_t n) {
    const int64_t shortest = (n + r.least - 1) / r.least, best = (n + r.best - 1) / r.best;
    return (int)std::max<int64_t>(1, std::min(shortest, std::max<int64_t>(8, std::min<int64_t>(best, kMaxSplits))));
}

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

constexpr int64_t kMostRows = INT32_MAX - 4096;  // numbers of tiles' rows behind the last stay in 32 bits
__device__ __forceinline__ int rows_of(const DecodeParams& a, int seq) {
    const long room = min((long)a.max_pages * a.page, (long)kMostRows);
    return (int)min((long)max(a.lengths[seq], 0), room);
}

// What a workgroup is to do: of sequence `seq` the positions [begin, end) for
// the rows of q from `first_row` on.
struct Unit {
    int seq, split, splits, first_row, begin, end, n, length;
};
// The row tiles of a split follow one another on one XCD, whose L2 has the rows.
// First splits of all sequences come first: those that a sequence is too short to
// have are behind the others, where their workgroups, which end at once, do not
// disturb their distribution over the CUs (32 x 4096 positions, 128 rows: 73 us, and
// 113 with every ninth workgroup such a one).
template <typename T>
__device__ __forceinline__ bool unit_of(const DecodeParams& a, int tile_rows, Unit& u) {
    const int k = blockIdx.x >> 3, unit = k / a.row_tiles * 8 + (blockIdx.x & 7);
    if (unit >= a.batch * a.splits) return false;
    u.seq = unit % a.batch, u.split = unit / a.batch, u.first_row = k % a.row_tiles * tile_rows;
    u.length = a.lengths[u.seq];
    u.n = rows_of(a, u.seq);
    u.splits = splits_of(kRule<T>, u.n);
    u.begin = u.split * split_rows(kRule<T>, u.n);
    u.end = min(u.n, u.begin + split_rows(kRule<T>, u.n));
    return u.split < u.splits;
}
// Cache row of position j, -1 where its page is outside the cache.
__device__ __forceinline__ int cache_row(const DecodeParams& a, int seq, int j) {
    const int page = a.table[(long)seq * a.max_pages + j / a.page];
    return page >= 0 && page < a.num_pages ? page * a.page + j % a.page : -1;
}
// Positions that row r of q sees, by the length that the caller gave.
__device__ __forceinline__ int sees(const DecodeParams& a, const Unit& u, int r) {
    return (int)min((long)u.n, (long)u.length - a.steps + r / a.heads + 1);
}

// The unit's columns [d0, d0 + cols) of one row of q summed again over what the
// row sees, for rows that came out not finite (attn_device.hpp).
template <int N, typename T>
__device__ __forceinline__ void sum_unit_row_again(const DecodeParams& a, const Unit& u, int row, int d0, int cols, float m,
                                                   float f, int lane) {
    const float c = a.scale * kLog2e, mc = m == -INFINITY ? 0.f : m * c;
    const T* cache = (const T*)a.cache;
    const long at = (long)u.seq * a.steps * a.heads + row;
    const Rows<T> q = {(const T*)a.q + at * a.D, (const T*)a.q, 0, 0, a.D, 0}, k = {cache, cache, a.D, 0, a.D, 0};
    sum_row_again<N>(
        u.begin, min(u.end, sees(a, u, row)), cols, lane,
        [&](long j) {
            const int r = cache_row(a, u.seq, (int)j);
            return r < 0 ? 0.f : __builtin_amdgcn_exp2f(fmaf(dot_rows(q, 0, k, r), c, -mc)) * f;
        },
        [&](long j, int d) {
            const int r = cache_row(a, u.seq, (int)j);
            return r < 0 ? 0.f : Elem<T>::load(cache, (long)r * a.D + d0 + d);
        },
        [&](int d, float x) {
            if (u.splits > 1)
                a.part[(((long)u.seq * a.splits + u.split) * a.steps * a.heads + row) * a.d_c + d0 + d] = x;
            else
                Elem<T>::store((T*)a.o, at * a.d_c + d0 + d, x);
        });
}
// Maximum and sum of row r of q: to the workspace, or the logarithm where this is all.
__device__ __forceinline__ void store_sums(const DecodeParams& a, const Unit& u, int r, float m, float l) {
    const int rows = a.steps * a.heads;
    if (u.splits > 1) {
        const long at = ((long)u.seq * a.splits + u.split) * rows + r;
        a.part_m[at] = m, a.part_l[at] = l;
    } else if (a.lse) {
        a.lse[(long)u.seq * rows + r] = l == 0.f ? -INFINITY : fmaf(m, a.scale, logf(l));
    }
}

// 16 bytes a lane from p + OFF to LDS at lds; the instruction's offset counts in LDS too.
template <int OFF>
__device__ __forceinline__ void load_to_lds16_from(const void* p, uint32_t lds) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%2" ::"{m0}"(lds - OFF), "v"(p), "n"(OFF) : "memory");
}
// Panels K, K + STEP .. of a cached row from the lane's chunk of panel 0 at p on,
// `left` bytes of the row being left from there.
template <int K, int PANELS, int STEP>
__device__ __forceinline__ void load_panels(const void* p, int left, int row_bytes, uint32_t lds, int panel_bytes) {
    if constexpr (K < PANELS) {
        if ((K + 1) * 128 <= row_bytes)
            load_to_lds16_from<K * 128>(p, lds + K * panel_bytes);
        else if (K * 128 < left)
            load_to_lds16_from<K * 128>(p, lds + K * panel_bytes);
        load_panels<K + STEP, PANELS, STEP>(p, left, row_bytes, lds, panel_bytes);
    }
}

// ------------------------------------------------------- many rows, or fp32
// Eight waves, 32 RT rows of q, tiles of 32 cached rows.  8 / RT waves share a row
// tile, each with a part of the columns.  Of a tile a wave sums q . k over its
// part; the parts meet in LDS, and every wave of a row tile adds them up, takes the
// softmax -- all of them the same -- and sums its part of the columns with it.  In
// bf16 the second half of the row tiles is half a tile behind the first: between
// two barriers one wave of a SIMD multiplies queries and keys while the other is at
// the softmax and the sums (16 x 4096 positions at 128 rows 64 -> 59 us against all
// in step, at 256 rows 130 -> 114).  What bounds it is a workgroup's own way from
// tile to tile -- scores, their exchange, softmax and sums between two barriers --
// and the card's memory little: the 16 tiles of a split take 37, 39 and 45 us at 64
// rows with 64, 128 and 256 workgroups (8, 16 and 32 x 4096 positions), 48, 50 and 58
// at 128.  LDS has no room for a fourth tile, and reading the sums' columns ahead of
// the products changes nothing.
template <typename T, int VD, int RT, bool VEC>
__global__ __launch_bounds__(512, 2) void latent_decode_kernel(DecodeParams a) {
    constexpr int E = kChunkElems<T>, KD = VD + 64, BUFS = sizeof(T) == 2 ? 3 : 1, NT = 512, WAVES = 8, KEYS = 32;
    constexpr int PARTS = WAVES / RT, QP = KD / (2 * E) / PARTS, VTW = VD / 32 < PARTS ? 1 : VD / 32 / PARTS;  // column tiles of a wave
    static_assert(KD / (2 * E) % PARTS == 0, "whole chunk pairs for every part");
    using TILE = Tile<T, KD, KEYS>;
    __shared__ TILE tiles[BUFS];
    // 18 chunk pairs of q beside 8 column tiles of sums are four registers more
    // than there are: one pair goes through LDS (a spilled one waits for the loads)
    constexpr int KEPT = QP > 17 ? 17 : QP;
    __shared__ f32x4 scores[WAVES][4][kWave];  // [part, row tile][registers by four][lane]
    __shared__ u32x4 q_rest[QP > KEPT ? WAVES : 1][kWave];
    __shared__ int row_at[kTable];
    __shared__ uint32_t there[BUFS];  // a bit for every row of a tile: that its page is in the cache
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5;
    const LaneReads at = lane_reads<T>(lane);
    Unit u;
    if (!unit_of<T>(a, 32 * RT, u)) return;
    const int rows = a.steps * a.heads, begin = u.begin, end = u.end;

    const int part = wave % PARTS, mine = wave / PARTS;
    u32x4 q[KEPT];
    {
        const Rows<T> qrows = {(const T*)a.q, (const T*)a.q, a.D, 0, a.D, 0};
        const int r = min(u.first_row + 32 * mine + (lane & 31), rows - 1);
        const auto pair = [&](int i) { return load_chunk<T, VEC>(qrows, (long)u.seq * rows + r, 0, 2 * (part * QP + i) + g); };
#pragma unroll
        for (int i = 0; i < KEPT; ++i) q[i] = pair(i);
        if constexpr (QP > KEPT) q_rest[wave][lane] = pair(KEPT);
    }
    static_assert(QP <= KEPT + 1, "one pair of chunks in LDS");
#pragma unroll
    for (int i = 0; i < KEPT; ++i) settle(q[i]);
    if (a.D < TILE::kPanels * 8 * E)  // columns that no load writes
        for (int b = 0; b < BUFS; ++b)
            for (int i = tid; i < TILE::kPanels * KEYS * 8; i += NT) tiles[b].chunk[i] = u32x4{0, 0, 0, 0};

    const auto fill_table = [&](int j0) {
        for (int i = tid; i < kTable && j0 + i < end + KEYS; i += NT) row_at[i] = cache_row(a, u.seq, min(j0 + i, end - 1));
    };
    // Tile of positions j0 ..: those beyond the end repeat the last, those whose
    // page is outside the cache take row 0, which costs time if that is not
    // finite (sum_unit_row_again).  Half of the waves have the odd panels.
    const int my_panel = wave >> 2;
    const auto start = [&](int j0, int b) {
        const int i = tid & 255, r = i >> 3, c = (i & 7) ^ twist(r);
        const int row = row_at[(j0 - begin + r) % kTable];
        const unsigned long long in = __ballot(row >= 0);  // eight lanes a row
        uint32_t bits = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) bits |= uint32_t(in >> (8 * k) & 1) << k;
        if (lane == 0 && wave < 4) reinterpret_cast<uint8_t*>(&there[b])[wave] = uint8_t(bits);
        const T* p = (const T*)a.cache + (long)max(row, 0) * a.D;
        const uint32_t lds = lds_offset(&tiles[b].chunk[0]) + (wave & 3) * 64 * 16;
        if constexpr (VEC) {
            const int bytes = a.D * int(sizeof(T));
            if (my_panel == 0)
                load_panels<0, TILE::kPanels, 2>(p + c * E, bytes - c * 16, bytes, lds, TILE::kPanelBytes);
            else
                load_panels<1, TILE::kPanels, 2>(p + c * E, bytes - c * 16, bytes, lds, TILE::kPanelBytes);
        } else {
            const Rows<T> one = {p, p, 0, 0, a.D, 0};
#pragma unroll 1
            for (int k = my_panel; k < TILE::kPanels; k += 2)
                tiles[b].chunk[k * KEYS * 8 + i] = load_chunk<T, false>(one, 0, 0, k * 8 + c);
        }
    };
    f32x16 o[VTW];
#pragma unroll
    for (int d = 0; d < VTW; ++d) o[d] = f32x16{};
    float m = -INFINITY, l = 0.f;
    const float c = a.scale * kLog2e;
    const int least_seen = sees(a, u, u.first_row);
    const bool sums = part * VTW * 32 < VD;  // the wave has columns
    if (end > begin) fill_table(begin);
    __syncthreads();
    const int tiles_n = (end - begin + KEYS - 1) / KEYS;
    // Whether a tile's loads are as many as the waits below count: not where the last
    // panel has no columns (d_r = 0), where a tile waits for the next one's loads too
    // (32 x 4096 positions at 64 rows, 512 + 0 channels 44 us, 512 + 64 45).
    const bool counted = VEC && (a.D + 8 * E - 1) / (8 * E) == TILE::kPanels;
    // The wave's part of tile i's scores, to LDS.
    const auto score = [&](int i) {
        const uint32_t tile = lds_offset(&tiles[i % BUFS]);
        f32x16 s = {};
        // reads ahead of the products, whatever the scheduler would have
        constexpr int AHEAD = QP < 4 ? QP : 4;
        u32x4 x[AHEAD];
        const auto read = [&](int k) {
            const int pair = part * QP + k;
            return lds_read<u32x4>(((tile + at.row) ^ (((2 * pair) & 7) << 4)) + (pair >> 2) * TILE::kPanelBytes);
        };
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) x[k] = read(k);
#pragma unroll
        for (int k = 0; k < QP; ++k) {
            dot_chunks(s, x[k % AHEAD], k < KEPT ? q[k < KEPT ? k : 0] : q_rest[wave][lane], T());
            if (k + AHEAD < QP) x[k % AHEAD] = read(k + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) scores[wave][k][lane] = f32x4{s[4 * k], s[4 * k + 1], s[4 * k + 2], s[4 * k + 3]};
    };
    // All parts of tile i's scores, their softmax, and the wave's columns of the sum.
    const auto sum = [&](int i) {
        const uint32_t tile = lds_offset(&tiles[i % BUFS]);
        const int j0 = begin + i * KEYS;
        f32x16 s;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            f32x4 x = scores[mine * PARTS][k][lane];
#pragma unroll
            for (int v = 1; v < PARTS; ++v) x += scores[mine * PARTS + v][k][lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * k + e] = x[e];
        }
        const uint32_t in = __builtin_amdgcn_readfirstlane(there[i % BUFS]);
        if (j0 + KEYS > min(end, least_seen) || in != ~0u) {
            const int seen = min(end, sees(a, u, min(u.first_row + 32 * mine + (lane & 31), rows - 1))) - j0 - 4 * g;
            const uint32_t mine_in = in >> (4 * g);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int r = (k & 3) + 8 * (k >> 2);
                if (r >= seen || !(mine_in & 1u << r)) s[k] = -INFINITY;
            }
        }
        float top = s[0];
#pragma unroll
        for (int k = 1; k < 16; ++k) top = fmaxf(top, s[k]);
        top = max_of_halves(top);
        if (__any((top - m) * c > 8.f)) {
            const float up = fmaxf(m, top);
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - up) * c);
            m = up;
            l *= f;
#pragma unroll
            for (int d = 0; d < VTW; ++d)
#pragma unroll
                for (int k = 0; k < 16; ++k) o[d][k] *= f;
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            s[k] = __builtin_amdgcn_exp2f(fmaf(s[k], c, -mc));
            l += s[k];
        }
        if (!sums) return;
        Weights<T> p;
        p.set(s);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < VTW; ++d) {
            Columns<T> x;
            x.template load<TILE>(tile, at, 0, part * VTW + d);
            sum_rows(o[d], x, p);
        }
    };
    if constexpr (BUFS == 3) {
        if (tiles_n > 0) start(begin, 0);
        if (tiles_n > 1) start(begin + KEYS, 1);
        // Tile i has landed for all, while the next may be on its way.
        const auto arrive = [&](int i) {
            if (counted && i + 1 < tiles_n) {
                if (my_panel == 0)
                    wait_loads<(TILE::kPanels + 1) / 2>();
                else
                    wait_loads<TILE::kPanels / 2>();
            } else {
                wait_loads<0>();
            }
            lds_barrier();
        };
        // Tile i - 1 has been read by all: its place takes the next but one.
        const auto leave = [&](int i) {
            lds_barrier();
            if (i + 2 >= tiles_n) return;
            if ((i + 2) * KEYS % kTable == 0) {
                fill_table(begin + (i + 2) * KEYS);
                __syncthreads();
            }
            start(begin + (i + 2) * KEYS, (i + 2) % BUFS);
        };
        // both kinds of waves meet 2 tiles_n + 1 barriers
        if (tiles_n > 0 && mine < RT / 2) {
            for (int i = 0; i < tiles_n; ++i) {
                arrive(i);
                score(i);
                leave(i);
                sum(i);
            }
            lds_barrier();
        } else if (tiles_n > 0) {
            arrive(0);
            leave(0);
            for (int i = 0; i < tiles_n; ++i) {
                score(i);
                arrive(i + 1);
                sum(i);
                if (i + 1 < tiles_n) leave(i + 1);
            }
        }
    } else {
        for (int i = 0; i < tiles_n; ++i) {
            if (i * KEYS % kTable == 0 && i > 0) {
                __syncthreads();
                fill_table(begin + i * KEYS);
            }
            __syncthreads();
            start(begin + i * KEYS, 0);
            landed();
            score(i);
            lds_barrier();
            sum(i);
        }
    }
    l = sum_of_halves(l);
    const int r = u.first_row + 32 * mine + (lane & 31);
    bool live = r < rows;
    if (part == 0 && g == 0 && live) store_sums(a, u, r, m, l);
    if (!sums) return;
    const int d0 = part * VTW * 32, cols = min(a.d_c - d0, VTW * 32);  // the wave's columns
    const bool vec = a.d_c % 4 == 0 && aligned16(a.o);
    const float f = l == 0.f ? 0.f : 1.f / l;
    uint32_t again = not_finite_rows(o) & rows_with(live && l == l);
    while (again) {
        const int i = __ffs(again) - 1;
        again &= again - 1;
        sum_unit_row_again<(VTW + 1) / 2, T>(a, u, u.first_row + 32 * mine + i, d0, cols, __shfl(m, i, kWave),
                                             __shfl(f, i, kWave), lane);
        if ((lane & 31) == i) live = false;
    }
    if (!live) return;
    float* to_part = a.part + (((long)u.seq * a.splits + u.split) * rows + r) * a.d_c;
    T* to_o = (T*)a.o + ((long)u.seq * rows + r) * a.d_c;
#pragma unroll
    for (int d = 0; d < VTW; ++d) {
        if (u.splits > 1)
            store_columns<float>(to_part, o[d], d0 + 32 * d, a.d_c, f, vec, lane);
        else
            store_columns<T>(to_o, o[d], d0 + 32 * d, a.d_c, f, vec, lane);
    }
}

// ----------------------------------------- 16 rows a workgroup, up to 32, in bf16
// Four waves, each with cached rows of its own -- every fourth tile of 16 -- and
// a part of LDS for one tile, so that they need no barrier before their sums meet
// at the end.  On 16x16 matrix instructions: the scores come out with the lane's
// row of q as column and cached rows 4 g .. 4 g + 3 (g = lane / 16) in registers,
// which is how the sum over a tile's rows takes its weights.  78 KB of LDS at d_c
// = 512: two workgroups share a CU, and while some of its eight waves compute the
// others' tiles are on their way.  Bound by the cache's bytes: 64 sequences of
// 2048 to 6084 positions, 16 heads, 300 MB in 81 us (3.7 TB/s) and 6 of the join.
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

template <int VD>
__global__ __launch_bounds__(256, 2) void latent_decode_narrow_kernel(DecodeParams a) {
    constexpr int KD = VD + 64, KC = KD / 32, VT = VD / 16, KEYS = 16, WAVES = 4;  // steps of the scores, column tiles
    using T = uint16_t;
    using TILE = Tile<T, KD, KEYS>;
    constexpr int P = TILE::kPanels, PB = TILE::kPanelBytes;
    __shared__ TILE tiles[WAVES];
    __shared__ float wave_m[WAVES][16], wave_l[WAVES][16];
    __shared__ int row_at[kTable];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    Unit u;
    if (!unit_of<T>(a, 16, u)) return;
    const int rows = a.steps * a.heads, begin = u.begin, end = u.end;

    const auto fill_table = [&](int j0) {
        for (int i = tid; i < kTable && j0 + i < end + KEYS; i += 64 * WAVES)
            row_at[i] = cache_row(a, u.seq, min(j0 + i, end - 1));
    };
    if (end > begin) fill_table(begin);
    u32x4 q[KC];
    const Rows<T> qrows = {(const T*)a.q, (const T*)a.q, a.D, 0, a.D, 0};
    const int kr = lane & 15, row = u.first_row + kr;  // the lane's row of q
    const long q_row = (long)u.seq * rows + min(row, rows - 1);
#pragma unroll
    for (int i = 0; i < KC; ++i) q[i] = load_chunk<T, true>(qrows, q_row, 0, 4 * i + g);
    if (a.D < P * 64)  // columns that no load writes
        for (int i = lane; i < P * KEYS * 8; i += 64) tiles[wave].chunk[i] = u32x4{0, 0, 0, 0};
    __syncthreads();

    const uint32_t tile = lds_offset(&tiles[wave]);
    // Tile of positions j0 .., the two rows of each lane; returns a bit for every
    // row whose page is in the cache, the others take row 0.
    const auto start = [&](int j0) {
        uint32_t bits = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 8 * h + (lane >> 3), c = (lane & 7) ^ twist(r);
            const int row = row_at[(j0 - begin + r) % kTable];
            const unsigned long long in = __ballot(row >= 0);  // eight lanes a row
#pragma unroll
            for (int k = 0; k < 8; ++k) bits |= uint32_t(in >> (8 * k) & 1) << (8 * h + k);
            const T* p = (const T*)a.cache + (long)max(row, 0) * a.D + c * 8;
            load_panels<0, P, 1>(p, a.D * 2 - c * 16, a.D * 2, tile + h * 1024, PB);
        }
        return __builtin_amdgcn_readfirstlane(bits);
    };

    f32x4 o[VT];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < VT; ++d) o[d] = f32x4{};
    const float c = a.scale * kLog2e;
    const int least_seen = sees(a, u, u.first_row), seen = min(end, sees(a, u, min(row, rows - 1)));
    // row lane % 16, chunk 4 i + g; and transposed: rows 4 g + (lane % 16) / 4
    const int vr = 4 * g + (kr >> 2);
    const uint32_t k_at = tile + kr * 128 + ((twist(kr) ^ g) << 4), k_odd = k_at ^ (4 << 4);
    const uint32_t v_at = tile + vr * 128 + ((twist(vr) ^ ((kr >> 1) & 1)) << 4) + (kr & 1) * 8;

    const int tiles_n = (end - begin + KEYS - 1) / KEYS;
    uint32_t there = 0;
    if (wave < tiles_n) there = start(begin + wave * KEYS);
#pragma unroll
    for (int i = 0; i < KC; ++i) settle(q[i]);
    for (int i0 = 0; i0 < tiles_n; i0 += WAVES) {
        const int i = i0 + wave, j0 = begin + i * KEYS;
        if (i < tiles_n) {
            wait_loads<0>();
            // five reads ahead of the products, whatever the scheduler would have
            constexpr int AHEAD = 5;
            f32x4 s[2] = {};
            u32x4 x[AHEAD];
            const auto read = [&](int k) { return lds_read<u32x4>((k & 1 ? k_odd : k_at) + (k >> 1) * PB); };
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) x[k] = read(k);
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                s[k & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[k % AHEAD]),
                                                                   __builtin_bit_cast(bf16x8, q[k]), s[k & 1], 0, 0, 0);
                if (k + AHEAD < KC) x[k % AHEAD] = read(k + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
            }
            s[0] += s[1];
            if (j0 + KEYS > min(end, least_seen) || there != 0xffffu) {
                const int left = seen - j0 - 4 * g;
                const uint32_t in = there >> (4 * g);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k >= left || !(in & 1u << k)) s[0][k] = -INFINITY;
            }
            float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
            top = fmaxf(top, __shfl_xor(top, 16, kWave));
            top = max_of_halves(top);
            if (__any((top - m) * c > 8.f)) {
                const float up = fmaxf(m, top);
                const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - up) * c);
                m = up;
                l *= f;
#pragma unroll
                for (int d = 0; d < VT; ++d) o[d] *= f;
            }
            const float mc = m == -INFINITY ? 0.f : m * c;
            bf16x4_t w;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[0][k], c, -mc));
                l += p;
                w[k] = (__bf16)p;
            }
            const s16x4_t p = __builtin_bit_cast(s16x4_t, w);
            s16x4_t y[2 * AHEAD];
            const auto column = [&](int d) {
                const uint32_t v = (v_at ^ ((2 * (d & 3)) << 4)) + (d >> 2) * PB;
                return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4_t*>(v));
            };
            constexpr int COLS = VT < 2 * AHEAD ? VT : 2 * AHEAD;
#pragma unroll
            for (int d = 0; d < COLS; ++d) y[d] = column(d);
#pragma unroll
            for (int d = 0; d < VT; ++d) {
                o[d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(y[d % COLS], p, o[d], 0, 0, 0);
                if (d + COLS < VT) y[d % COLS] = column(d + COLS);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        const int next = i0 + WAVES;
        if (next < tiles_n && next * KEYS % kTable == 0) {  // the table ends; every wave has started all tiles before
            __syncthreads();
            fill_table(begin + next * KEYS);
            __syncthreads();
        }
        if (next + wave < tiles_n) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile has been read
            there = start(begin + (next + wave) * KEYS);
        }
    }

    // The waves' sums at their common maximum: waves 2 and 3 hand theirs to 0 and
    // 1, which exchange halves, so that each has the whole of half of the columns.
    l += __shfl_xor(l, 16, kWave);
    l = sum_of_halves(l);
    if (g == 0) wave_m[wave][kr] = m, wave_l[wave][kr] = l;
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, wave_m[w][kr]);
    const float tc = top == -INFINITY ? 0.f : top * c;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum = fmaf(wave_l[w][kr], __builtin_amdgcn_exp2f(fmaf(wave_m[w][kr], c, -tc)), sum);
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    const float own = __builtin_amdgcn_exp2f(fmaf(m, c, -tc)) * f;
    f32x4* given = reinterpret_cast<f32x4*>(&tiles[0]) + lane;
    if (wave >= 2) {
#pragma unroll
        for (int d = 0; d < VT; ++d) given[((wave - 2) * VT + d) * kWave] = o[d] * own;
    }
    __syncthreads();
    if (wave < 2) {
#pragma unroll
        for (int d = 0; d < VT; ++d) o[d] = o[d] * own + given[(wave * VT + d) * kWave];
    }
    __syncthreads();
    // by value: a choice between two places of o is an index, which would put o into memory
    const auto of_half = [&](int half, int d) {
        const f32x4 first = o[d], second = o[VT / 2 + d];
        return half ? second : first;
    };
    if (wave < 2) {
#pragma unroll
        for (int d = 0; d < VT / 2; ++d) given[(wave * (VT / 2) + d) * kWave] = of_half(1 - wave, d);
    }
    __syncthreads();
    if (wave >= 2) return;
    bool live = row < rows;
    if (wave == 0 && g == 0 && live) store_sums(a, u, row, top, sum);
    const int d0 = wave * (VD / 2), cols = min(a.d_c - d0, VD / 2);
    f32x4 x[VT / 2];
    float bad = 0.f;  // as not_finite_rows
#pragma unroll
    for (int d = 0; d < VT / 2; ++d) {
        x[d] = of_half(wave, d) + given[((1 - wave) * (VT / 2) + d) * kWave];
#pragma unroll
        for (int k = 0; k < 4; ++k) bad = fmaf(x[d][k], 0.f, bad);
    }
    unsigned long long flags = __ballot(bad != 0.f && live && sum == sum);
    flags |= flags >> 32;
    uint32_t again = cols > 0 ? uint32_t(flags | flags >> 16) & 0xffffu : 0;
    while (again) {
        const int i = __ffs(again) - 1;
        again &= again - 1;
        sum_unit_row_again<VD / 128, T>(a, u, u.first_row + i, d0, cols, __shfl(top, i, kWave), __shfl(f, i, kWave), lane);
        if (kr == i) live = false;
    }
    if (!live) return;
    const bool vec = a.d_c % 4 == 0 && aligned16(a.o);
    const long at_row = ((long)u.seq * a.splits + u.split) * rows + row;
    float* part = a.part + at_row * a.d_c;
    T* out = (T*)a.o + ((long)u.seq * rows + row) * a.d_c;
#pragma unroll
    for (int d = 0; d < VT / 2; ++d) {
        const int at = d0 + 16 * d + 4 * g;
        if (vec) {
            if (at >= a.d_c) continue;
            if (u.splits > 1)
                *reinterpret_cast<f32x4*>(part + at) = x[d];
            else
                *reinterpret_cast<uint2*>(out + at) = make_uint2(pack_bf16x2(x[d][0], x[d][1]), pack_bf16x2(x[d][2], x[d][3]));
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (at + k >= a.d_c) continue;
                if (u.splits > 1)
                    part[at + k] = x[d][k];
                else
                    Elem<T>::store(out, at + k, x[d][k]);
            }
        }
    }
}

// 256 columns of one row of q a workgroup: its splits by their shares of the sum
// of weights, every fourth split on one wave, the waves' sums added in order.
constexpr int kJoinThreads = 256, kJoinColumns = 256;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void latent_join_kernel(DecodeParams a) {
    __shared__ float weight[kMaxSplits];
    __shared__ f32x4 sums[3][kWave];
    const int rows = a.steps * a.heads, parts = (a.d_c + kJoinColumns - 1) / kJoinColumns;
    const int d = blockIdx.x % parts * kJoinColumns + (threadIdx.x & 63) * 4;
    const int unit = blockIdx.x / parts, seq = unit / rows, r = unit % rows, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int splits = splits_of(kRule<T>, rows_of(a, seq));
    if (splits == 1) return;
    const float c = a.scale * kLog2e;
    const long first = (long)seq * a.splits * rows + r;  // slot 0's; the next split's is `rows` further
    float m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool in = lane + 64 * i < splits;
        m[i] = in ? a.part_m[first + (long)(lane + 64 * i) * rows] : -INFINITY;
        l[i] = in ? a.part_l[first + (long)(lane + 64 * i) * rows] : 0.f;
    }
    const float top = wave_max(fmaxf(m[0], m[1])), tc = top == -INFINITY ? 0.f : top * c;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] *= __builtin_amdgcn_exp2f(fmaf(m[i], c, -tc));
        sum += l[i];
    }
    sum = row_sum<64>(sum);
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    if (wave == 0)
#pragma unroll
        for (int i = 0; i < 2; ++i) weight[lane + 64 * i] = l[i] * f;
    __syncthreads();
    const long row = (long)seq * rows + r;
    if (threadIdx.x == 0 && d == 0 && a.lse) a.lse[row] = sum == 0.f ? -INFINITY : fmaf(top, a.scale, logf(sum));
    const float* p = a.part + first * a.d_c + d;
    const long step = (long)rows * a.d_c;
    const bool vec = a.d_c % 4 == 0 && aligned16(a.o), in = d < a.d_c;
    f32x4 x = {};
    if (vec && in) {
#pragma unroll 8
        for (int i = wave; i < splits; i += 4) x += weight[i] * *reinterpret_cast<const f32x4*>(p + i * step);
    } else if (in) {
        for (int i = wave; i < splits; i += 4)
            for (int k = 0; k < 4 && d + k < a.d_c; ++k) x[k] = fmaf(weight[i], p[i * step + k], x[k]);
    }
    if (wave) sums[wave - 1][lane] = x;
    __syncthreads();
    if (wave || !in) return;
    x = ((x + sums[0][lane]) + sums[1][lane]) + sums[2][lane];
    T* out = (T*)a.o + row * a.d_c + d;
    if (!vec) {
        for (int k = 0; k < 4 && d + k < a.d_c; ++k) Elem<T>::store(out, k, x[k]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4*>(out) = x;
    } else {
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    }
}

int most_splits(const rhz_latent_decode_args& a) {
    return most_splits_of(a.dtype == RHZ_F32 ? kRule<float> : kRule<uint16_t>, std::min<int64_t>((int64_t)a.max_pages * a.page_size, kMostRows));
}

// The join's workgroups, none where no sequence can have two splits; -1 if there are too many.
int64_t join_blocks(const DecodeParams& p) {
    const int64_t blocks = (int64_t)p.batch * p.steps * p.heads * ((p.d_c + kJoinColumns - 1) / kJoinColumns);
    if (p.splits == 1) return 0;
    return check_grid(blocks, kJoinThreads) == hipSuccess ? blocks : -1;
}
template <typename T>
hipError_t join(const DecodeParams& p, int64_t blocks, hipStream_t stream) {
    if (blocks) latent_join_kernel<T><<<(unsigned)blocks, kJoinThreads, 0, stream>>>(p);
    return hipGetLastError();
}

// Workgroups of `threads` with `tile` rows of q each; 0 if there are too many.
unsigned blocks_of(DecodeParams& p, int tile, int threads) {
    p.row_tiles = (p.steps * p.heads + tile - 1) / tile;
    const int64_t blocks = ((int64_t)p.batch * p.splits + 7) / 8 * 8 * p.row_tiles;
    return blocks > INT32_MAX || check_grid(blocks, threads) != hipSuccess ? 0 : (unsigned)blocks;
}

template <typename T, int VD, int RT, bool VEC>
hipError_t launch(DecodeParams p, hipStream_t stream) {
    const unsigned blocks = blocks_of(p, 32 * RT, 512);
    const int64_t joins = join_blocks(p);
    if (!blocks || joins < 0) return hipErrorInvalidConfiguration;
    latent_decode_kernel<T, VD, RT, VEC><<<blocks, 512, 0, stream>>>(p);
    return join<T>(p, joins, stream);
}

template <int VD>
hipError_t launch_narrow(DecodeParams p, hipStream_t stream) {
    const unsigned blocks = blocks_of(p, 16, 256);
    const int64_t joins = join_blocks(p);
    if (!blocks || joins < 0) return hipErrorInvalidConfiguration;
    latent_decode_narrow_kernel<VD><<<blocks, 256, 0, stream>>>(p);
    return join<uint16_t>(p, joins, stream);
}

// By the rows of q of a sequence.  bf16, 32 sequences of 4096 positions, by the
// kernel of 16 rows, of 64, of 128: at 32 rows 42 / 49 / - us, at 64 68 / 54 / 69,
// at 96 94 / 93 / 66, at 128 119 / 95 / 72.  fp32, 16 sequences, by tiles of 32 or
// 64 rows: at 32 rows 116 / 173, at 64 121 / 178, so that all have 32.
template <typename T, int VD>
hipError_t pick_rows(const DecodeParams& p, bool vec, hipStream_t stream) {
    if constexpr (sizeof(T) == 4) {
        return vec ? launch<T, VD, 1, true>(p, stream) : launch<T, VD, 1, false>(p, stream);
    } else {
        const int rows = p.steps * p.heads;
        if (!vec) return launch<T, VD, 2, false>(p, stream);
        if (rows <= 32) return launch_narrow<VD>(p, stream);
        return rows <= 64 ? launch<T, VD, 2, true>(p, stream) : launch<T, VD, 4, true>(p, stream);
    }
}

// By the width of a latent: 32 sequences of 4096 positions, d_c 128 on the kernels
// of 128 and of 512 at 16 rows 18.4 / 27.0 us, at 64 rows 36.3 / 43.9, d_c 256 on
// those of 256 and of 512 24.6 / 29.1 and 41 / 45.  Not vec, the wide kernel reads
// values one by one: d_c 512, 64 rows 54 -> 128 us.
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
