// Grouped products of 16-bit operands on tcgen05 with operands by TMA.
//
// All three products are tiles D[128 features][TN rows of the output] of sums over `depth`:
//   linear           features: columns of W, rows: gathered rows of x, depth: k
//   input gradient   features: rows of W,    rows: gathered rows of y, depth: n
//   weight gradient  features: columns of y, rows: columns of x,       depth: the rows of a group, gathered
// The features lie on the 128 accumulator lanes because they are many whatever the group: the other side of the tile shrinks to
// the rows a group has (multiples of 16), so a group of one row costs an MMA of 16 columns, and an accumulator column is
// a run of the output row: 32 lanes store 64 or 128 consecutive bytes.
//
// Rows are where the groups' order says: they come by TMA gather (four row numbers an instruction), which fills what is no row
// with zeros, so that the linears permute nothing in memory. Of the weight gradient the same holds where it has few tiles; where
// it has many, each of which would gather its rows anew, both matrices are first laid by groups (plan_of). Weights come by TMA
// tiles from the caller's layout. Operands whose depth runs along memory are K-major tiles, the others MN-major ones; both with
// the 128-byte swizzle. What TMA cannot take (rows or weights at no multiple of 16 bytes) is copied to aligned rows first.
//
// What bounds it: few rows, the bytes of the weights (8 rows, 8 groups of 2,048 x 2,048: see launch_rows); many, the tensor cores
// (16,384 rows of 4,096 x 4,096 in 4 groups: 1.52 PFLOP/s) and with deep gathers the 30 cycles that one takes.

#include "grouped_tc.cuh"

#include <algorithm>

namespace fmb {
namespace grp {

namespace {

using namespace tc;

constexpr int kEpilogueWarps = 8;
constexpr int kChunk = 512;                      // weight gradient: depth after which an accumulator moves to registers

// SORTED, of the weight gradient: the rows lie by groups (sort_rows)
template <int MODE, int TN, bool PAIR, bool SORTED> struct Shape {
    static constexpr bool kWeights = MODE == kWeightGradient;
    static constexpr int kCtas = PAIR ? 2 : 1, kRows = TN / kCtas;                 // rows of the tile that a CTA brings
    static constexpr bool kSplits = !kWeights && TN == 32;                         // may share the depth of a tile (Args::split)
    static constexpr int kFeatureBytes = 128 * kDepth * 2, kRowBytes = kRows * kDepth * 2;
    static constexpr int kStageBytes = kFeatureBytes + kRowBytes;
    static constexpr int kRowsPerWarp = PAIR ? 16 : 32, kQuads = kRowsPerWarp / 4;
    // Warps that issue copies: of the linears warp 0 for the features, the others for rows, 32 (16 of a pair) each; of the weight
    // gradient one per 64 columns of y or x, or one in all where the rows are sorted. An SM takes in a gather (512 bytes) every 18
    // cycles at best, one warp issues one every 30. Then the warp that issues MMAs, and eight that take results out, two sets of
    // four.
    static constexpr int kGathers = kWeights ? 2 + kRows / 64 : kRows / kRowsPerWarp, kCopyWarps = SORTED ? 1 : kWeights ? kGathers : 1 + kGathers;
    static constexpr int kMmaWarp = kCopyWarps;
    static constexpr int kFirstEpilogue = kWeights ? 8 : kMmaWarp + 1;             // whole warpgroups, so that registers can be dealt
    static constexpr int kThreads = 32 * (kFirstEpilogue + kEpilogueWarps);
    // results turn through shared memory, 32 rows of 128 features at a time and set
    static constexpr int kTurnBytes = 32 * 128 * (kWeights ? 4 : 2);
    static constexpr int kRoom = 226 * 1024 - 2 * kTurnBytes - 1024 - (FMB_MAX_GROUPS + 1) * 4 - 256 - kCopyWarps * 512 - (kWeights ? (FMB_MAX_GROUPS + 1) * 8 : 0);
    static constexpr int kStages = kRoom / kStageBytes < 8 ? kRoom / kStageBytes : 8;
    static constexpr int kTurn0 = kStages * kStageBytes, kRows0 = kTurn0 + 2 * kTurnBytes, kUnits0 = kRows0 + kCopyWarps * 512,
                         kCosts0 = kUnits0 + ((FMB_MAX_GROUPS + 1) * 4 + 7) / 8 * 8, kBars0 = kCosts0 + (kWeights ? (FMB_MAX_GROUPS + 1) * 8 : 0);
    static constexpr int kSmem = 1024 + kBars0 + 256;
    static constexpr int kTmem = 2 * TN < 32 ? 32 : 2 * TN;
    static_assert(!kSplits || 7 * TN * 128 * 4 <= kStages * kStageBytes, "room for the sums of seven CTAs");
    static_assert(kStages >= 3 && kSmem <= 227 * 1024 && kMmaWarp < kFirstEpilogue, "fits an SM");
};

struct Args {
    fmb_grouped_t a;
    int feature_tiles, row_tiles;                // of the output; row_tiles 1 where rows are gathered
    int unit_rows;                               // entries of a group per unit
    int split = 1;                               // linears of few rows: CTAs, a cluster, that share the depth of a tile; one tile each
    int wide_store;                              // output rows may be written 16 bytes at a time
    int by_tma;                                  // weight gradient: as boxes of 16 rows, by weight_map
    const int32_t* first_block;                  // SORTED: blocks of 64 rows of the groups before each
};

template <typename T, int MODE, int TN, bool PAIR, bool SORTED>
__global__ void __launch_bounds__(Shape<MODE, TN, PAIR, SORTED>::kThreads, 1)
k_grouped_tc(const __grid_constant__ Args p, const __grid_constant__ CUtensorMap feature_map, const __grid_constant__ CUtensorMap row_map,
             const __grid_constant__ CUtensorMap weight_map) {
    using S = Shape<MODE, TN, PAIR, SORTED>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    int* const first_unit = reinterpret_cast<int*>(smem + S::kUnits0);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + S::kBars0);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S::kStages + 4);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars), stage0 = smem_u32(smem);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (S::kStages + s); };
    auto acc_full = [&](int b) { return bar0 + 8u * (2 * S::kStages + b); };
    auto acc_empty = [&](int b) { return bar0 + 8u * (2 * S::kStages + 2 + b); };
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    constexpr bool kWeights = S::kWeights;
    constexpr int kMmaWarp = S::kMmaWarp;

    // of a pair: CTA 0 leads; both walk the same tiles, each with its own 128 features and half of the rows to bring
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;
    auto copy_bar = [&](int s) { return PAIR ? in_leader(full(s)) : full(s); };
    auto expect = [&](uint32_t bar, uint32_t bytes) {
        if constexpr (PAIR) {
            if (bytes) remote_expect_tx(bar, bytes);
            else remote_arrive(bar);
        } else {
            if (bytes) mbar_expect_tx(bar, bytes);
            else mbar_arrive(bar);
        }
    };
    auto gather = [&](uint32_t dst, const CUtensorMap* map, int column, const int4& r, uint32_t bar) {
        if constexpr (PAIR) tma_gather4_pair(dst, map, column, r.x, r.y, r.z, r.w, bar);
        else tma_gather4(dst, map, column, r.x, r.y, r.z, r.w, bar);
    };
    auto tile = [&](uint32_t dst, const CUtensorMap* map, int column, int row, uint32_t bar) {
        if constexpr (PAIR) tma_tile_2d_pair(dst, map, column, row, bar);
        else tma_tile_2d(dst, map, column, row, bar);
    };
    auto box = [&](uint32_t dst, int c0, int c1, int c2, uint32_t bar) {
        if constexpr (PAIR) tma_tile_3d_pair(dst, &feature_map, c0, c1, c2, bar);
        else tma_tile_3d(dst, &feature_map, c0, c1, c2, bar);
    };

    if (warp == 0) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(tmem_slot)), "r"(S::kTmem) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            tmem_alloc(smem_u32(tmem_slot), S::kTmem);
        }
    }
    if (warp == kMmaWarp && elect_one()) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(full(s), S::kCopyWarps * S::kCtas);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), kEpilogueWarps * S::kCtas);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    count_units<S::kThreads>(p.a.offsets, p.a.groups, p.a.rows, p.unit_rows, kWeights ? 1 : 0, first_unit);
    fence_before_sync();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    // Tiles of the linears cost the same, and go round: those that share rows or weights run at the same time and find them in L2
    // (16,384 rows of 4,096 x 4,096 in 4 groups: 376 us, and 614 in consecutive runs of the same cost). Those of the weight gradient
    // cost what their group has rows: every CTA (pair) takes consecutive tiles of the same cost in all (where tiles went round sizes
    // that differ by a factor of three cost 40 %; equal shares of the cost going round leave CTAs with a tile too many: 224 -> 273 us
    // for 100,000 rows of 768 x 768 in 128 groups).
    const bool split = S::kSplits && p.split > 1;
    const int ctas = split ? p.split : S::kCtas, walkers = gridDim.x / ctas, walker = blockIdx.x / ctas, part = split ? blockIdx.x % p.split : 0;
    const int all_tiles = units_in_all(first_unit, p.a.groups, p.a.rows, p.unit_rows) * p.feature_tiles * p.row_tiles;
    int t_first = walker, t_end = split ? min(all_tiles, walkers) : all_tiles;
    const int t_step = kWeights ? 1 : walkers;
    if constexpr (kWeights) {
        long long* const cost = reinterpret_cast<long long*>(smem + S::kCosts0);
        if (warp == 0) {
            long long before = 0;
            for (int g0 = 0; g0 < p.a.groups; g0 += 32) {
                const int g = g0 + lane;
                long long mine = 0;
                if (g < p.a.groups) {
                    int begin, end;
                    group_span(p.a.offsets, g, p.a.rows, begin, end);
                    const int units = first_unit[g + 1] - first_unit[g];
                    // a tile takes as long as its blocks or, 128 KB written per CTA, as four of them (0, 4, 6, 9: 160, 147, 152, 154 us
                    // for 16,384 rows of 2,048 x 1,024 in 32 groups)
                    mine = (max((long long)(end - begin + kDepth - 1) / kDepth, 4ll * units) + units) * p.feature_tiles * p.row_tiles;
                }
                long long inclusive = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long up = __shfl_up_sync(0xffffffffu, inclusive, o);
                    if (lane >= o) inclusive += up;
                }
                if (g < p.a.groups) cost[g] = before + inclusive - mine;
                before += __shfl_sync(0xffffffffu, inclusive, 31);
            }
            if (lane == 0) cost[p.a.groups] = before;
        }
        __syncthreads();
        auto first_tile = [&](int c) {
            if (c >= walkers) return all_tiles;
            const long long target = cost[p.a.groups] / walkers * c + cost[p.a.groups] % walkers * c / walkers;
            int low = 0, high = p.a.groups - 1;
            while (low < high) {
                const int mid = (low + high + 1) >> 1;
                if (cost[mid] <= target) low = mid; else high = mid - 1;
            }
            const long long tiles_of = (long long)(first_unit[low + 1] - first_unit[low]) * p.feature_tiles * p.row_tiles, span = cost[low + 1] - cost[low];
            const long long skip = span > 0 ? ((target - cost[low]) * tiles_of + span / 2) / span : 0;
            return first_unit[low] * p.feature_tiles * p.row_tiles + (int)min(skip, tiles_of);
        };
        t_first = min(first_tile(walker), all_tiles);
        t_end = min(first_tile(walker + 1), all_tiles);
    }
    // not of the weight gradient
    const int depth_of_row = MODE == kLinear ? p.a.k : p.a.n, row_blocks = (depth_of_row + kDepth - 1) / kDepth;
    const int first_block = split ? row_blocks * part / p.split : 0, last_block = split ? row_blocks * (part + 1) / p.split : row_blocks;

    Walk w(p.a, first_unit, p.unit_rows, p.feature_tiles, p.row_tiles, TN);
    if (warp >= S::kFirstEpilogue) {
        // of the weight gradient eight warps with 72 registers a thread and eight with 184: 256 x 256, as at the launch
        if constexpr (kWeights) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        // ---------------------------------------------------------------- results
        const int quarter = warp & 3, set = (warp - S::kFirstEpilogue) >> 2, id = quarter * 32 + lane;     // lanes 32 quarter + [0, 32)
        int acc = 0;
        uint32_t acc_phase = 0;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        auto accumulator_read = [&](int b) {
            if constexpr (PAIR) remote_arrive(in_leader(acc_empty(b)));
            else mbar_arrive(acc_empty(b));
        };
        // a wait that runs out does not end these loops: the set's warps meet at barriers, and all have to come
        if constexpr (kWeights) {
            constexpr int kCols = TN / 2;                        // of a set
            float* const turn = reinterpret_cast<float*>(smem + S::kTurn0 + set * S::kTurnBytes);
            for (int t = t_first; t < t_end; t += t_step) {
                if (t == t_first) w.start(t);
                else w.step(t_step);
                const int chunks = (w.count + kChunk - 1) / kChunk;
                float sum[kCols];
#pragma unroll
                for (int j = 0; j < kCols; ++j) sum[j] = 0.0f;
                for (int c = 0; c < chunks; ++c) {
                    mbar_wait(acc_full(acc), acc_phase, abort_flag, kSpin);
                    fence_after_sync();
#pragma unroll
                    for (int j0 = 0; j0 < kCols; j0 += 32) {
                        float v[32];
                        tmem_load_32(tmem + lanes + acc * TN + set * kCols + j0, v);
#pragma unroll
                        for (int j = 0; j < 32; ++j) sum[j0 + j] += v[j];
                    }
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) accumulator_read(acc);
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1;
                }
                const bool direct = w.units <= 1;
                const long long stride = direct ? p.a.w_row_stride : p.a.n;
                const int feature = w.feature0 * S::kCtas + rank * 128 + 4 * lane, live = p.a.n - feature;
                float* const out = (direct ? (float*)p.a.w + w.g * p.a.w_group_stride : p.a.scratch + w.slot * p.a.k * p.a.n) + feature;
                const bool add = direct && p.a.accumulate, wide = direct ? p.wide_store : p.a.n % 4 == 0;
                const int row0 = w.row0 + set * kCols;
                if (direct && p.by_tma) {
                    // 16 rows at a time through two buffers, and on by TMA (threads that wrote the rows themselves, 32 at a time, as
                    // below: 269 us for 100,000 rows of 768 x 768 in 128 groups, and 223 so)
#pragma unroll
                    for (int j0 = 0; j0 < kCols; j0 += 16) {
                        float* const box = turn + (j0 & 16) * 128;
                        if (id == 0) bulk_wait_read<1>();
                        named_barrier(1 + set, 128);              // what was in the box has been read
#pragma unroll
                        for (int j = 0; j < 16; ++j) box[j * 128 + id] = sum[j0 + j];
                        fence_to_async();
                        named_barrier(1 + set, 128);
                        if (id == 0) {
                            const int column = w.feature0 * S::kCtas + rank * 128;
                            if (row0 + j0 < p.a.k && column < p.a.n) tma_store_3d(&weight_map, smem_u32(box), column, row0 + j0, w.g);
                            bulk_commit();
                        }
                    }
                    continue;
                }
                if (id == 0) bulk_wait_read<0>();
#pragma unroll
                for (int j0 = 0; j0 < kCols; j0 += 32) {
                    named_barrier(1 + set, 128);                  // what was here has been read
#pragma unroll
                    for (int j = 0; j < 32; ++j) turn[j * 128 + id] = sum[j0 + j];
                    named_barrier(1 + set, 128);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int r = j * 4 + quarter, row = row0 + j0 + r;
                        float4 v = *reinterpret_cast<const float4*>(turn + r * 128 + 4 * lane);
                        if (row >= p.a.k) continue;
                        float* const to = out + row * stride;
                        if (wide) {
                            if (live > 0) {
                                if (add) {
                                    const float4 old = *reinterpret_cast<const float4*>(to);
                                    v.x += old.x; v.y += old.y; v.z += old.z; v.w += old.w;
                                }
                                *reinterpret_cast<float4*>(to) = v;
                            }
                        } else {
                            if (live > 0) to[0] = add ? to[0] + v.x : v.x;
                            if (live > 1) to[1] = add ? to[1] + v.y : v.y;
                            if (live > 2) to[2] = add ? to[2] + v.z : v.z;
                            if (live > 3) to[3] = add ? to[3] + v.w : v.w;
                        }
                    }
                }
            }
            if (id == 0) bulk_wait();
        } else {
            T* const out = (T*)(MODE == kLinear ? p.a.y : p.a.x);
            const long long stride = MODE == kLinear ? p.a.y_stride : p.a.x_stride;
            const int width = MODE == kLinear ? p.a.n : p.a.k;
            T* const turn = reinterpret_cast<T*>(smem + S::kTurn0 + set * S::kTurnBytes);      // [32 rows][128 features]
            if (p.a.zero_rest) {
                // rows of no group
                const int from = min(max(p.a.offsets[p.a.groups], 0), p.a.rows), first = blockIdx.x * kEpilogueWarps + warp - S::kFirstEpilogue;
                for (int i = from + first; i < p.a.rows; i += gridDim.x * kEpilogueWarps) {
                    const int row = row_at(p, i, p.a.rows);
                    if (row >= 0)
                        for (int c = lane; c < width; c += 32) out[row * stride + c] = from_float<T>(0.0f);
                }
            }
            for (int t = t_first; t < t_end; t += t_step) {
                if (t == t_first) w.start(t);
                else w.step(t_step);
                mbar_wait(acc_full(acc), acc_phase, abort_flag, kSpin);
                fence_after_sync();
                if constexpr (S::kSplits) {
                    __syncwarp();
                    if (split) cluster_sync();       // every CTA's products are done, and the stages of the first one free
                    if (split && part > 0) {
                        // its sums [32 rows][128 features] into the place of this one in the first CTA's stages
                        float v[32];
                        const uint32_t to = in_leader(stage0) + (uint32_t)((part - 1) * 32 * 128 + id) * 4;
                        if (set == 0) {
                            tmem_load_32(tmem + lanes, v);
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (j < w.count) asm volatile("st.shared::cluster.f32 [%0], %1;" :: "r"(to + j * 512), "f"(v[j]) : "memory");
                        }
                        __syncwarp();
                        cluster_sync();
                        break;
                    }
                    if (split) cluster_sync();
                }
                const int feature = w.feature0 * S::kCtas + rank * 128 + 8 * (lane & 15), live = width - feature;
                // the sets take turns at blocks of 32 rows
#pragma unroll 1
                for (int j0 = set * 32; j0 < w.count; j0 += 64) {
                    const int mine = row_at(p, w.first + j0 + lane, w.first + w.count);
                    float v[32];
                    tmem_load_32(tmem + lanes + acc * TN + j0, v);
                    if constexpr (S::kSplits) {
                        for (int q = 1; q < ctas; ++q) {
                            const float* const from = reinterpret_cast<const float*>(smem) + (q - 1) * 32 * 128 + id;
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] += j < w.count ? from[j * 128] : 0.0f;
                        }
                    }
                    named_barrier(1 + set, 128);                  // what was here has been read
#pragma unroll
                    for (int j = 0; j < 32; ++j) turn[j * 128 + id] = from_float<T>(v[j]);
                    named_barrier(1 + set, 128);
                    uint4 q[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        q[j] = *reinterpret_cast<const uint4*>(turn + (j * 8 + quarter * 2 + (lane >> 4)) * 128 + 8 * (lane & 15));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int row = __shfl_sync(0xffffffffu, mine, j * 8 + quarter * 2 + (lane >> 4));
                        T* const to = out + row * stride + feature;
                        if (row < 0) continue;
                        if (p.wide_store) {
                            if (live > 0) *reinterpret_cast<uint4*>(to) = q[j];
                        } else {
                            const T* const each = reinterpret_cast<const T*>(&q[j]);
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                if (i < live) to[i] = each[i];
                        }
                    }
                }
                fence_before_sync();
                __syncwarp();
                if (lane == 0) accumulator_read(acc);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
        }
    } else {
        if constexpr (kWeights) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp < S::kCopyWarps) {
            // ---------------------------------------------------------------- copies
            int at = 0;
            uint32_t phase = 0;
            bool alive = true;
            auto advance = [&] {
                if (++at == S::kStages) {
                    at = 0;
                    phase ^= 1;
                }
            };
            // The row numbers of this warp's gathers, in shared memory: read four at a time at an address the whole warp shares,
            // they get to the gather on the short way (with shuffles 47 cycles a gather, lanes that issue their own 62).
            int4* const rows = reinterpret_cast<int4*>(smem + S::kRows0 + warp * 512);
            int* const my_rows = reinterpret_cast<int*>(rows) + 2 * lane;
            auto row_or_zeros = [&](int entry, int end) {
                const int row = row_at(p, entry, end);
                return row < 0 ? p.a.rows : row;               // TMA fills what is past the last row with zeros
            };
            // weight gradient: the tile and block whose row numbers come next
            Walk ahead = w;
            int ahead_tile = t_first, ahead_block = -1, next0 = p.a.rows, next1 = p.a.rows, buffer = 0;
            auto look_ahead = [&] {
                ++ahead_block;
                while (ahead_tile < t_end && ahead_block * kDepth >= ahead.count) {
                    ahead_block = 0;
                    if (++ahead_tile < t_end) ahead.step(1);
                }
                if (ahead_tile >= t_end) return;
                const int end = ahead.first + ahead.count;
                next0 = row_or_zeros(ahead.first + ahead_block * kDepth + 2 * lane, end);
                next1 = row_or_zeros(ahead.first + ahead_block * kDepth + 2 * lane + 1, end);
            };
            if (kWeights && !SORTED && t_first < t_end) {
                // row numbers are asked for two blocks ahead, and put in place one ahead, across tiles
                ahead.start(t_first);
                look_ahead();
                my_rows[0] = next0;
                my_rows[1] = next1;
                look_ahead();
            }
            for (int t = t_first; alive && t < t_end; t += t_step) {
                if (t == t_first) w.start(t);
                else w.step(t_step);
                const int depth = kWeights ? w.count : depth_of_row, blocks = kWeights ? (depth + kDepth - 1) / kDepth : last_block;
                const int end = w.first + w.count, feature0 = w.feature0 * S::kCtas + rank * 128;
                if constexpr (!kWeights) {
                    if (warp > 0) {
                        // of a pair's MMA columns the first half are CTA 0's rows
                        const int half = PAIR ? (w.count + 31) / 32 * 16 : TN, mine = min(half, max(0, w.count - rank * half));
                        const int quads = min(S::kQuads, max(0, (mine + 3) / 4 - (warp - 1) * S::kQuads));
                        const int entry = w.first + rank * half + (warp - 1) * S::kRowsPerWarp + 2 * lane;
                        __syncwarp();
                        if (lane < S::kRowsPerWarp / 2) {
                            my_rows[0] = row_or_zeros(entry, end);
                            my_rows[1] = row_or_zeros(entry + 1, end);
                        }
                        __syncwarp();
                        for (int b = first_block; b < blocks; ++b) {
                            alive = mbar_wait(empty(at), phase ^ 1, abort_flag, kSpin);
                            if (!alive) break;
                            const uint32_t dst = stage0 + at * S::kStageBytes + S::kFeatureBytes + (warp - 1) * S::kQuads * 512, bar = copy_bar(at);
                            if (elect_one()) {
                                expect(bar, quads * 512);
#pragma unroll
                                for (int q = 0; q < S::kQuads; ++q) {
                                    const int4 r = rows[q];
                                    if (q < quads) gather(dst + q * 512, &row_map, b * kDepth, r, bar);
                                }
                            }
                            __syncwarp();
                            advance();
                        }
                    } else {
                        for (int b = first_block; b < blocks; ++b) {
                            alive = mbar_wait(empty(at), phase ^ 1, abort_flag, kSpin);
                            if (!alive) break;
                            const uint32_t dst = stage0 + at * S::kStageBytes, bar = copy_bar(at);
                            if (elect_one()) {
                                expect(bar, S::kFeatureBytes);
                                if constexpr (MODE == kLinear) {
                                    box(dst, feature0, b * kDepth, w.g, bar);
                                    box(dst + 8192, feature0 + 64, b * kDepth, w.g, bar);
                                } else {
                                    box(dst, b * kDepth, feature0, w.g, bar);
                                }
                            }
                            __syncwarp();
                            advance();
                        }
                    }
                } else if constexpr (SORTED) {
                    const int from = __ldg(p.first_block + w.g) * kDepth + w.first - w.begin;
                    for (int b = 0; b < blocks; ++b) {
                        alive = mbar_wait(empty(at), phase ^ 1, abort_flag, kSpin);
                        if (!alive) break;
                        const uint32_t dst = stage0 + at * S::kStageBytes, bar = copy_bar(at);
                        if (elect_one()) {
                            expect(bar, S::kStageBytes);
#pragma unroll
                            for (int c = 0; c < 2; ++c) tile(dst + c * 8192, &feature_map, feature0 + c * 64, from + b * kDepth, bar);
#pragma unroll
                            for (int c = 0; c < S::kRows / 64; ++c)
                                tile(dst + S::kFeatureBytes + c * 8192, &row_map, w.row0 + rank * S::kRows + c * 64, from + b * kDepth, bar);
                        }
                        __syncwarp();
                        advance();
                    }
                } else {
                    const CUtensorMap* const map = warp < 2 ? &feature_map : &row_map;
                    const int column = warp < 2 ? feature0 + warp * 64 : w.row0 + rank * S::kRows + (warp - 2) * 64;
                    for (int b = 0; b < blocks; ++b, buffer ^= 64) {
                        my_rows[(buffer ^ 64)] = next0;
                        my_rows[(buffer ^ 64) + 1] = next1;
                        look_ahead();
                        __syncwarp();
                        alive = mbar_wait(empty(at), phase ^ 1, abort_flag, kSpin);
                        if (!alive) break;
                        const uint32_t dst = stage0 + at * S::kStageBytes + warp * 8192, bar = copy_bar(at);
                        const int quads = min(16, (w.count - b * kDepth + 15) / 16 * 4);     // depths past the end, up to a multiple of 16, are zeros
                        const int4* const mine = rows + buffer / 4;
                        if (elect_one()) {
                            expect(bar, quads * 512);
#pragma unroll 4
                            for (int q = 0; q < quads; ++q) {
                                const int4 r = mine[q];
                                gather(dst + q * 512, map, column, r, bar);
                            }
                        }
                        __syncwarp();
                        advance();
                    }
                }
            }
        } else if (warp == kMmaWarp && rank == 0) {
            // ---------------------------------------------------------------- MMAs
            int at = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            auto advance = [&] {
                if (++at == S::kStages) {
                    at = 0;
                    phase ^= 1;
                }
            };
            constexpr uint32_t kType = __is_same(T, __nv_bfloat16) ? 1 : 0;
            constexpr uint32_t kMajor = MODE == kLinear ? 1u << 15 : MODE == kWeightGradient ? 3u << 15 : 0;
            constexpr uint32_t kDesc = (1u << 4) | (kType << 7) | (kType << 10) | kMajor | ((uint32_t)(128 * S::kCtas >> 4) << 24);
            bool alive = true;
            for (int t = t_first; alive && t < t_end; t += t_step) {
                if (t == t_first) w.start(t);
                else w.step(t_step);
                const int depth = kWeights ? w.count : depth_of_row, blocks = kWeights ? (depth + kDepth - 1) / kDepth : last_block;
                constexpr int kUnit = 16 * S::kCtas;
                const int columns = kWeights ? TN : max(kUnit, min(TN, (w.count + kUnit - 1) / kUnit * kUnit));
                const uint32_t idesc = kDesc | ((uint32_t)(columns >> 3) << 17);
                for (int b = kWeights ? 0 : first_block; b < blocks; ++b) {
                    const bool fresh = b == (kWeights ? 0 : first_block) || (kWeights && b % (kChunk / kDepth) == 0);
                    if (fresh) alive = mbar_wait(acc_empty(acc), acc_phase ^ 1, abort_flag, kSpin);
                    alive = alive && mbar_wait(full(at), phase, abort_flag, kSpin);
                    if (!alive) break;
                    fence_after_sync();
                    const uint32_t base = stage0 + at * S::kStageBytes;
                    const uint64_t fd = MODE == kInputGradient ? make_desc(base) : make_desc_mn(base);
                    const uint64_t rd = kWeights ? make_desc_mn(base + S::kFeatureBytes) : make_desc(base + S::kFeatureBytes);
                    const int steps = min(4, (depth - b * kDepth + 15) / 16);
                    const uint32_t d = tmem + acc * TN;
                    if (elect_one()) {
                        for (int k = 0; k < steps; ++k) {
                            constexpr uint64_t kF = MODE == kInputGradient ? 2 : 128, kR = kWeights ? 128 : 2;
                            if constexpr (PAIR) mma_f16_pair(d, fd + k * kF, rd + k * kR, idesc, k > 0 || !fresh);
                            else mma_f16(d, fd + k * kF, rd + k * kR, idesc, k > 0 || !fresh);
                        }
                        const bool last = b == blocks - 1 || (kWeights && (b + 1) % (kChunk / kDepth) == 0);
                        if constexpr (PAIR) {
                            mma_commit_pair(empty(at));
                            if (last) mma_commit_pair(acc_full(acc));
                        } else {
                            mma_commit(empty(at));
                            if (last) mma_commit(acc_full(acc));
                        }
                    }
                    __syncwarp();
                    if (b == blocks - 1 || (kWeights && (b + 1) % (kChunk / kDepth) == 0)) {
                        acc ^= 1;
                        if (acc == 0) acc_phase ^= 1;
                    }
                    advance();
                }
            }
        }
        if (split && t_first < t_end) {
            // (as the warps that join the sums)
            __syncwarp();
            cluster_sync();
            cluster_sync();
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 0) {
        fence_after_sync();
        if (*abort_flag) {
            // a wait ran out: what was requested lands before the CTA gives its memory back
            for (int i = 0; i < 20000; ++i) __nanosleep(1000);
            if (lane == 0 && p.a.status) atomicOr(p.a.status, FMB_STATUS_TENSOR_TIMEOUT);
        }
        __syncwarp();
    }
    // neither CTA of a pair gives up its memory while the other's copies and arrivals may still come
    if constexpr (PAIR) cluster_sync();
    if (warp == 0) {
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(S::kTmem) : "memory");
        else tmem_free(tmem, S::kTmem);
    }
}

typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                           const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                           CUtensorMapFloatOOBfill);

Encode encoder() {
    static Encode found = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &result) != cudaSuccess ||
            result != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return (Encode)fn;
    }();
    return found;
}

template <typename T, int MODE, int TN, bool PAIR, bool SORTED = false>
int launch(const Args& p, const CUtensorMap& features, const CUtensorMap& rows, const CUtensorMap& weights, long long tiles, cudaStream_t stream) {
    using S = Shape<MODE, TN, PAIR, SORTED>;
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_grouped_tc<T, MODE, TN, PAIR, SORTED>, S::kSmem));
    const int ctas = S::kSplits ? p.split : S::kCtas, grid = (int)(p.split > 1 ? tiles : std::min<long long>(tiles, sm_count() / ctas)) * ctas;
    if (ctas > 1) {
        cudaLaunchConfig_t config = {};
        cudaLaunchAttribute cluster;
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = ctas;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
        config.gridDim = dim3(grid);
        config.blockDim = dim3(S::kThreads);
        config.dynamicSmemBytes = S::kSmem;
        config.stream = stream;
        config.attrs = &cluster;
        config.numAttrs = 1;
        FMB_CUDA_CHECK(cudaLaunchKernelEx(&config, k_grouped_tc<T, MODE, TN, PAIR, SORTED>, p, features, rows, weights));
    } else {
        k_grouped_tc<T, MODE, TN, PAIR, SORTED><<<grid, S::kThreads, S::kSmem, stream>>>(p, features, rows, weights);
    }
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

template <typename T, int MODE>
int launch_rows(Args& p, const CUtensorMap& features, const CUtensorMap& rows, cudaStream_t stream) {
    const fmb_grouped_t* a = &p.a;
    const int average = a->rows / a->groups, width = MODE == kLinear ? a->n : a->k;
    // pairs of CTAs where there is a tile of 256 x 256 for each, and the groups fill half of one
    if (average >= 128 && width > 128 && most_units(a, 256) * ((width + 255) / 256) >= 74) {
        p.unit_rows = 256;
        p.feature_tiles = ceil_div(width, 256);
        return launch<T, MODE, 256, true>(p, features, rows, rows, most_units(a, 256) * p.feature_tiles, stream);
    }
    // else the widest tile that still leaves one per SM, but none much wider than the groups are on average
    int tn = 256;
    while (tn > 32 && (tn > std::max(32, 2 * average) || most_units(a, tn) * p.feature_tiles < 148)) tn /= 2;
    p.unit_rows = tn;
    long long tiles = most_units(a, tn) * p.feature_tiles;
    if (tn == 32) {
        // Few rows: as many CTAs as there is room for share the depth of a tile, at least four blocks each, and the first adds up.
        // (8 rows in 8 groups of 2,048 x 1,024, two CTAs a tile: 16.4 us, 18.5 with one; one row, eight: 12.3, 16.4; 30 rows
        // of 4,096 x 4,096 in one group, four: 18.4, 34.8)
        const long long with_rows = std::min<long long>(a->rows, most_units(a, tn)) * p.feature_tiles;
        const int blocks = ((MODE == kLinear ? a->k : a->n) + kDepth - 1) / kDepth;
        for (int split = 2; split <= 8; split *= 2)
            if (with_rows * split <= (split == 2 ? 148 : 128) && blocks >= 4 * split) p.split = split;
        if (p.split > 1) tiles = with_rows;
    }
    if (tn == 256) return launch<T, MODE, 256, false>(p, features, rows, rows, tiles, stream);
    if (tn == 128) return launch<T, MODE, 128, false>(p, features, rows, rows, tiles, stream);
    if (tn == 64) return launch<T, MODE, 64, false>(p, features, rows, rows, tiles, stream);
    return launch<T, MODE, 32, false>(p, features, rows, rows, tiles, stream);
}

bool by_sixteen(const void* base, long long stride) { return ((uintptr_t)base & 15) == 0 && stride % 8 == 0 && stride > 0; }

// What a call does before its products, and where in its scratch (byte offsets; -1: not needed).
struct Plan {
    long long x = -1, y = -1, w = -1, units = -1, first_block = -1, bytes = 0;
    int tn = 0, unit_rows = 1 << 30;             // weight gradient
    bool pair = false, sorted = false;

    long long take(long long size) {
        const long long at = bytes;
        bytes += (size + 255) / 256 * 256;
        return at;
    }
};

Plan plan_of(const fmb_grouped_t* a, Mode mode) {
    Plan p;
    const long long k8 = (a->k + 7) / 8 * 8, n8 = (a->n + 7) / 8 * 8;
    const bool x_fits = by_sixteen(a->x, a->x_stride), y_fits = by_sixteen(a->y, a->y_stride);
    if (mode != kWeightGradient) {
        // the input, and the weights (their strides may be anything where there is one row, or one matrix)
        if (mode == kLinear && !x_fits) p.x = p.take(a->rows * k8 * 2);
        if (mode == kInputGradient && !y_fits) p.y = p.take(a->rows * n8 * 2);
        if (!by_sixteen(a->w, a->k > 1 ? a->w_row_stride : 8) || (a->groups > 1 && (a->w_group_stride % 8 || a->w_group_stride <= 0)))
            p.w = p.take(a->groups * a->k * n8 * 2);
        return p;
    }
    // Units: a group's rows, cut at half an SM's share of the work, so that every SM has some and one long group does not keep the
    // others waiting (208,333 rows of 64 x 512 in 103 groups, the largest of 40,000: 173 us, and 305 uncut). Where the tiles of one
    // group are enough for a quarter of the SMs, a launch for sums costs more than balance gives (16,384 rows of 2,048 x 1,024 in 32
    // groups: 5 us more with it)
    p.tn = a->k > 128 ? 256 : 128;
    const long long row_tiles = (a->k + p.tn - 1) / p.tn, of_group = ((a->n + 127) / 128) * row_tiles;
    const long long unit_rows = std::max<long long>(128, (a->rows * of_group / (2 * 148) + 63) / 64 * 64);
    if (unit_rows < a->rows && (a->groups * of_group < 2 * 148 || of_group < 148 / 4)) p.unit_rows = (int)unit_rows;
    if (p.unit_rows < a->rows) p.units = p.take(unit_slots(a->rows, p.unit_rows) * a->k * a->n * 4);
    p.pair = p.tn == 256 && a->n > 128 && most_units(a, p.unit_rows) * row_tiles * ((a->n + 255) / 256) >= 74;
    // Sorting reads and writes every row once, at the rate of memory; gathering costs a CTA pair 1,000 cycles more per 64 rows of a
    // tile. Against each other per row: 256 (n / 256 + k / 256) x 4 bytes, 1.6e-4 us per 256 columns, and 1.1e-4 us per tile of
    // 256 x 256. In us, sorted and gathered: 16,384 rows of 2,048 x 1,024: 147, 217; 65,536 of 2,048 x 2,048: 626, 1,111; 30,000 of
    // 1,024 x 1,024: 132, 189; 30,000 of 256 x 512: 77, 71; 300,000 of 128 x 128: 132, 89.
    const long long n_tiles = (a->n + 255) / 256, k_tiles = (a->k + 255) / 256;
    p.sorted = !x_fits || !y_fits || 2 * n_tiles * k_tiles > 3 * (n_tiles + k_tiles);
    if (p.sorted) {
        const long long rows = a->rows + 64ll * a->groups;
        p.x = p.take(rows * k8 * 2);
        p.y = p.take(rows * n8 * 2);
        p.first_block = p.take((a->groups + 1) * 4);
    }
    return p;
}

template <typename T>
int weight_gradient(const fmb_grouped_t* a, const Plan& plan, cudaStream_t stream) {
    Args p;
    p.a = *a;
    p.a.scratch = plan.units >= 0 ? (float*)((char*)a->scratch + plan.units) : nullptr;
    p.first_block = nullptr;
    p.wide_store = four_at_a_time(a->w, a->w_row_stride, 4) && a->w_group_stride % 4 == 0 && a->n % 4 == 0;
    p.unit_rows = plan.unit_rows;
    p.row_tiles = ceil_div(a->k, plan.tn);
    p.feature_tiles = ceil_div(a->n, plan.pair ? 256 : 128);
    const long long tiles = most_units(a, plan.unit_rows) * p.feature_tiles * p.row_tiles;
    CUtensorMap features, rows, weights = {};
    // (a store writes whole pieces of 16 bytes: of rows that end within one, it would write zeros over what lies beside them)
    p.by_tma = !a->accumulate && a->n % 4 == 0 && encode_map(&weights, FMB_TYPE_F32, a->w, a->n, a->k, a->groups, a->w_row_stride, a->w_group_stride, 16, 3, 128, false);
    int rc;
    if (plan.sorted) {
        void* const x = (char*)a->scratch + plan.x;
        void* const y = (char*)a->scratch + plan.y;
        int32_t* const first_block = (int32_t*)((char*)a->scratch + plan.first_block);
        rc = sort_rows(a, x, y, first_block, stream);
        if (rc) return rc;
        p.first_block = first_block;
        const int all = a->rows + 64 * a->groups;
        FMB_REQUIRE(encode_map(&features, a->type, y, a->n, all, 1, (a->n + 7) / 8 * 8, 0, 64, 2, 64, true) &&
                        encode_map(&rows, a->type, x, a->k, all, 1, (a->k + 7) / 8 * 8, 0, 64, 2, 64, true),
                    "fmb_grouped_weight_gradient: tensor maps");
        rc = plan.pair        ? launch<T, kWeightGradient, 256, true, true>(p, features, rows, weights, tiles, stream)
             : plan.tn == 256 ? launch<T, kWeightGradient, 256, false, true>(p, features, rows, weights, tiles, stream)
                              : launch<T, kWeightGradient, 128, false, true>(p, features, rows, weights, tiles, stream);
    } else {
        FMB_REQUIRE(encode_map(&features, a->type, a->y, a->n, a->rows, 1, a->y_stride, 0, 1, 2, 64, true) &&
                        encode_map(&rows, a->type, a->x, a->k, a->rows, 1, a->x_stride, 0, 1, 2, 64, true),
                    "fmb_grouped_weight_gradient: tensor maps");
        rc = plan.pair        ? launch<T, kWeightGradient, 256, true>(p, features, rows, weights, tiles, stream)
             : plan.tn == 256 ? launch<T, kWeightGradient, 256, false>(p, features, rows, weights, tiles, stream)
                              : launch<T, kWeightGradient, 128, false>(p, features, rows, weights, tiles, stream);
    }
    return rc || plan.units < 0 ? rc : sum_units(&p.a, plan.unit_rows, stream);
}

template <typename T>
int linear(const fmb_grouped_t* a, bool forward, const Plan& plan, cudaStream_t stream) {
    Args p;
    p.a = *a;
    p.first_block = nullptr;
    p.row_tiles = 1;
    const int width = forward ? a->n : a->k, depth = forward ? a->k : a->n;
    const void* const out = forward ? a->y : a->x;
    const void* in = forward ? a->x : a->y;
    const void* w = a->w;
    long long in_stride = forward ? a->x_stride : a->y_stride, w_row = a->w_row_stride, w_group = a->w_group_stride;
    p.feature_tiles = ceil_div(width, 128);
    p.wide_store = ((uintptr_t)out & 15) == 0 && (forward ? a->y_stride : a->x_stride) % 8 == 0 && width % 8 == 0;
    const long long packed = forward ? plan.x : plan.y;
    void* const packed_rows = packed >= 0 ? (char*)a->scratch + packed : nullptr;
    void* const packed_weights = plan.w >= 0 ? (char*)a->scratch + plan.w : nullptr;
    if (packed_rows || packed_weights) {
        const int rc = pack(a, in, in_stride, depth, packed_rows, packed_weights, stream);
        if (rc) return rc;
    }
    if (packed_rows) {
        in = packed_rows;
        in_stride = (depth + 7) / 8 * 8;
    }
    if (packed_weights) {
        w = packed_weights;
        w_row = (a->n + 7) / 8 * 8;
        w_group = a->k * w_row;
    }
    CUtensorMap features, rows;
    FMB_REQUIRE(encode_map(&features, a->type, w, a->n, a->k, a->groups, w_row, w_group, forward ? 64 : 128, 3, 64, true) &&
                    encode_map(&rows, a->type, in, depth, a->rows, 1, in_stride, 0, 1, 2, 64, true),
                "grouped product: tensor maps");
    return forward ? launch_rows<T, kLinear>(p, features, rows, stream) : launch_rows<T, kInputGradient>(p, features, rows, stream);
}

template <typename T>
int typed(const fmb_grouped_t* a, Mode mode, const Plan& plan, cudaStream_t stream) {
    return mode == kWeightGradient ? weight_gradient<T>(a, plan, stream) : linear<T>(a, mode == kLinear, plan, stream);
}

}  // namespace

bool encode_map(CUtensorMap* map, int type, const void* base, int columns, int rows, int groups, long long row_stride,
                long long group_stride, int box_rows, int dims, int box_columns, bool swizzled) {
    const Encode encode = encoder();
    const int bytes = type == FMB_TYPE_F32 ? 4 : 2, unit = 16 / bytes;           // values in 16 bytes
    if (!encode || ((uintptr_t)base & 15) != 0) return false;
    // (what is never used may have any value at the caller's: the stride of a single row, or of a single group)
    if (rows == 1) row_stride = (columns + unit - 1) / unit * unit;
    if (groups == 1) group_stride = unit;
    if (row_stride <= 0 || row_stride % unit || row_stride >= (1ll << 37)) return false;
    if (dims == 3 && (group_stride <= 0 || group_stride % unit || group_stride >= (1ll << 37))) return false;
    const cuuint64_t size[3] = {(cuuint64_t)columns, (cuuint64_t)rows, (cuuint64_t)groups};
    const cuuint64_t stride[2] = {(cuuint64_t)row_stride * bytes, (cuuint64_t)group_stride * bytes};
    const cuuint32_t box[3] = {(cuuint32_t)box_columns, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    const CUtensorMapDataType kind = type == FMB_TYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : type == FMB_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return encode(map, kind, dims, const_cast<void*>(base), size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

long long tma_scratch_bytes(const fmb_grouped_t* a, Mode mode) { return plan_of(a, mode).bytes; }

int tma_launch(const fmb_grouped_t* a, Mode mode, cudaStream_t stream) {
    const Plan plan = plan_of(a, mode);
    FMB_REQUIRE(plan.bytes == 0 || a->scratch, "grouped product: null scratch");
    FMB_REQUIRE(((uintptr_t)a->scratch & 255) == 0, "grouped product: scratch starts at a multiple of 256 bytes");
    return a->type == FMB_TYPE_BF16 ? typed<__nv_bfloat16>(a, mode, plan, stream) : typed<__half>(a, mode, plan, stream);
}

}  // namespace grp
}  // namespace fmb
