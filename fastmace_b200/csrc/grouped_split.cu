// Grouped products whose operands threads bring: fp32 operands, split on the way into three bf16 parts, and 16-bit operands of
// an alignment that TMA does not take. The tiles are those of grouped_tc.cu: D[128 features][64 rows of the output].
//
// fp32: x = hi + mid + lo with eight significant bits each, cut off rather than rounded, is exact, at every size a float
// has (no scales). Of the nine products of two such triples the six largest are taken,
//     hi hi | hi mid + mid hi | hi lo + mid mid + lo hi        (what is left out is below 2^-21 of |x| |w|, 2^-24 on average)
// in three MMAs per 16 of the depth, because the parts of the output rows lie side by side: hi x [hi mid lo], mid x [hi mid],
// lo x [hi] with accumulators [hh | .. | ..] of 64 columns. The tensor core cuts its accumulator off at every instruction, so
// hi hi has columns of its own -- the others are 2^-8 of it -- and accumulators move to fp32 registers every kChunk of the
// depth. Against tf32 pairs: the same tensor time (six at twice the rate against three), a seventh of the error, and transposed
// operands, which tf32 does not have in this swizzle.
//
// RESIDENT: depth up to 128, the linears of a model of 128 channels. The split weights stay in shared memory while a CTA goes
// through the rows of one group; else they are split again for each tile.
//
// Two groups of eight warps bring blocks of 64 of the depth in turn, one's loads under way while the other splits.

#include "grouped_tc.cuh"

#include <algorithm>

namespace fmb {
namespace grp {

namespace {

using namespace tc;

constexpr int kTN = 64;
constexpr int kGroupWarps = 8, kLoaderWarps = 2 * kGroupWarps, kEpilogueWarps = 4;
constexpr int kMmaWarp = kLoaderWarps + kEpilogueWarps;
constexpr int kThreads = 32 * (kMmaWarp + 1);

template <typename T, bool RESIDENT> struct Shape {
    static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
    static constexpr int kFeaturePart = 128 * kDepth * 2, kRowPart = kTN * kDepth * 2;
    static constexpr int kFeatureBytes = kParts * kFeaturePart, kRowBytes = kParts * kRowPart;
    static constexpr int kStageBytes = kRowBytes + (RESIDENT ? 0 : kFeatureBytes);
    static constexpr int kStages = RESIDENT ? 4 : 3;
    static constexpr int kResidentBytes = RESIDENT ? 2 * kFeatureBytes : 0;
    static constexpr int kUnits = kResidentBytes + kStages * kStageBytes;          // where the units' table starts
    static constexpr int kSmem = 1024 + kUnits + (FMB_MAX_GROUPS + 1) * 4 + 256;
    static constexpr int kChunk = sizeof(T) == 4 ? 256 : 512;
    static constexpr int kColumns = kParts * kTN;                                  // of an accumulator
    static constexpr int kTmem = kParts == 3 ? 512 : 128;
};

// The features' side of a block: `count` quads per thread from thread `i` of `step` threads on.
// LINEAR: W[g] rows are the depth. INPUT GRADIENT: W[g] rows are the features. WEIGHT GRADIENT: rows of y, by number.
template <typename T, int MODE, int N, int THREADS, typename RowOf>
__device__ __forceinline__ void load_features(const SplitArgs& p, const Walk& w, int d0, int depth, int i, RowOf row_of, Quad<T> (&q)[N]) {
    const int width = MODE == kInputGradient ? p.a.k : p.a.n;
    const T* const weights = (const T*)p.a.w + (MODE == kWeightGradient ? 0 : w.g * p.a.w_group_stride);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int at = i + j * THREADS;
        if constexpr (MODE == kInputGradient) {
            const int f = w.feature0 + (at >> 4), d = d0 + 4 * (at & 15);
            q[j] = load_quad(weights + (long long)f * p.a.w_row_stride + d, f < width ? depth - d : 0, p.wide_features);
        } else if constexpr (MODE == kLinear) {
            const int d = d0 + (at >> 5), f = w.feature0 + 4 * (at & 31);
            q[j] = load_quad(weights + (long long)d * p.a.w_row_stride + f, d < depth ? width - f : 0, p.wide_features);
        } else {
            const int row = row_of(at >> 5), f = w.feature0 + 4 * (at & 31);
            q[j] = load_quad((const T*)p.a.y + (long long)row * p.a.y_stride + f, row >= 0 ? width - f : 0, p.wide_features);
        }
    }
}

template <typename T, int MODE, int N, int THREADS>
__device__ __forceinline__ void store_features(uint8_t* tile, int i, const Quad<T> (&q)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int at = i + j * THREADS;
        if constexpr (MODE == kInputGradient) store_quad<T, 128 * kDepth * 2>(tile, quad_offset(at >> 4, at & 15), q[j]);
        else store_quad<T, 128 * kDepth * 2>(tile, (uint32_t)((at >> 4) & 1) * 8192 + quad_offset(at >> 5, at & 15), q[j]);
    }
}

template <typename T, int MODE, bool RESIDENT>
__global__ void __launch_bounds__(kThreads, 1)
k_grouped_split(const __grid_constant__ SplitArgs p) {
    using S = Shape<T, RESIDENT>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    int* const first_unit = reinterpret_cast<int*>(smem + S::kUnits);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + S::kUnits + ((FMB_MAX_GROUPS + 1) * 4 + 7) / 8 * 8);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S::kStages + 6);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (S::kStages + s); };
    auto acc_full = [&](int b) { return bar0 + 8u * (2 * S::kStages + b); };
    auto acc_empty = [&](int b) { return bar0 + 8u * (2 * S::kStages + 2 + b); };
    const uint32_t w_full = bar0 + 8u * (2 * S::kStages + 4), w_empty = w_full + 8;
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    constexpr bool kWeights = MODE == kWeightGradient;

    if (warp == 0) tmem_alloc(smem_u32(tmem_slot), S::kTmem);
    if (warp == kMmaWarp && elect_one()) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(full(s), kGroupWarps);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), kEpilogueWarps);
        }
        mbar_init(w_full, kLoaderWarps);
        mbar_init(w_empty, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    count_units<kThreads>(p.a.offsets, p.a.groups, p.a.rows, p.unit_rows, kWeights ? 1 : 0, first_unit);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const long long tiles = (long long)units_in_all(first_unit, p.a.groups, p.a.rows, p.unit_rows) * p.feature_tiles * p.row_tiles;
    const int t_begin = (int)(tiles * blockIdx.x / gridDim.x), t_end = (int)(tiles * (blockIdx.x + 1) / gridDim.x);
    const int depth_of_row = MODE == kLinear ? p.a.k : p.a.n;
    const T* const row_source = (const T*)(MODE == kInputGradient ? p.a.y : p.a.x);
    const long long row_stride = MODE == kInputGradient ? p.a.y_stride : p.a.x_stride;

    Walk w(p.a, first_unit, p.unit_rows, p.feature_tiles, p.row_tiles, kTN);

    if (warp < kLoaderWarps) {
        // ---------------------------------------------------------------- loaders
        const int group = warp / kGroupWarps, gw = warp % kGroupWarps, i = gw * 32 + lane;
        constexpr int kFeatureQuads = 128 * kDepth / 4 / 256, kRowQuads = kTN * kDepth / 4 / 256;      // per thread of a group
        int block = 0, at = 0, held_g = -1, held_f = -1;
        uint32_t phase = 0, w_phase = 0;
        bool alive = true;
        for (int t = t_begin; alive && t < t_end; ++t) {
            if (t == t_begin) w.start(t);
            else w.step(1);
            const int depth = kWeights ? w.count : depth_of_row, blocks = (depth + kDepth - 1) / kDepth;
            const int end = w.first + w.count;
            if constexpr (RESIDENT) {
                if (w.g != held_g || w.feature0 != held_f) {
                    held_g = w.g;
                    held_f = w.feature0;
                    alive = mbar_wait(w_empty, w_phase ^ 1, abort_flag, kSpin);
                    w_phase ^= 1;
                    if (!alive) break;
#pragma unroll 1
                    for (int b = 0; b < blocks; ++b) {
                        Quad<T> q[kFeatureQuads / 2];
                        load_features<T, MODE, kFeatureQuads / 2, 512>(p, w, b * kDepth, depth, warp * 32 + lane, [](int) { return 0; }, q);
                        store_features<T, MODE, kFeatureQuads / 2, 512>(smem + b * S::kFeatureBytes, warp * 32 + lane, q);
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(w_full);
                }
            }
            // row numbers of the tile's 64 output rows, or of a block's 64 depths: lane l holds the l-th and the 32 + l-th
            int low = row_at(p, w.first + lane, end), high = row_at(p, w.first + 32 + lane, end);
            for (int b = 0; b < blocks; ++b, ++block) {
                const int s = at;
                const uint32_t ph = phase;
                if (++at == S::kStages) {
                    at = 0;
                    phase ^= 1;
                }
                const int d0 = b * kDepth;
                if ((block & 1) == group) {
                    auto row_of = [&](int r) {
                        const int a = __shfl_sync(0xffffffffu, low, r & 31), c = __shfl_sync(0xffffffffu, high, r & 31);
                        return r < 32 ? a : c;
                    };
                    if (kWeights && b > 0) {
                        low = row_at(p, w.first + d0 + lane, end);
                        high = row_at(p, w.first + d0 + 32 + lane, end);
                    }
                    Quad<T> fq[RESIDENT ? 1 : kFeatureQuads], rq[kRowQuads];
#pragma unroll
                    for (int j = 0; j < kRowQuads; ++j) {
                        const int n = i + j * 256, row = row_of(n >> 4), q4 = 4 * (n & 15);
                        if constexpr (kWeights)
                            rq[j] = load_quad(row_source + (long long)row * row_stride + w.row0 + q4, row >= 0 ? p.a.k - w.row0 - q4 : 0, p.wide_rows);
                        else
                            rq[j] = load_quad(row_source + (long long)row * row_stride + d0 + q4, row >= 0 ? depth - d0 - q4 : 0, p.wide_rows);
                    }
                    if constexpr (!RESIDENT) load_features<T, MODE, kFeatureQuads, 256>(p, w, d0, depth, i, row_of, fq);
                    alive = mbar_wait(empty(s), ph ^ 1, abort_flag, kSpin);
                    if (!alive) break;
                    uint8_t* const stage = smem + S::kResidentBytes + s * S::kStageBytes;
#pragma unroll
                    for (int j = 0; j < kRowQuads; ++j) {
                        const int n = i + j * 256;
                        store_quad<T, S::kRowPart>(stage, quad_offset(n >> 4, n & 15), rq[j]);
                    }
                    if constexpr (!RESIDENT) store_features<T, MODE, kFeatureQuads, 256>(stage + S::kRowBytes, i, fq);
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full(s));
                }
            }
        }
    } else if (warp == kMmaWarp) {
        // ---------------------------------------------------------------- MMAs
        int at = 0, acc = 0, held_g = -1, held_f = -1;
        uint32_t phase = 0, acc_phase = 0, w_phase = 0;
        constexpr uint32_t kType = __is_same(T, __half) ? 0 : 1;
        constexpr uint32_t kMajor = MODE == kLinear ? 1u << 15 : MODE == kWeightGradient ? 3u << 15 : 0;
        constexpr uint32_t kDesc = (1u << 4) | (kType << 7) | (kType << 10) | kMajor | ((uint32_t)(128 >> 4) << 24);
        constexpr int kChunkBlocks = S::kChunk / kDepth;
        bool alive = true;
        for (int t = t_begin; alive && t < t_end; ++t) {
            if (t == t_begin) w.start(t);
            else w.step(1);
            const int depth = kWeights ? w.count : depth_of_row, blocks = (depth + kDepth - 1) / kDepth;
            bool release = false;
            if constexpr (RESIDENT) {
                if (w.g != held_g || w.feature0 != held_f) {
                    held_g = w.g;
                    held_f = w.feature0;
                    alive = mbar_wait(w_full, w_phase, abort_flag, kSpin);
                    w_phase ^= 1;
                    if (!alive) break;
                }
                if (t + 1 < t_end) {
                    Walk next = w;
                    next.step(1);
                    release = next.g != held_g || next.feature0 != held_f;
                }
            }
            for (int b = 0; b < blocks; ++b) {
                const bool fresh = b % kChunkBlocks == 0, last = b == blocks - 1 || (b + 1) % kChunkBlocks == 0;
                if (fresh) alive = mbar_wait(acc_empty(acc), acc_phase ^ 1, abort_flag, kSpin);
                alive = alive && mbar_wait(full(at), phase, abort_flag, kSpin);
                if (!alive) break;
                fence_after_sync();
                const uint32_t stage = smem_u32(smem) + S::kResidentBytes + at * S::kStageBytes;
                const uint32_t features = RESIDENT ? smem_u32(smem) + b * S::kFeatureBytes : stage + S::kRowBytes;
                const uint64_t fd = MODE == kInputGradient ? make_desc(features) : make_desc_mn(features);
                const uint64_t rd = kWeights ? make_desc_mn(stage) : make_desc(stage);
                constexpr uint64_t kF = MODE == kInputGradient ? 2 : 128, kR = kWeights ? 128 : 2;
                const int steps = min(4, (depth - b * kDepth + 15) / 16);
                const uint32_t d = tmem + acc * (S::kTmem / 2);
                if (elect_one()) {
                    for (int k = 0; k < steps; ++k) {
                        const uint32_t go = k > 0 || !fresh;
                        constexpr uint32_t n1 = (uint32_t)(kTN >> 3) << 17;
                        const uint64_t f = fd + k * kF, r = rd + k * kR;
                        if constexpr (S::kParts == 3) {
                            constexpr uint64_t kPart = S::kFeaturePart >> 4;
                            mma_f16(d, f, r, kDesc | 3 * n1, go);
                            mma_f16(d + kTN, f + kPart, r, kDesc | 2 * n1, 1);
                            mma_f16(d + 2 * kTN, f + 2 * kPart, r, kDesc | n1, 1);
                        } else {
                            mma_f16(d, f, r, kDesc | n1, go);
                        }
                    }
                    mma_commit(empty(at));
                    if (last) mma_commit(acc_full(acc));
                    if (release && b == blocks - 1) mma_commit(w_empty);
                }
                __syncwarp();
                if (last) {
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1;
                }
                if (++at == S::kStages) {
                    at = 0;
                    phase ^= 1;
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        const int quarter = warp & 3;
        int acc = 0;
        uint32_t acc_phase = 0;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const int width = MODE == kInputGradient ? p.a.k : p.a.n;
        T* const out = (T*)(MODE == kLinear ? p.a.y : p.a.x);
        const long long out_stride = MODE == kLinear ? p.a.y_stride : p.a.x_stride;
        if (!kWeights && p.a.zero_rest) {
            const int from = min(max(p.a.offsets[p.a.groups], 0), p.a.rows);
            for (int e = from + blockIdx.x * kEpilogueWarps + quarter; e < p.a.rows; e += gridDim.x * kEpilogueWarps) {
                const int row = row_at(p, e, p.a.rows);
                if (row >= 0)
                    for (int c = lane; c < width; c += 32) out[row * out_stride + c] = from_float<T>(0.0f);
            }
        }
        bool alive = true;
        for (int t = t_begin; alive && t < t_end; ++t) {
            if (t == t_begin) w.start(t);
            else w.step(1);
            const int feature = w.feature0 + quarter * 32 + lane;
            const int depth = kWeights ? w.count : depth_of_row, chunks = (depth + S::kChunk - 1) / S::kChunk;
            float sum[kTN];
#pragma unroll
            for (int j = 0; j < kTN; ++j) sum[j] = 0.0f;
            for (int c = 0; c < chunks; ++c) {
                alive = mbar_wait(acc_full(acc), acc_phase, abort_flag, kSpin);
                if (!alive) break;
                fence_after_sync();
                const uint32_t d = tmem + lanes + acc * (S::kTmem / 2);
#pragma unroll
                for (int j0 = 0; j0 < kTN; j0 += 16) {
                    float v[16];
                    if constexpr (S::kParts == 3) {
                        float u[16];
                        tmem_load_16x2(d + kTN + j0, d + 2 * kTN + j0, v, u);
#pragma unroll
                        for (int j = 0; j < 16; ++j) u[j] += v[j];
                        tmem_load_16(d + j0, v);
#pragma unroll
                        for (int j = 0; j < 16; ++j) sum[j0 + j] += v[j] + u[j];
                    } else {
                        tmem_load_16(d + j0, v);
#pragma unroll
                        for (int j = 0; j < 16; ++j) sum[j0 + j] += v[j];
                    }
                }
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty(acc));
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
            if (!alive) break;
            if constexpr (kWeights) {
                const bool direct = w.units <= 1;
                const long long stride = direct ? p.a.w_row_stride : p.a.n;
                float* const to = (direct ? (float*)p.a.w + w.g * p.a.w_group_stride : p.a.scratch + (long long)w.unit * p.a.k * p.a.n) + feature;
                if (feature < p.a.n) {
#pragma unroll
                    for (int j = 0; j < kTN; ++j) {
                        if (w.row0 + j >= p.a.k) break;
                        float* const one = to + (w.row0 + j) * stride;
                        *one = direct && p.a.accumulate ? *one + sum[j] : sum[j];
                    }
                }
            } else {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int row = row_at(p, w.first + half * 32 + lane, w.first + w.count);
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const int r = __shfl_sync(0xffffffffu, row, j);
                        if (r >= 0 && feature < width) out[r * out_stride + feature] = from_float<T>(sum[half * 32 + j]);
                    }
                }
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 0) {
        fence_after_sync();
        if (*abort_flag) {
            // a wait ran out: MMAs under way end before the CTA gives its memory back
            for (int n = 0; n < 20000; ++n) __nanosleep(1000);
            if (lane == 0 && p.a.status) atomicOr(p.a.status, FMB_STATUS_TENSOR_TIMEOUT);
        }
        __syncwarp();
        tmem_free(tmem, S::kTmem);
    }
}

template <typename T, int MODE, bool RESIDENT>
int launch(const SplitArgs& p, long long tiles, cudaStream_t stream) {
    using S = Shape<T, RESIDENT>;
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_grouped_split<T, MODE, RESIDENT>, S::kSmem));
    k_grouped_split<T, MODE, RESIDENT><<<(int)std::min<long long>(tiles, sm_count()), kThreads, S::kSmem, stream>>>(p);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

template <typename T>
int typed(const fmb_grouped_t* a, Mode mode, cudaStream_t stream) {
    SplitArgs p;
    p.a = *a;
    const int bytes = (int)sizeof(T);
    const bool x_wide = four_at_a_time(a->x, a->x_stride, bytes), y_wide = four_at_a_time(a->y, a->y_stride, bytes);
    if (mode == kWeightGradient) {
        p.feature_tiles = ceil_div(a->n, 128);
        p.row_tiles = ceil_div(a->k, kTN);
        p.unit_rows = split_unit_rows(a);
        p.wide_features = y_wide;
        p.wide_rows = x_wide;
        FMB_REQUIRE(p.unit_rows >= a->rows || a->scratch, "fmb_grouped_weight_gradient: null scratch");
        const int rc = launch<T, kWeightGradient, false>(p, most_units(a, p.unit_rows) * p.feature_tiles * p.row_tiles, stream);
        return rc || p.unit_rows >= a->rows ? rc : sum_units(a, p.unit_rows, stream);
    }
    const bool forward = mode == kLinear;
    p.feature_tiles = ceil_div(forward ? a->n : a->k, 128);
    p.row_tiles = 1;
    p.unit_rows = kTN;
    p.wide_features = four_at_a_time(a->w, a->w_row_stride, bytes) && a->w_group_stride % 4 == 0;
    p.wide_rows = forward ? x_wide : y_wide;
    const long long tiles = most_units(a, p.unit_rows) * p.feature_tiles;
    const bool resident = (forward ? a->k : a->n) <= 2 * kDepth;
    if (forward) return resident ? launch<T, kLinear, true>(p, tiles, stream) : launch<T, kLinear, false>(p, tiles, stream);
    return resident ? launch<T, kInputGradient, true>(p, tiles, stream) : launch<T, kInputGradient, false>(p, tiles, stream);
}

}  // namespace

// rows per unit of the weight gradient: all of a group's, or fewer where there are few tiles
int split_unit_rows(const fmb_grouped_t* a) {
    const long long tiles = (long long)a->groups * ((a->n + 127) / 128) * ((a->k + kTN - 1) / kTN);
    if (tiles >= 2 * 148 || a->rows <= 128) return 1 << 30;
    const long long wanted = (2 * 148 + tiles - 1) / tiles * a->groups;          // units in all
    const int unit_rows = (int)std::max<long long>(128, (a->rows / wanted + 63) / 64 * 64);
    return unit_rows < a->rows ? unit_rows : 1 << 30;
}

int split_launch(const fmb_grouped_t* a, Mode mode, cudaStream_t stream) { return typed<float>(a, mode, stream); }

}  // namespace grp
}  // namespace fmb
