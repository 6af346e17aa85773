// Grouped linear and its input gradient in fp32 for any depth and alignment: threads bring the operands and split them on the way
// into three bf16 parts. The tiles are those of grouped_tc.cu: D[128 features][64 rows of the output].
//
// x = hi + mid + lo with eight significant bits each, cut off rather than rounded, is exact, at every size a float has (no
// scales). Of the nine products of two such triples the six largest are taken,
//     hi hi | hi mid + mid hi | hi lo + mid mid + lo hi        (what is left out is below 2^-21 of |x| |w|, 2^-24 on average)
// in three MMAs per 16 of the depth, because the parts of the output rows lie side by side: hi x [hi mid lo], mid x [hi mid],
// lo x [hi] with accumulators [hh | .. | ..] of 64 columns. The tensor core cuts its accumulator off at every instruction, so
// hi hi has columns of its own -- the others are 2^-8 of it -- and accumulators move to fp32 registers every kChunk of the
// depth. Against tf32 pairs: the same tensor time (six at twice the rate against three), a seventh of the error, and transposed
// operands, which tf32 does not have in this swizzle.
//
// Two groups of eight warps bring blocks of 64 of the depth in turn, one's loads under way while the other splits. Bound by that: the
// tensor cores are busy a fifth of the time.

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
constexpr int kFeaturePart = 128 * kDepth * 2, kRowPart = kTN * kDepth * 2;
constexpr int kFeatureBytes = 3 * kFeaturePart, kRowBytes = 3 * kRowPart, kStageBytes = kFeatureBytes + kRowBytes, kStages = 2;
constexpr int kTurnBytes = 32 * 128 * 4;                       // results on their way out: 32 rows of 128 features
constexpr int kTurn0 = kStages * kStageBytes, kUnits0 = kTurn0 + kTurnBytes;
constexpr int kSmem = 1024 + kUnits0 + (FMB_MAX_GROUPS + 1) * 4 + 256;
constexpr int kChunk = 256, kChunkBlocks = kChunk / kDepth;
constexpr int kFeatureQuads = 128 * kDepth / 4 / 256, kRowQuads = kTN * kDepth / 4 / 256;      // per thread of a group
static_assert(kSmem <= 227 * 1024, "fits an SM");

// the features' side of a block: rows of W[g] are the depth (linear) or the features (input gradient)
template <int MODE>
__device__ __forceinline__ void load_features(const SplitArgs& p, const Walk& w, int d0, int depth, int i, Quad<float> (&q)[kFeatureQuads]) {
    const int width = MODE == kInputGradient ? p.a.k : p.a.n;
    const float* const weights = (const float*)p.a.w + w.g * p.a.w_group_stride;
#pragma unroll
    for (int j = 0; j < kFeatureQuads; ++j) {
        const int at = i + j * 256;
        if constexpr (MODE == kInputGradient) {
            const int f = w.feature0 + (at >> 4), d = d0 + 4 * (at & 15);
            q[j] = load_quad(weights + (long long)f * p.a.w_row_stride + d, f < width ? depth - d : 0, p.wide_features);
        } else {
            const int d = d0 + (at >> 5), f = w.feature0 + 4 * (at & 31);
            q[j] = load_quad(weights + (long long)d * p.a.w_row_stride + f, d < depth ? width - f : 0, p.wide_features);
        }
    }
}

template <int MODE>
__device__ __forceinline__ void store_features(uint8_t* tile, int i, const Quad<float> (&q)[kFeatureQuads]) {
#pragma unroll
    for (int j = 0; j < kFeatureQuads; ++j) {
        const int at = i + j * 256;
        if constexpr (MODE == kInputGradient) store_quad<float, kFeaturePart>(tile, quad_offset(at >> 4, at & 15), q[j]);
        else store_quad<float, kFeaturePart>(tile, (uint32_t)((at >> 4) & 1) * 8192 + quad_offset(at >> 5, at & 15), q[j]);
    }
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
k_grouped_split(const __grid_constant__ SplitArgs p, int wide_out) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    int* const first_unit = reinterpret_cast<int*>(smem + kUnits0);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + kUnits0 + ((FMB_MAX_GROUPS + 1) * 4 + 7) / 8 * 8);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 4);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
    auto acc_full = [&](int b) { return bar0 + 8u * (2 * kStages + b); };
    auto acc_empty = [&](int b) { return bar0 + 8u * (2 * kStages + 2 + b); };
    const int warp = uniform_warp(), lane = threadIdx.x & 31;

    if (warp == 0) tmem_alloc(smem_u32(tmem_slot), 512);
    if (warp == kMmaWarp && elect_one()) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full(s), kGroupWarps);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), kEpilogueWarps);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    count_units<kThreads>(p.a.offsets, p.a.groups, p.a.rows, kTN, 0, first_unit);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const long long tiles = (long long)units_in_all(first_unit, p.a.groups, p.a.rows, kTN) * p.feature_tiles;
    const int t_begin = (int)(tiles * blockIdx.x / gridDim.x), t_end = (int)(tiles * (blockIdx.x + 1) / gridDim.x);
    const int depth = MODE == kLinear ? p.a.k : p.a.n, blocks = (depth + kDepth - 1) / kDepth;
    Walk w(p.a, first_unit, kTN, p.feature_tiles, 1, kTN);
    bool alive = true;

    if (warp < kLoaderWarps) {
        // ---------------------------------------------------------------- loaders
        const float* const in = (const float*)(MODE == kLinear ? p.a.x : p.a.y);
        const long long stride = MODE == kLinear ? p.a.x_stride : p.a.y_stride;
        const int group = warp / kGroupWarps, i = threadIdx.x & 255;
        int block = 0, at = 0;
        uint32_t phase = 0;
        for (int t = t_begin; alive && t < t_end; ++t) {
            if (t == t_begin) w.start(t);
            else w.step(1);
            // this thread's rows of the output
            const float* from[kRowQuads];
            bool there[kRowQuads];
#pragma unroll
            for (int j = 0; j < kRowQuads; ++j) {
                const int row = row_at(p, w.first + ((i + j * 256) >> 4), w.first + w.count);
                there[j] = row >= 0;
                from[j] = in + (row >= 0 ? row : 0) * stride + 4 * (i & 15);
            }
            for (int b = 0; b < blocks; ++b, ++block) {
                const int s = at;
                const uint32_t ph = phase;
                if (++at == kStages) {
                    at = 0;
                    phase ^= 1;
                }
                if ((block & 1) != group) continue;
                const int d0 = b * kDepth;
                Quad<float> fq[kFeatureQuads], rq[kRowQuads];
#pragma unroll
                for (int j = 0; j < kRowQuads; ++j) rq[j] = load_quad(from[j] + d0, there[j] ? depth - d0 - 4 * (i & 15) : 0, p.wide_rows);
                load_features<MODE>(p, w, d0, depth, i, fq);
                alive = mbar_wait(empty(s), ph ^ 1, abort_flag, kSpin);
                if (!alive) break;
                uint8_t* const stage = smem + s * kStageBytes;
#pragma unroll
                for (int j = 0; j < kRowQuads; ++j) store_quad<float, kRowPart>(stage, quad_offset((i + j * 256) >> 4, i & 15), rq[j]);
                store_features<MODE>(stage + kRowBytes, i, fq);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full(s));
            }
        }
    } else if (warp == kMmaWarp) {
        // ---------------------------------------------------------------- MMAs
        int at = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        constexpr uint32_t kMajor = MODE == kLinear ? 1u << 15 : 0;
        constexpr uint32_t kDesc = (1u << 4) | (1u << 7) | (1u << 10) | kMajor | ((uint32_t)(128 >> 4) << 24), k64 = (uint32_t)(kTN >> 3) << 17;
        for (int t = t_begin; alive && t < t_end; ++t) {
            for (int b = 0; b < blocks; ++b) {
                const bool fresh = b % kChunkBlocks == 0, last = b == blocks - 1 || (b + 1) % kChunkBlocks == 0;
                if (fresh) alive = mbar_wait(acc_empty(acc), acc_phase ^ 1, abort_flag, kSpin);
                alive = alive && mbar_wait(full(at), phase, abort_flag, kSpin);
                if (!alive) break;
                fence_after_sync();
                const uint32_t stage = smem_u32(smem) + at * kStageBytes, features = stage + kRowBytes;
                const uint64_t fd = MODE == kInputGradient ? make_desc(features) : make_desc_mn(features), rd = make_desc(stage);
                constexpr uint64_t kF = MODE == kInputGradient ? 2 : 128, kNext = kFeaturePart >> 4;
                const int steps = min(4, (depth - b * kDepth + 15) / 16);
                const uint32_t d = tmem + acc * 256;
                if (elect_one()) {
                    for (int k = 0; k < steps; ++k) {
                        const uint64_t f = fd + k * kF, r = rd + k * 2;
                        mma_f16(d, f, r, kDesc | 3 * k64, k > 0 || !fresh);
                        mma_f16(d + kTN, f + kNext, r, kDesc | 2 * k64, 1);
                        mma_f16(d + 2 * kTN, f + 2 * kNext, r, kDesc | k64, 1);
                    }
                    mma_commit(empty(at));
                    if (last) mma_commit(acc_full(acc));
                }
                __syncwarp();
                if (last) {
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1;
                }
                if (++at == kStages) {
                    at = 0;
                    phase ^= 1;
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- results
        const int quarter = warp & 3, id = quarter * 32 + lane;
        int acc = 0;
        uint32_t acc_phase = 0;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const int width = MODE == kInputGradient ? p.a.k : p.a.n, chunks = (depth + kChunk - 1) / kChunk;
        float* const out = (float*)(MODE == kLinear ? p.a.y : p.a.x);
        const long long stride = MODE == kLinear ? p.a.y_stride : p.a.x_stride;
        float* const turn = reinterpret_cast<float*>(smem + kTurn0);
        if (p.a.zero_rest) {
            const int from = min(max(p.a.offsets[p.a.groups], 0), p.a.rows);
            for (int e = from + blockIdx.x * kEpilogueWarps + quarter; e < p.a.rows; e += gridDim.x * kEpilogueWarps) {
                const int row = row_at(p, e, p.a.rows);
                if (row >= 0)
                    for (int c = lane; c < width; c += 32) out[row * stride + c] = 0.0f;
            }
        }
        // (a wait that runs out does not end the loop: the warps meet at barriers, and all have to come)
        for (int t = t_begin; t < t_end; ++t) {
            if (t == t_begin) w.start(t);
            else w.step(1);
            const int low = row_at(p, w.first + lane, w.first + w.count), high = row_at(p, w.first + 32 + lane, w.first + w.count);
            float sum[kTN];
#pragma unroll
            for (int j = 0; j < kTN; ++j) sum[j] = 0.0f;
            for (int c = 0; c < chunks; ++c) {
                mbar_wait(acc_full(acc), acc_phase, abort_flag, kSpin);
                fence_after_sync();
                const uint32_t d = tmem + lanes + acc * 256;
#pragma unroll
                for (int j0 = 0; j0 < kTN; j0 += 8) {
                    float v[8], u[8];
                    tmem_load_8(d + kTN + j0, v);
                    tmem_load_8(d + 2 * kTN + j0, u);
#pragma unroll
                    for (int j = 0; j < 8; ++j) u[j] += v[j];
                    tmem_load_8(d + j0, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum[j0 + j] += v[j] + u[j];
                }
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty(acc));
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
            const int live = width - w.feature0 - 4 * lane;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                named_barrier(1, 128);                            // what was here has been read
#pragma unroll
                for (int j = 0; j < 32; ++j) turn[j * 128 + id] = sum[half * 32 + j];
                named_barrier(1, 128);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int row = __shfl_sync(0xffffffffu, half ? high : low, quarter * 8 + j);
                    const float4 q = *reinterpret_cast<const float4*>(turn + (quarter * 8 + j) * 128 + 4 * lane);
                    if (row < 0) continue;
                    float* const to = out + row * stride + w.feature0 + 4 * lane;
                    if (wide_out) {
                        if (live > 0) *reinterpret_cast<float4*>(to) = q;
                    } else {
                        if (live > 0) to[0] = q.x;
                        if (live > 1) to[1] = q.y;
                        if (live > 2) to[2] = q.z;
                        if (live > 3) to[3] = q.w;
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
        tmem_free(tmem, 512);
    }
}

template <int MODE>
int launch(const SplitArgs& p, int wide_out, cudaStream_t stream) {
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_grouped_split<MODE>, kSmem));
    const long long tiles = most_units(&p.a, kTN) * p.feature_tiles;
    k_grouped_split<MODE><<<(int)std::min<long long>(tiles, sm_count()), kThreads, kSmem, stream>>>(p, wide_out);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

}  // namespace

int split_launch(const fmb_grouped_t* a, Mode mode, cudaStream_t stream) {
    const bool forward = mode == kLinear;
    const int width = forward ? a->n : a->k;
    SplitArgs p;
    p.a = *a;
    p.feature_tiles = ceil_div(width, 128);
    p.row_tiles = 1;
    p.unit_rows = kTN;
    p.wide_features = four_at_a_time(a->w, a->w_row_stride, 4) && a->w_group_stride % 4 == 0;
    p.wide_rows = four_at_a_time(forward ? a->x : a->y, forward ? a->x_stride : a->y_stride, 4);
    const int wide_out = width % 4 == 0 && four_at_a_time(forward ? a->y : a->x, forward ? a->y_stride : a->x_stride, 4);
    return forward ? launch<kLinear>(p, wide_out, stream) : launch<kInputGradient>(p, wide_out, stream);
}

}  // namespace grp
}  // namespace fmb
