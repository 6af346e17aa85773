// Grouped linear and its input gradient in fp32 for a depth of up to 128, the linears of a model of 128 channels: the
// split weights of 128 features stay in tensor memory while a CTA goes through the rows of their group.
//
// The numbers and their six products are those of grouped_parts.cu. What bounds the work here is memory, 8 bytes per row and
// channel, so the SM's own paths are kept short of that:
//   * rows come by TMA gather, 4 whole rows an instruction, into a ring of three tiles of 64 rows: 64 KB on their way while
//     one is worked on (threads' own loads, 32 KB and waits in between, brought 2.2 TB/s);
//   * eight warps split a tile into three K-major planes (48 KB, two of them);
//   * the weights, as the MMAs' first operand in TMEM (three planes of 64 columns), take no shared-memory reads: a tile
//     costs 96 KB of reads there instead of 192. Two accumulators, hi hi and the five others, twice (448 columns in all);
//   * the result turns through shared memory, so that a store writes 512 bytes of a row. A lane that stored its own
//     feature row by row took longer than everything else together.
// 884,736 rows of 128 x 128 in 5 groups take 180 us (5.1 TB/s of 910 MB; 141 us at the rate of a copy), 1,944 rows in 2 groups 12.

#include "grouped_tc.cuh"

#include <algorithm>

namespace fmb {
namespace grp {

namespace {

using namespace tc;

constexpr int kTN = 64, kK = 128;                          // rows of a tile, depth
constexpr int kRaw = 3, kRawBytes = kTN * kK * 4;
constexpr int kPlanes = 2, kPlaneTile = kTN * kDepth * 2, kPlaneBytes = 3 * 2 * kPlaneTile;      // [part][half of the depth]
constexpr int kTurnRows = 16, kTurnBytes = kTurnRows * 128 * 4;      // rows of results that turn at a time, one buffer per set
constexpr int kPlane0 = kRaw * kRawBytes, kTurn0 = kPlane0 + kPlanes * kPlaneBytes, kUnits0 = kTurn0 + 2 * kTurnBytes;
constexpr int kSmem = 1024 + kUnits0 + (FMB_MAX_GROUPS + 1) * 4 + 256;
constexpr int kEpilogueWarps = 8, kSplitWarps = 8,           // two sets of four, which take the tiles in turn; eight that split
              kThreads = 32 * (4 + kEpilogueWarps + kSplitWarps);
constexpr uint32_t kAccumulators = 192;                    // TMEM columns before them: the weights
static_assert(kSmem <= 227 * 1024, "fits an SM");

__device__ __forceinline__ void tmem_store_8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// this lane's feature of the tile's weights, split, into the TMEM columns of the three planes (two values a column)
template <int MODE>
__device__ __forceinline__ void bring_weights(const SplitArgs& p, const Walk& w, int feature, int depth, uint32_t tmem) {
    const int width = MODE == kInputGradient ? p.a.k : p.a.n;
    const float* const from = (const float*)p.a.w + w.g * p.a.w_group_stride + (MODE == kInputGradient ? feature * p.a.w_row_stride : feature);
    const bool live = feature < width;
    // 32 values on their way while 32 are split: one round trip to memory in all, where eight of 16 took 5 us of a small call
    auto load = [&](int d0, float (&v)[32]) {
        if constexpr (MODE == kInputGradient) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const float4 q = load_quad(from + d0 + i, live ? depth - d0 - i : 0, p.wide_features);
                v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = live && d0 + i < depth ? __ldg(from + (d0 + i) * p.a.w_row_stride) : 0.0f;
        }
    };
    float next[32];
    load(0, next);
#pragma unroll 1
    for (int d0 = 0; d0 < depth; d0 += 32) {
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = next[i];
        if (d0 + 32 < depth) load(d0 + 32, next);
#pragma unroll
        for (int part = 0; part < 3; ++part) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t two[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) two[i] = upper_halves(v[16 * h + 2 * i], v[16 * h + 2 * i + 1]);
                tmem_store_8(tmem + part * 64 + d0 / 2 + 8 * h, two);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = without_upper(v[i]);
        }
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
k_grouped_resident(const __grid_constant__ SplitArgs p, const __grid_constant__ CUtensorMap row_map, int wide_out) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    int* const first_unit = reinterpret_cast<int*>(smem + kUnits0);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + kUnits0 + ((FMB_MAX_GROUPS + 1) * 4 + 7) / 8 * 8);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kRaw + 2 * kPlanes + 5);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto raw_full = [&](int s) { return bar0 + 8u * s; };
    auto raw_empty = [&](int s) { return bar0 + 8u * (kRaw + s); };
    auto plane_full = [&](int s) { return bar0 + 8u * (2 * kRaw + s); };
    auto plane_empty = [&](int s) { return bar0 + 8u * (2 * kRaw + kPlanes + s); };
    auto acc_full = [&](int b) { return bar0 + 8u * (2 * kRaw + 2 * kPlanes + b); };
    auto acc_empty = [&](int b) { return bar0 + 8u * (2 * kRaw + 2 * kPlanes + 2 + b); };
    const uint32_t w_full = bar0 + 8u * (2 * kRaw + 2 * kPlanes + 4);
    const int warp = uniform_warp(), lane = threadIdx.x & 31;

    if (warp == 2) tmem_alloc(smem_u32(tmem_slot), 512);
    if (warp == 1 && elect_one()) {
        for (int s = 0; s < kRaw; ++s) {
            mbar_init(raw_full(s), 1);
            mbar_init(raw_empty(s), kSplitWarps);
        }
        for (int s = 0; s < kPlanes; ++s) {
            mbar_init(plane_full(s), kSplitWarps);
            mbar_init(plane_empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 4);
        }
        mbar_init(w_full, 4);
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
    const int depth = MODE == kLinear ? p.a.k : p.a.n, width = MODE == kLinear ? p.a.n : p.a.k;
    const int columns = depth <= 64 ? 64 : 128;              // of a row in the ring
    bool alive = true;
    Walk w(p.a, first_unit, kTN, p.feature_tiles, 1, kTN);

    if (warp == 0 || warp == 2 || warp == 3) {
        // ---------------------------------------------------------------- rows: a warp per tile of the ring
        const int at = warp == 0 ? 0 : warp - 1;
        int rows[4], quads = 0;
        auto find = [&] {
            quads = (w.count + 3) / 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = lane < 16 ? row_at(p, w.first + 4 * lane + i, w.first + w.count) : -1;
                rows[i] = row < 0 ? p.a.rows : row;           // what is no row is filled with zeros
            }
        };
        if (t_begin + at < t_end) {
            w.start(t_begin + at);
            find();
        }
        uint32_t phase = 0;
        for (int t = t_begin + at; t < t_end; t += kRaw, phase ^= 1) {
            alive = mbar_wait(raw_empty(at), phase ^ 1, abort_flag, kSpin);
            if (!alive) break;
            const uint32_t dst = smem_u32(smem) + at * kRawBytes, bar = raw_full(at);
            if (elect_one()) mbar_expect_tx(bar, quads * columns * 16);
            __syncwarp();
            if (lane < quads) tma_gather4(dst + lane * columns * 16, &row_map, 0, rows[0], rows[1], rows[2], rows[3], bar);
            __syncwarp();
            if (t + kRaw < t_end) {
                w.step(kRaw);
                find();
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMAs
        constexpr uint32_t kDesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kTN >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        uint32_t w_phase = 0;
        const int steps = (depth + 15) / 16;
        for (int t = t_begin, n = 0; t < t_end; ++t, ++n) {
            const int s = n & 1;
            const uint32_t phase = (n >> 1) & 1;
            if (n == 0) w.start(t);
            else w.step(1);
            if (n == 0 || w.leads()) {
                alive = mbar_wait(w_full, w_phase, abort_flag, kSpin);
                w_phase ^= 1;
            }
            alive = alive && mbar_wait(acc_empty(s), phase ^ 1, abort_flag, kSpin);
            alive = alive && mbar_wait(plane_full(s), phase, abort_flag, kSpin);
            if (!alive) break;
            fence_after_sync();
            const uint64_t plane = make_desc(smem_u32(smem) + kPlane0 + s * kPlaneBytes);
            const uint32_t main = tmem + kAccumulators + s * 2 * kTN, rest = main + kTN;
            if (elect_one()) {
                for (int k = 0; k < steps; ++k) {
                    const uint64_t b = plane + (uint64_t)((k >> 2) * kPlaneTile + (k & 3) * 32) / 16;
                    constexpr uint64_t kPart = 2 * kPlaneTile / 16;
                    const uint32_t a = tmem + k * 8;
                    mma_f16_ts(rest, a + 128, b, kDesc, k > 0);              // lo hi
                    mma_f16_ts(rest, a + 64, b + kPart, kDesc, 1);           // mid mid
                    mma_f16_ts(rest, a, b + 2 * kPart, kDesc, 1);            // hi lo
                    mma_f16_ts(rest, a + 64, b, kDesc, 1);                   // mid hi
                    mma_f16_ts(rest, a, b + kPart, kDesc, 1);                // hi mid
                    mma_f16_ts(main, a, b, kDesc, k > 0);                    // hi hi
                }
                mma_commit(plane_empty(s));
                mma_commit(acc_full(s));
            }
            __syncwarp();
        }
    } else if (warp >= 4 && warp < 4 + kEpilogueWarps) {
        // ---------------------------------------------------------------- weights in, results out
        const int quarter = warp & 3, set = (warp - 4) >> 2, id = quarter * 32 + lane;
        float* const out = (float*)(MODE == kLinear ? p.a.y : p.a.x);
        const long long stride = MODE == kLinear ? p.a.y_stride : p.a.x_stride;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        float* const turn = reinterpret_cast<float*>(smem + kTurn0 + set * kTurnBytes);      // [rows][128 features]
        if (p.a.zero_rest) {
            const int from = min(max(p.a.offsets[p.a.groups], 0), p.a.rows);
            for (int e = from + blockIdx.x * kEpilogueWarps + warp - 4; e < p.a.rows; e += gridDim.x * kEpilogueWarps) {
                const int row = row_at(p, e, p.a.rows);
                if (row >= 0)
                    for (int c = lane; c < width; c += 32) out[row * stride + c] = 0.0f;
            }
        }
        int row_low = -1, row_high = -1;
        auto find = [&] {
            row_low = row_at(p, w.first + lane, w.first + w.count);
            row_high = row_at(p, w.first + 32 + lane, w.first + w.count);
        };
        if (t_begin + set < t_end) {
            w.start(t_begin + set);
            find();
        }
        for (int t = t_begin + set, n = set; t < t_end; t += 2, n += 2) {
            if (n == 0 || w.leads()) {
                // other weights: nobody reads the old ones once the tile before, the other set's, has its accumulators
                if (n > 0) mbar_wait(acc_full(set ^ 1), ((n - 1) >> 1) & 1, abort_flag, kSpin);
                fence_after_sync();
                bring_weights<MODE>(p, w, w.feature0 + id, depth, tmem + lanes);
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(w_full);
            }
            // (one that runs out does not end the loop: the set's warps meet at barriers, and all have to come)
            mbar_wait(acc_full(set), (n >> 1) & 1, abort_flag, kSpin);
            fence_after_sync();
            const uint32_t main = tmem + lanes + kAccumulators + set * 2 * kTN;
            const int low = row_low, high = row_high, feature0 = w.feature0;
#pragma unroll 1
            for (int r0 = 0; r0 < kTN; r0 += kTurnRows) {
                float v[16], u[16];
                tmem_load_16x2(main + r0, main + kTN + r0, v, u);
                if (r0 == kTN - kTurnRows) {
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty(set));
                    if (t + 2 < t_end) {
                        w.step(2);
                        find();
                    }
                }
                named_barrier(1 + set, 128);                 // what was here has been read
#pragma unroll
                for (int j = 0; j < kTurnRows; ++j) turn[j * 128 + id] = infinite(v[j]) ? v[j] : v[j] + u[j];
                named_barrier(1 + set, 128);
                float4 q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const float4*>(turn + (quarter * 4 + j) * 128 + 4 * lane);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = r0 + quarter * 4 + j, row = __shfl_sync(0xffffffffu, r0 < 32 ? low : high, at & 31);
                    float* const to = out + row * stride + feature0 + 4 * lane;
                    const int live = row < 0 ? 0 : width - feature0 - 4 * lane;
                    if (wide_out) {
                        if (live > 0) *reinterpret_cast<float4*>(to) = q[j];
                    } else {
                        if (live > 0) to[0] = q[j].x;
                        if (live > 1) to[1] = q[j].y;
                        if (live > 2) to[2] = q[j].z;
                        if (live > 3) to[3] = q[j].w;
                    }
                }
            }
        }
    } else if (warp >= 4 + kEpilogueWarps) {
        // ---------------------------------------------------------------- split
        const int i = threadIdx.x - 32 * (4 + kEpilogueWarps);
        const int row_shift = columns == 64 ? 4 : 5;           // quads of a row
        for (int t = t_begin, n = 0, at = 0, raw_phase = 0; t < t_end; ++t, ++n) {
            const int s = n & 1;
            alive = mbar_wait(raw_full(at), raw_phase, abort_flag, kSpin);
            if (!alive) break;
            float4 q[8];
            const float4* const raw = reinterpret_cast<const float4*>(smem + at * kRawBytes);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < 4 || columns == 128) q[j] = raw[i + j * 256];
            __syncwarp();
            if (lane == 0) mbar_arrive(raw_empty(at));
            alive = mbar_wait(plane_empty(s), ((n >> 1) & 1) ^ 1, abort_flag, kSpin);
            if (!alive) break;
            uint8_t* const plane = smem + kPlane0 + s * kPlaneBytes;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < 4 || columns == 128) {
                    const int idx = i + j * 256, row = idx >> row_shift, quad = idx & ((1 << row_shift) - 1);
                    store_quad<2 * kPlaneTile>(plane, (quad >> 4) * kPlaneTile + quad_offset(row, quad & 15), q[j]);
                }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(plane_full(s));
            if (++at == kRaw) {
                at = 0;
                raw_phase ^= 1;
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 2) {
        fence_after_sync();
        if (*abort_flag) {
            // a wait ran out: copies and MMAs under way end before the CTA gives its memory back
            for (int n = 0; n < 20000; ++n) __nanosleep(1000);
            if (lane == 0 && p.a.status) atomicOr(p.a.status, FMB_STATUS_TENSOR_TIMEOUT);
        }
        __syncwarp();
        tmem_free(tmem, 512);
    }
}

template <int MODE>
int launch(const SplitArgs& p, const CUtensorMap& rows, int wide_out, cudaStream_t stream) {
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_grouped_resident<MODE>, kSmem));
    const long long tiles = most_units(&p.a, kTN) * p.feature_tiles;
    k_grouped_resident<MODE><<<(int)std::min<long long>(tiles, sm_count()), kThreads, kSmem, stream>>>(p, rows, wide_out);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

}  // namespace

int resident_launch(const fmb_grouped_t* a, Mode mode, cudaStream_t stream) {
    const bool forward = mode == kLinear;
    const int depth = forward ? a->k : a->n, width = forward ? a->n : a->k;
    CUtensorMap rows;
    FMB_REQUIRE(encode_map(&rows, a->type, forward ? a->x : a->y, depth, a->rows, 1, forward ? a->x_stride : a->y_stride, 0, 1, 2,
                           depth <= 64 ? 64 : 128, false),
                "grouped product: tensor maps");
    SplitArgs p;
    p.a = *a;
    p.feature_tiles = ceil_div(width, 128);
    p.row_tiles = 1;
    p.unit_rows = kTN;
    p.wide_features = four_at_a_time(a->w, a->w_row_stride, 4) && a->w_group_stride % 4 == 0;
    const int wide_out = width % 4 == 0 && four_at_a_time(forward ? a->y : a->x, forward ? a->y_stride : a->x_stride, 4);
    return forward ? launch<kLinear>(p, rows, wide_out, stream) : launch<kInputGradient>(p, rows, wide_out, stream);
}

}  // namespace grp
}  // namespace fmb
