// Grouped products in fp32: linear, input gradient and weight gradient (linears of a depth of up to 128: grouped_resident.cu).
//
// x = hi + mid + lo with eight significant bits each, cut off rather than rounded, is exact from 2^-110 on, without scales: bf16 reaches
// down to 2^-133, and what of a smaller x lies below that is lost. Of the nine products of two such triples of bf16 the six largest are taken,
//     hi hi | hi mid + mid hi | hi lo + mid mid + lo hi        (what is left out is below 2^-21 of |x| |w|, 2^-24 on average)
// The tensor core cuts its accumulator off at every instruction, so hi hi has columns of its own -- the others are 2^-8 of
// it -- and accumulators move to fp32 registers every kChunk of the depth. Against tf32 pairs: the same tensor time (six products
// at twice the rate against three), a seventh of the error, and operands whose depth does not run along memory.
//
// A tile is D[128 features][128 rows of the output] as in grouped_tc.cu, over blocks of 32 of the depth. TMA brings both sides into
// a ring of three blocks (rows named by the groups' order by gather, weights by tiles), four warps split them into bf16 planes of
// the layout the MMAs read, one warp issues five MMAs per 16 of the depth (hi x [hi | mid] with 256 columns into [hi hi | rest], then
// hi lo, mid hi, mid mid, lo hi into rest), and eight warps add the accumulators up and write rows of 512 bytes.
//
// Bound by the tensor cores where there is work (9,000 x 2048 x 1024: a PFLOP/s of bf16 products, 166 TFLOP/s of the fp32 ones), by
// memory for the weight gradient of 128 channels: 1 KB of rows per tile and row, 1,390 cycles of memory's share per block against
// 770 of MMAs. Where that leaves few tiles (a few species: one per group) the rows of a group are cut into units whose sums
// k_sum_units adds up in order.

#include "grouped_tc.cuh"

#include <algorithm>

namespace fmb {
namespace grp {

namespace {

using namespace tc;

constexpr int kStep = 32;                                  // depth of a block
constexpr int kRaw = 3, kRawSide = kStep * 128 * 4, kRawBytes = 2 * kRawSide;           // features, then rows of the output
constexpr int kPlanes = 2, kChunkTile = kStep * 64 * 2, kPart = 2 * kChunkTile, kSide = 3 * kPart, kPlaneBytes = 2 * kSide;
constexpr int kTurnRows = 16, kTurnBytes = kTurnRows * 128 * 4;
constexpr int kPlane0 = kRaw * kRawBytes, kTurn0 = kPlane0 + kPlanes * kPlaneBytes, kUnits0 = kTurn0 + 2 * kTurnBytes;
constexpr int kSmem = 1024 + kUnits0 + (FMB_MAX_GROUPS + 1) * 4 + 256;
constexpr int kEpilogueWarps = 8, kSplitWarps = 4, kThreads = 32 * (4 + kEpilogueWarps + kSplitWarps);
constexpr int kChunk = 256, kChunkBlocks = kChunk / kStep;
static_assert(kSmem <= 227 * 1024, "fits an SM");

// A plane of 128 features or rows is MN-major (32 depths of 64 each, 4 KB apart, 1024 bytes between 8 depths, 128-byte swizzle) or
// K-major (64-byte rows, 512 bytes between 8 of them, 64-byte swizzle).
template <bool K_MAJOR>
__device__ __forceinline__ uint64_t plane_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3ffff) >> 4);
    d |= K_MAJOR ? (uint64_t)1 << 16 : (uint64_t)(kChunkTile >> 4) << 16;
    d |= (uint64_t)((K_MAJOR ? 512 : 1024) >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)(K_MAJOR ? 4 : 2) << 61;
    return d;
}

// one side of a block, 128 x 32 values in rows of memory, by 128 threads into its planes
template <bool K_MAJOR>
__device__ __forceinline__ void split_side(const float4* raw, uint8_t* plane, int i) {
    float4 q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = raw[i + j * 128];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int idx = i + j * 128;
        if constexpr (K_MAJOR) {
            const int row = idx >> 3, quad = idx & 7;
            store_quad<kPart>(plane, (uint32_t)(row * 64 + (((quad >> 1) ^ ((row >> 1) & 3)) << 4) + (quad & 1) * 8), q[j]);
        } else {
            const int depth = idx >> 5, quad = idx & 31;
            store_quad<kPart>(plane, (quad >> 4) * kChunkTile + quad_offset(depth, quad & 15), q[j]);
        }
    }
}

// sums of the five smaller products as they are to be added to those of hi hi (one look at sixteen: a choice for each costs a weight
// gradient of 9,000 x 2,048 x 1,024 4 %, this 1)
__device__ __forceinline__ void finite_rest(const float (&main)[16], float (&rest)[16]) {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; j += 2) top = fmaxf(fmaxf(fabsf(main[j]), fabsf(main[j + 1])), top);
    if (__any_sync(0xffffffffu, infinite(top))) {        // (by the whole warp: what follows is too)
#pragma unroll
        for (int j = 0; j < 16; ++j) rest[j] = infinite(main[j]) ? 0.0f : rest[j];
    }
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
k_grouped_parts(const __grid_constant__ SplitArgs p, const __grid_constant__ CUtensorMap feature_map, const __grid_constant__ CUtensorMap row_map, int wide_out) {
    constexpr bool kWeights = MODE == kWeightGradient;
    constexpr bool kFeaturesK = MODE == kInputGradient, kRowsK = !kWeights;       // sides whose depth runs along memory
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    int* const first_unit = reinterpret_cast<int*>(smem + kUnits0);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + kUnits0 + ((FMB_MAX_GROUPS + 1) * 4 + 7) / 8 * 8);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kRaw + 2 * kPlanes + 4);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto raw_full = [&](int s) { return bar0 + 8u * s; };
    auto raw_empty = [&](int s) { return bar0 + 8u * (kRaw + s); };
    auto plane_full = [&](int s) { return bar0 + 8u * (2 * kRaw + s); };
    auto plane_empty = [&](int s) { return bar0 + 8u * (2 * kRaw + kPlanes + s); };
    auto acc_full = [&](int b) { return bar0 + 8u * (2 * kRaw + 2 * kPlanes + b); };
    auto acc_empty = [&](int b) { return bar0 + 8u * (2 * kRaw + 2 * kPlanes + 2 + b); };
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
            mbar_init(acc_empty(b), kEpilogueWarps);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    count_units<kThreads>(p.a.offsets, p.a.groups, p.a.rows, p.unit_rows, kWeights ? 1 : 0, first_unit);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const bool split = !kWeights && p.split > 1;
    const int t_first = split ? blockIdx.x / p.split : blockIdx.x, t_step = split ? gridDim.x / p.split : gridDim.x, part = split ? blockIdx.x % p.split : 0;
    const int all_tiles = units_in_all(first_unit, p.a.groups, p.a.rows, p.unit_rows) * p.feature_tiles * p.row_tiles;
    const int tiles = split ? min(all_tiles, t_step) : all_tiles;
    // not of the weight gradient: depth, and the blocks of it that are this CTA's
    const int depth_of_row = MODE == kLinear ? p.a.k : p.a.n, row_blocks = (depth_of_row + kStep - 1) / kStep;
    const int first_block = split ? row_blocks * part / p.split : 0, my_blocks = split ? row_blocks * (part + 1) / p.split - first_block : row_blocks;
    bool alive = true;
    Walk w(p.a, first_unit, p.unit_rows, p.feature_tiles, p.row_tiles, 128);

    if (warp == 0 || warp == 2 || warp == 3) {
        // ---------------------------------------------------------------- rows: a warp per block of the ring
        const int mine = warp == 0 ? 0 : warp - 1;
        uint32_t phase = 0;
        int slot = 0;                                         // of the ring, the next block's
        for (int t = t_first; alive && t < tiles; t += t_step) {
            if (t == t_first) w.start(t);
            else w.step(t_step);
            const int blocks = kWeights ? (w.count + kStep - 1) / kStep : my_blocks, end = w.first + w.count;
            int b = mine - slot;                              // this warp's first block of the tile
            if (b < 0) b += kRaw;
            slot = (slot + blocks) % kRaw;
            int rows[4];
            auto find = [&](int entry) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = row_at(p, entry + i, end);
                    rows[i] = row < 0 ? p.a.rows : row;       // what is no row is filled with zeros
                }
            };
            if (!kWeights) find(w.first + 4 * lane);          // a lane brings four rows of the output
            for (; b < blocks; b += kRaw, phase ^= 1) {
                if (kWeights) find(w.first + b * kStep + 4 * (lane & 7));       // lanes 0 to 7 bring four rows of y each, lanes 8 to 15 the same of x
                alive = mbar_wait(raw_empty(mine), phase ^ 1, abort_flag, kSpin);
                if (!alive) break;
                const uint32_t dst = smem_u32(smem) + mine * kRawBytes, bar = raw_full(mine);
                if constexpr (kWeights) {
                    const int quads = min(8, (w.count - b * kStep + 15) / 16 * 4);       // rows past the end, up to a multiple of 16, are zeros
                    if (elect_one()) mbar_expect_tx(bar, quads * 4096);
                    __syncwarp();
                    if (lane < quads) tma_gather4(dst + lane * 2048, &feature_map, w.feature0, rows[0], rows[1], rows[2], rows[3], bar);
                    if (lane >= 8 && lane < 8 + quads)
                        tma_gather4(dst + kRawSide + (lane - 8) * 2048, &row_map, w.row0, rows[0], rows[1], rows[2], rows[3], bar);
                } else {
                    const int quads = (w.count + 3) / 4, column = (first_block + b) * kStep;
                    if (elect_one()) {
                        mbar_expect_tx(bar, kRawSide + quads * 512);
                        if constexpr (MODE == kLinear) tma_tile_3d(dst, &feature_map, w.feature0, column, w.g, bar);
                        else tma_tile_3d(dst, &feature_map, column, w.feature0, w.g, bar);
                    }
                    __syncwarp();
                    if (lane < quads) tma_gather4(dst + kRawSide + lane * 512, &row_map, column, rows[0], rows[1], rows[2], rows[3], bar);
                }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMAs
        constexpr uint32_t kMajor = (kFeaturesK ? 0 : 1u << 15) | (kRowsK ? 0 : 1u << 16);
        constexpr uint32_t kDesc = (1u << 4) | (1u << 7) | (1u << 10) | kMajor | ((uint32_t)(128 >> 4) << 24);
        constexpr uint32_t k128 = (uint32_t)(128 >> 3) << 17, k256 = (uint32_t)(256 >> 3) << 17;
        int at = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        for (int t = t_first; alive && t < tiles; t += t_step) {
            if (t == t_first) w.start(t);
            else w.step(t_step);
            const int depth = kWeights ? w.count : depth_of_row - first_block * kStep, blocks = kWeights ? (depth + kStep - 1) / kStep : my_blocks;
            for (int b = 0; b < blocks; ++b) {
                const bool fresh = b % kChunkBlocks == 0, last = b == blocks - 1 || (b + 1) % kChunkBlocks == 0;
                if (fresh) alive = mbar_wait(acc_empty(acc), acc_phase ^ 1, abort_flag, kSpin);
                alive = alive && mbar_wait(plane_full(at), phase, abort_flag, kSpin);
                if (!alive) break;
                fence_after_sync();
                const uint32_t plane = smem_u32(smem) + kPlane0 + at * kPlaneBytes;
                const uint64_t f = plane_desc<kFeaturesK>(plane), r = plane_desc<kRowsK>(plane + kSide);
                const uint32_t main = tmem + acc * 256, rest = main + 128;
                const int steps = min(2, (depth - b * kStep + 15) / 16);
                if (elect_one()) {
                    for (int k = 0; k < steps; ++k) {
                        const uint64_t fk = f + k * (kFeaturesK ? 2 : 128), rk = r + k * (kRowsK ? 2 : 128);       // 16 of the depth: 32 or 2048 bytes
                        constexpr uint64_t kNext = kPart / 16;
                        mma_f16(main, fk, rk, kDesc | k256, k > 0 || !fresh);        // hi hi | hi mid
                        mma_f16(rest, fk, rk + 2 * kNext, kDesc | k128, 1);          // hi lo
                        mma_f16(rest, fk + kNext, rk, kDesc | k128, 1);              // mid hi
                        mma_f16(rest, fk + kNext, rk + kNext, kDesc | k128, 1);      // mid mid
                        mma_f16(rest, fk + 2 * kNext, rk, kDesc | k128, 1);          // lo hi
                    }
                    mma_commit(plane_empty(at));
                    if (last) mma_commit(acc_full(acc));
                }
                __syncwarp();
                if (last) {
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1;
                }
                if (++at == kPlanes) {
                    at = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp < 4 + kEpilogueWarps) {
        // ---------------------------------------------------------------- sums: a set of four warps per 64 rows of the output
        const int quarter = warp & 3, set = (warp - 4) >> 2, id = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        float* const turn = reinterpret_cast<float*>(smem + kTurn0 + set * kTurnBytes);      // [rows of dW][128]
        const int width = MODE == kInputGradient ? p.a.k : p.a.n;
        int acc = 0;
        uint32_t acc_phase = 0;
        if (!kWeights && p.a.zero_rest) {
            float* const out = (float*)(MODE == kLinear ? p.a.y : p.a.x);
            const long long stride = MODE == kLinear ? p.a.y_stride : p.a.x_stride;
            const int from = min(max(p.a.offsets[p.a.groups], 0), p.a.rows);
            for (int e = from + blockIdx.x * kEpilogueWarps + warp - 4; e < p.a.rows; e += gridDim.x * kEpilogueWarps) {
                const int row = row_at(p, e, p.a.rows);
                if (row >= 0)
                    for (int c = lane; c < width; c += 32) out[row * stride + c] = 0.0f;
            }
        }
        // (a wait that runs out does not end the loop: the set's warps meet at barriers, and all have to come)
        for (int t = t_first; t < tiles; t += t_step) {
            if (t == t_first) w.start(t);
            else w.step(t_step);
            const int chunks = kWeights ? (w.count + kChunk - 1) / kChunk : (my_blocks + kChunkBlocks - 1) / kChunkBlocks;
            int low = -1, high = -1;                         // rows of the output of a linear
            if (!kWeights) {
                low = row_at(p, w.first + set * 64 + lane, w.first + w.count);
                high = row_at(p, w.first + set * 64 + 32 + lane, w.first + w.count);
            }
            float sum[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) sum[j] = 0.0f;
            for (int c = 0; c < chunks; ++c) {
                mbar_wait(acc_full(acc), acc_phase, abort_flag, kSpin);
                fence_after_sync();
                const uint32_t d = tmem + lanes + acc * 256 + set * 64;
#pragma unroll
                for (int j0 = 0; j0 < 64; j0 += 16) {
                    float v[16], u[16];
                    tmem_load_16x2(d + j0, d + 128 + j0, v, u);
                    finite_rest(v, u);
#pragma unroll
                    for (int j = 0; j < 16; ++j) sum[j0 + j] += v[j] + u[j];
                }
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty(acc));
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
            if constexpr (!kWeights) {
                if (split) {
                    // every CTA's products are done, and the ring and planes of the first one free; the sums [row][128 features] of the
                    // others go there, and it adds them up in order
                    __syncwarp();
                    cluster_sync();
                    if (part > 0) {
                        const uint32_t to = in_leader(smem_u32(smem)) + (uint32_t)((((part - 1) * p.slot_rows + set * 64) * 128 + id) * 4);
#pragma unroll
                        for (int j = 0; j < 64; ++j)
                            if (set * 64 + j < w.count) asm volatile("st.shared::cluster.f32 [%0], %1;" :: "r"(to + j * 512), "f"(sum[j]) : "memory");
                    }
                    __syncwarp();
                    cluster_sync();
                    if (part > 0) break;
                    for (int q = 1; q < p.split; ++q) {
                        const float* const from = reinterpret_cast<const float*>(smem) + ((q - 1) * p.slot_rows + set * 64) * 128 + id;
#pragma unroll
                        for (int j = 0; j < 64; ++j) sum[j] += set * 64 + j < w.count ? from[j * 128] : 0.0f;
                    }
                }
            }
            const bool direct = !kWeights || w.units <= 1, add = kWeights && direct && p.a.accumulate, wide = direct ? wide_out : p.a.n % 4 == 0;
            const int feature = w.feature0 + 4 * lane, live = width - feature;
            long long stride;
            float* out;
            if constexpr (kWeights) {
                stride = direct ? p.a.w_row_stride : p.a.n;
                out = (direct ? (float*)p.a.w + w.g * p.a.w_group_stride : p.a.scratch + w.slot * p.a.k * p.a.n) + feature;
            } else {
                stride = MODE == kLinear ? p.a.y_stride : p.a.x_stride;
                out = (float*)(MODE == kLinear ? p.a.y : p.a.x) + feature;
            }
#pragma unroll
            for (int r0 = 0; r0 < 64; r0 += kTurnRows) {
                named_barrier(1 + set, 128);                 // what was here has been read
#pragma unroll
                for (int j = 0; j < kTurnRows; ++j) turn[j * 128 + id] = sum[r0 + j];
                named_barrier(1 + set, 128);
                float4 q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const float4*>(turn + (quarter * 4 + j) * 128 + 4 * lane);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = r0 + quarter * 4 + j;
                    int row;
                    if constexpr (kWeights) row = w.row0 + set * 64 + at < p.a.k ? w.row0 + set * 64 + at : -1;
                    else row = __shfl_sync(0xffffffffu, r0 < 32 ? low : high, at & 31);
                    if (row < 0) continue;
                    float* const to = out + row * stride;
                    if (wide) {
                        if (live > 0) {
                            if (add) {
                                const float4 old = *reinterpret_cast<const float4*>(to);
                                q[j].x += old.x; q[j].y += old.y; q[j].z += old.z; q[j].w += old.w;
                            }
                            *reinterpret_cast<float4*>(to) = q[j];
                        }
                    } else {
                        if (live > 0) to[0] = add ? to[0] + q[j].x : q[j].x;
                        if (live > 1) to[1] = add ? to[1] + q[j].y : q[j].y;
                        if (live > 2) to[2] = add ? to[2] + q[j].z : q[j].z;
                        if (live > 3) to[3] = add ? to[3] + q[j].w : q[j].w;
                    }
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- split
        const int i = threadIdx.x - 32 * (4 + kEpilogueWarps);
        int at = 0, s = 0;
        uint32_t raw_phase = 0, phase = 0;
        for (int t = t_first; alive && t < tiles; t += t_step) {
            if (t == t_first) w.start(t);
            else w.step(t_step);
            const int blocks = kWeights ? (w.count + kStep - 1) / kStep : my_blocks;
            for (int b = 0; b < blocks; ++b) {
                alive = mbar_wait(raw_full(at), raw_phase, abort_flag, kSpin);
                alive = alive && mbar_wait(plane_empty(s), phase ^ 1, abort_flag, kSpin);
                if (!alive) break;
                const float4* const raw = reinterpret_cast<const float4*>(smem + at * kRawBytes);
                uint8_t* const plane = smem + kPlane0 + s * kPlaneBytes;
                split_side<kFeaturesK>(raw, plane, i);
                split_side<kRowsK>(raw + kRawSide / 16, plane + kSide, i);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(raw_empty(at));
                    mbar_arrive(plane_full(s));
                }
                if (++at == kRaw) {
                    at = 0;
                    raw_phase ^= 1;
                }
                if (++s == kPlanes) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    }
    if (split && t_first < tiles && (warp < 4 || warp >= 4 + kEpilogueWarps)) {
        // (as the warps that join the sums)
        __syncwarp();
        cluster_sync();
        cluster_sync();
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

bool rows_fit(const void* base, long long stride) { return four_at_a_time(base, stride, 4) && stride > 0; }

// linears whose split weights fit in tensor memory (grouped_resident.cu, whose threads read the weights from where they are)
bool is_resident(const fmb_grouped_t* a, Mode mode) { return mode != kWeightGradient && (mode == kLinear ? a->k : a->n) <= 128; }

// Scratch: sums of units of the weight gradient, then copies of rows and matrices that TMA does not take as they are (floats).
struct Plan {
    int unit_rows = 1 << 30;
    long long units = 0, x = 0, y = 0, w = 0;
    long long floats() const { return units + x + y + w; }
};

Plan plan_of(const fmb_grouped_t* a, Mode mode) {
    Plan p;
    auto whole = [](long long floats) { return (floats + 63) / 64 * 64; };
    const long long k4 = (a->k + 3ll) / 4 * 4, n4 = (a->n + 3ll) / 4 * 4;
    if (mode != kInputGradient && !rows_fit(a->x, a->x_stride)) p.x = whole(a->rows * k4);
    if (mode != kLinear && !rows_fit(a->y, a->y_stride)) p.y = whole(a->rows * n4);
    if (mode != kWeightGradient) {
        // (the strides may be anything where there is one row, or one matrix, and where the weights do not come by TMA)
        if (!is_resident(a, mode) && (!rows_fit(a->w, a->k > 1 ? a->w_row_stride : 4) || (a->groups > 1 && (a->w_group_stride % 4 || a->w_group_stride <= 0))))
            p.w = whole(a->groups * a->k * n4);
        return p;
    }
    // a unit per SM where there is not a tile for each; else a group's rows, cut at an SM's share of the work; none of less than 64
    const long long of_group = ((a->n + 127) / 128) * (long long)((a->k + 127) / 128), tiles = a->groups * of_group;
    const long long units = tiles < 148 ? std::max<long long>(1, 148 * a->groups / tiles - a->groups) : std::max<long long>(1, 148 / of_group);
    const long long unit_rows = std::max<long long>(64, (a->rows / units + 31) / 32 * 32);
    if (unit_rows < a->rows) p.unit_rows = (int)unit_rows;
    if (p.unit_rows < a->rows) p.units = whole(unit_slots(a->rows, p.unit_rows) * a->k * a->n);
    return p;
}

// of a linear
long long tiles_with_rows(const fmb_grouped_t* a, int feature_tiles) { return std::min<long long>(a->rows, most_units(a, 128)) * feature_tiles; }

template <int MODE>
int launch(const SplitArgs& p, const CUtensorMap& features, const CUtensorMap& rows, int wide_out, cudaStream_t stream) {
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_grouped_parts<MODE>, kSmem));
    if (p.split > 1) {
        cudaLaunchConfig_t config = {};
        cudaLaunchAttribute cluster;
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = p.split;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
        config.gridDim = dim3((int)tiles_with_rows(&p.a, p.feature_tiles) * p.split);
        config.blockDim = dim3(kThreads);
        config.dynamicSmemBytes = kSmem;
        config.stream = stream;
        config.attrs = &cluster;
        config.numAttrs = 1;
        FMB_CUDA_CHECK(cudaLaunchKernelEx(&config, k_grouped_parts<MODE>, p, features, rows, wide_out));
        FMB_LAUNCH_CHECK();
        return FMB_OK;
    }
    const long long tiles = most_units(&p.a, p.unit_rows) * p.feature_tiles * p.row_tiles;
    k_grouped_parts<MODE><<<(int)std::min<long long>(tiles, sm_count()), kThreads, kSmem, stream>>>(p, features, rows, wide_out);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

}  // namespace

long long parts_scratch(const fmb_grouped_t* a, Mode mode) { return plan_of(a, mode).floats(); }

int parts_launch(const fmb_grouped_t* a, Mode mode, cudaStream_t stream) {
    const Plan plan = plan_of(a, mode);
    FMB_REQUIRE(plan.floats() == 0 || a->scratch, "grouped product: null scratch");
    FMB_REQUIRE(((uintptr_t)a->scratch & 255) == 0, "grouped product: scratch starts at a multiple of 256 bytes");
    SplitArgs p;
    p.a = *a;
    float* const x = a->scratch + plan.units;
    float* const y = x + plan.x;
    float* const weights = y + plan.y;
    int rc = FMB_OK;
    if (plan.x) {
        rc = pack_32(a, a->x, a->x_stride, a->k, x, plan.w ? weights : nullptr, stream);
        p.a.x = x;
        p.a.x_stride = (a->k + 3) / 4 * 4;
    }
    if (!rc && plan.y) {
        rc = pack_32(a, a->y, a->y_stride, a->n, y, plan.w ? weights : nullptr, stream);
        p.a.y = y;
        p.a.y_stride = (a->n + 3) / 4 * 4;
    }
    if (!rc && plan.w) {
        if (!plan.x && !plan.y) rc = pack_32(a, nullptr, 0, 0, nullptr, weights, stream);
        p.a.w = weights;
        p.a.w_row_stride = (a->n + 3) / 4 * 4;
        p.a.w_group_stride = a->k * p.a.w_row_stride;
    }
    if (rc) return rc;
    if (is_resident(a, mode)) return resident_launch(&p.a, mode, stream);
    CUtensorMap features, rows;
    if (mode == kWeightGradient) {
        FMB_REQUIRE(encode_map(&features, a->type, p.a.y, a->n, a->rows, 1, p.a.y_stride, 0, 1, 2, 128, false) &&
                        encode_map(&rows, a->type, p.a.x, a->k, a->rows, 1, p.a.x_stride, 0, 1, 2, 128, false),
                    "fmb_grouped_weight_gradient: tensor maps");
        p.feature_tiles = ceil_div(a->n, 128);
        p.row_tiles = ceil_div(a->k, 128);
        p.unit_rows = plan.unit_rows;
        const int wide_out = four_at_a_time(a->w, a->w_row_stride, 4) && a->w_group_stride % 4 == 0 && a->n % 4 == 0;
        rc = launch<kWeightGradient>(p, features, rows, wide_out, stream);
        return rc || !plan.units ? rc : sum_units(a, plan.unit_rows, stream);
    }
    const bool forward = mode == kLinear;
    const int width = forward ? a->n : a->k, depth = forward ? a->k : a->n;
    FMB_REQUIRE(encode_map(&features, a->type, p.a.w, a->n, a->k, a->groups, p.a.w_row_stride, p.a.w_group_stride, forward ? kStep : 128, 3,
                           forward ? 128 : kStep, false) &&
                    encode_map(&rows, a->type, forward ? p.a.x : p.a.y, depth, a->rows, 1, forward ? p.a.x_stride : p.a.y_stride, 0, 1, 2, kStep, false),
                "grouped product: tensor maps");
    p.feature_tiles = ceil_div(width, 128);
    p.row_tiles = 1;
    p.unit_rows = 128;
    // Few rows: as many CTAs as there is room for share the depth of a tile, at least eight blocks each (285 rows of 4,096 x 256 in
    // one group: 44 us, and 115 with one CTA a tile; 8 rows in 8 groups of 2,048 x 1,024: 37, 53; with four blocks each 100 rows of
    // 256 x 256 take 17.4, and 16.4)
    p.slot_rows = std::min(128, a->rows);
    for (int split = 2; split <= 8; split *= 2)
        if (tiles_with_rows(a, p.feature_tiles) * split <= (split == 2 ? 148 : 128) && ceil_div(depth, kStep) >= 8 * split &&
            (split - 1) * p.slot_rows * 512 <= kTurn0)
            p.split = split;
    const int wide_out = width % 4 == 0 && four_at_a_time(forward ? a->y : a->x, forward ? a->y_stride : a->x_stride, 4);
    return forward ? launch<kLinear>(p, features, rows, wide_out, stream) : launch<kInputGradient>(p, features, rows, wide_out, stream);
}

}  // namespace grp
}  // namespace fmb
