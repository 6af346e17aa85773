// Weight gradient of a grouped linear in fp32: dW[g] = sum over the rows r of g of x[r]^T y[r].
//
// A tile is 128 columns of y (the accumulator lanes, contiguous in dW) by 128 columns of x; the depth are the rows of a unit, 32 at a
// time. The numbers and their products are those of grouped_split.cu, the flow is that of grouped_resident.cu: rows come by TMA
// gather (four of 512 bytes an instruction) into a ring of three blocks, four warps split them into MN-major bf16 planes, one warp
// issues five MMAs per 16 rows (hi x [hi | mid] with 256 columns into [hi hi | rest], then hi lo, mid hi, mid mid, lo hi into rest),
// and eight warps add the accumulators up in fp32 every kChunk rows and write whole rows of dW.
//
// What bounds it: 1 KB of rows per 128 x 128 tile and row, 1,390 cycles of memory's share per block of 32 against 770 of MMAs. Where
// there are few tiles (128 channels, a few species: one per group) the rows of a group are cut into units whose sums
// k_sum_units adds up in order.

#include "grouped_tc.cuh"

#include <algorithm>

namespace fmb {
namespace grp {

namespace {

using namespace tc;

constexpr int kRows = 32;                                  // of a block
constexpr int kRaw = 3, kRawSide = kRows * 128 * 4, kRawBytes = 2 * kRawSide;           // y, then x
constexpr int kPlanes = 2, kChunkTile = kRows * 64 * 2, kPart = 2 * kChunkTile, kSide = 3 * kPart, kPlaneBytes = 2 * kSide;
constexpr int kTurnRows = 16, kTurnBytes = kTurnRows * 128 * 4;
constexpr int kPlane0 = kRaw * kRawBytes, kTurn0 = kPlane0 + kPlanes * kPlaneBytes, kUnits0 = kTurn0 + 2 * kTurnBytes;
constexpr int kSmem = 1024 + kUnits0 + (FMB_MAX_GROUPS + 1) * 4 + 256;
constexpr int kEpilogueWarps = 8, kSplitWarps = 4, kThreads = 32 * (4 + kEpilogueWarps + kSplitWarps);
constexpr int kChunk = 256, kChunkBlocks = kChunk / kRows;
static_assert(kSmem <= 227 * 1024, "fits an SM");

// MN-major tile: 32 rows of 64 columns each, 4 KB apart, 1024 bytes between 8 rows
__device__ __forceinline__ uint64_t plane_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3ffff) >> 4);
    d |= (uint64_t)(kChunkTile >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

__global__ void __launch_bounds__(kThreads, 1)
k_grouped_weights(const __grid_constant__ SplitArgs p, const __grid_constant__ CUtensorMap y_map, const __grid_constant__ CUtensorMap x_map, int wide_out) {
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
    count_units<kThreads>(p.a.offsets, p.a.groups, p.a.rows, p.unit_rows, 1, first_unit);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const int tiles = units_in_all(first_unit, p.a.groups, p.a.rows, p.unit_rows) * p.feature_tiles * p.row_tiles;
    const int t_first = blockIdx.x, t_step = gridDim.x;
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
            const int blocks = (w.count + kRows - 1) / kRows, end = w.first + w.count;
            int b = mine - slot;                              // this warp's first block of the tile
            if (b < 0) b += kRaw;
            slot = (slot + blocks) % kRaw;
            for (; b < blocks; b += kRaw, phase ^= 1) {
                // lanes 0 to 7 bring four rows of y each, lanes 8 to 15 the same of x
                int rows[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = lane < 16 ? row_at(p, w.first + b * kRows + 4 * (lane & 7) + i, end) : -1;
                    rows[i] = row < 0 ? p.a.rows : row;       // what is no row is filled with zeros
                }
                alive = mbar_wait(raw_empty(mine), phase ^ 1, abort_flag, kSpin);
                if (!alive) break;
                const uint32_t dst = smem_u32(smem) + mine * kRawBytes, bar = raw_full(mine);
                const int quads = min(8, (w.count - b * kRows + 15) / 16 * 4);       // rows past the end, up to a multiple of 16, are zeros
                if (elect_one()) mbar_expect_tx(bar, quads * 4096);
                __syncwarp();
                if (lane < quads) tma_gather4(dst + lane * 2048, &y_map, w.feature0, rows[0], rows[1], rows[2], rows[3], bar);
                if (lane >= 8 && lane < 8 + quads)
                    tma_gather4(dst + kRawSide + (lane - 8) * 2048, &x_map, w.row0, rows[0], rows[1], rows[2], rows[3], bar);
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMAs
        constexpr uint32_t kDesc = (1u << 4) | (1u << 7) | (1u << 10) | (3u << 15) | ((uint32_t)(128 >> 4) << 24);
        constexpr uint32_t k128 = (uint32_t)(128 >> 3) << 17, k256 = (uint32_t)(256 >> 3) << 17;
        int at = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        for (int t = t_first; alive && t < tiles; t += t_step) {
            if (t == t_first) w.start(t);
            else w.step(t_step);
            const int blocks = (w.count + kRows - 1) / kRows;
            for (int b = 0; b < blocks; ++b) {
                const bool fresh = b % kChunkBlocks == 0, last = b == blocks - 1 || (b + 1) % kChunkBlocks == 0;
                if (fresh) alive = mbar_wait(acc_empty(acc), acc_phase ^ 1, abort_flag, kSpin);
                alive = alive && mbar_wait(plane_full(at), phase, abort_flag, kSpin);
                if (!alive) break;
                fence_after_sync();
                const uint64_t f = plane_desc(smem_u32(smem) + kPlane0 + at * kPlaneBytes), r = f + kSide / 16;
                const uint32_t main = tmem + acc * 256, rest = main + 128;
                const int steps = min(2, (w.count - b * kRows + 15) / 16);
                if (elect_one()) {
                    for (int k = 0; k < steps; ++k) {
                        const uint64_t fk = f + k * 128, rk = r + k * 128;           // 16 rows: 2048 bytes
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
        // ---------------------------------------------------------------- sums: a set of four warps per 64 columns of x
        const int quarter = warp & 3, set = (warp - 4) >> 2, id = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        float* const turn = reinterpret_cast<float*>(smem + kTurn0 + set * kTurnBytes);      // [rows of dW][128]
        int acc = 0;
        uint32_t acc_phase = 0;
        // (a wait that runs out does not end the loop: the set's warps meet at barriers, and all have to come)
        for (int t = t_first; t < tiles; t += t_step) {
            if (t == t_first) w.start(t);
            else w.step(t_step);
            const int chunks = (w.count + kChunk - 1) / kChunk;
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
#pragma unroll
                    for (int j = 0; j < 16; ++j) sum[j0 + j] += v[j] + u[j];
                }
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty(acc));
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
            const bool direct = w.units <= 1, add = direct && p.a.accumulate, wide = direct ? wide_out : p.a.n % 4 == 0;
            const long long stride = direct ? p.a.w_row_stride : p.a.n;
            const int feature = w.feature0 + 4 * lane, live = p.a.n - feature;
            float* const out = (direct ? (float*)p.a.w + w.g * p.a.w_group_stride : p.a.scratch + (long long)w.unit * p.a.k * p.a.n) + feature;
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
                    const int row = w.row0 + set * 64 + r0 + quarter * 4 + j;
                    if (row >= p.a.k) continue;
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
            const int blocks = (w.count + kRows - 1) / kRows;
            for (int b = 0; b < blocks; ++b) {
                alive = mbar_wait(raw_full(at), raw_phase, abort_flag, kSpin);
                alive = alive && mbar_wait(plane_empty(s), phase ^ 1, abort_flag, kSpin);
                if (!alive) break;
                // y, then x: 32 rows of 32 quads each, eight per thread
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    const float4* const raw = reinterpret_cast<const float4*>(smem + at * kRawBytes + side * kRawSide);
                    uint8_t* const plane = smem + kPlane0 + s * kPlaneBytes + side * kSide;
                    Quad<float> q[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) q[j].v = raw[i + j * 128];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int idx = i + j * 128, row = idx >> 5, quad = idx & 31;
                        store_quad<float, kPart>(plane, (quad >> 4) * kChunkTile + quad_offset(row, quad & 15), q[j]);
                    }
                }
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

// Scratch: sums of units, then rows of x and of y that TMA does not take as they are.
struct Plan {
    int unit_rows = 1 << 30;
    long long units = 0, x = 0, y = 0;           // floats
    long long floats() const { return units + x + y; }
};

Plan plan_of(const fmb_grouped_t* a) {
    Plan p;
    auto whole = [](long long floats) { return (floats + 63) / 64 * 64; };
    // a unit per SM where there is not a tile for each; none of less than 64 rows
    const long long tiles = a->groups * ((a->n + 127) / 128) * (long long)((a->k + 127) / 128);
    if (tiles < 148) {
        const long long wanted = std::max<long long>(1, 148 * a->groups / tiles - a->groups);
        const int unit_rows = (int)std::max<long long>(64, (a->rows / wanted + 31) / 32 * 32);
        if (unit_rows < a->rows) p.unit_rows = unit_rows;
    }
    if (p.unit_rows < a->rows) p.units = whole(most_units(a, p.unit_rows) * a->k * a->n);
    if (!rows_fit(a->x, a->x_stride)) p.x = whole(a->rows * ((a->k + 3ll) / 4 * 4));
    if (!rows_fit(a->y, a->y_stride)) p.y = whole(a->rows * ((a->n + 3ll) / 4 * 4));
    return p;
}

}  // namespace

long long weights_scratch(const fmb_grouped_t* a) { return plan_of(a).floats(); }

int weights_launch(const fmb_grouped_t* a, cudaStream_t stream) {
    const Plan plan = plan_of(a);
    FMB_REQUIRE(plan.floats() == 0 || a->scratch, "fmb_grouped_weight_gradient: null scratch");
    FMB_REQUIRE(((uintptr_t)a->scratch & 255) == 0, "grouped product: scratch starts at a multiple of 256 bytes");
    SplitArgs p;
    p.a = *a;
    if (plan.x) {
        const int rc = pack_rows_32(a->x, a->x_stride, a->k, a->rows, a->scratch + plan.units, stream);
        if (rc) return rc;
        p.a.x = a->scratch + plan.units;
        p.a.x_stride = (a->k + 3) / 4 * 4;
    }
    if (plan.y) {
        const int rc = pack_rows_32(a->y, a->y_stride, a->n, a->rows, a->scratch + plan.units + plan.x, stream);
        if (rc) return rc;
        p.a.y = a->scratch + plan.units + plan.x;
        p.a.y_stride = (a->n + 3) / 4 * 4;
    }
    CUtensorMap y_map, x_map;
    FMB_REQUIRE(encode_map(&y_map, a->type, p.a.y, a->n, a->rows, 1, p.a.y_stride, 0, 1, 2, 128, false) &&
                    encode_map(&x_map, a->type, p.a.x, a->k, a->rows, 1, p.a.x_stride, 0, 1, 2, 128, false),
                "fmb_grouped_weight_gradient: tensor maps");
    p.feature_tiles = ceil_div(a->n, 128);
    p.row_tiles = ceil_div(a->k, 128);
    p.unit_rows = plan.unit_rows;
    p.wide_features = p.wide_rows = 1;
    const int wide_out = four_at_a_time(a->w, a->w_row_stride, 4) && a->w_group_stride % 4 == 0 && a->n % 4 == 0;
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_grouped_weights, kSmem));
    const long long tiles = most_units(a, plan.unit_rows) * p.feature_tiles * p.row_tiles;
    k_grouped_weights<<<(int)std::min<long long>(tiles, sm_count()), kThreads, kSmem, stream>>>(p, y_map, x_map, wide_out);
    FMB_LAUNCH_CHECK();
    return plan.units ? sum_units(a, plan.unit_rows, stream) : FMB_OK;
}

}  // namespace grp
}  // namespace fmb
