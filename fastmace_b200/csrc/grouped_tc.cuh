// Tensor-core side of the grouped products: TMA, MMAs of 16-bit operands, tiles, and the split of fp32 into bf16 parts.
#pragma once

#include "grouped.cuh"
#include "tc_common.cuh"

#include <cuda.h>

namespace fmb {
namespace grp {

constexpr int kDepth = 64;                       // depth of a stage: 128 bytes of 16-bit values
constexpr unsigned kSpin = 1u << 20;

__device__ __forceinline__ void tma_tile_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar) : "memory");
}

__device__ __forceinline__ void tma_tile_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}

__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, int col, int r0, int r1, int r2, int r3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
                 :: "r"(dst), "l"(map), "r"(col), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar) : "memory");
}

// from shared memory, by threads that a proxy fence of the writers and a barrier precede; what lies outside the tensor is not written,
// apart from the rest of a row's last 16 bytes
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                 :: "l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" :: "n"(LEFT) : "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The forms of a CTA pair: copies may complete on a barrier of either CTA, the leader (rank 0) issues the MMAs of both.
__device__ __forceinline__ void tma_tile_3d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}

__device__ __forceinline__ void tma_tile_2d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar) : "memory");
}

__device__ __forceinline__ void tma_gather4_pair(uint32_t dst, const CUtensorMap* map, int col, int r0, int r1, int r2, int r3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
                 :: "r"(dst), "l"(map), "r"(col), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar) : "memory");
}

__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n"
        :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// arrives on the barrier at this address in both CTAs
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 :: "r"(bar), "h"((uint16_t)3) : "memory");
}

// the address of the leader's copy of a shared variable
__device__ __forceinline__ uint32_t in_leader(uint32_t address) {
    uint32_t there;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(address));
    return there;
}

// (release at CTA scope: what it announces -- copies that have completed, accumulators that have been read -- is ordered by
// the barriers and proxy fences before it. At cluster scope the instruction takes 2,000 cycles while copies are under way.)
__device__ __forceinline__ void remote_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(bar) : "memory");
}

__device__ __forceinline__ void remote_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n"
        :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// the same with the first operand in tensor memory
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, int accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n"
        :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// MN-major tile with the 128-byte swizzle: 64 depths of 64 features each, 8 KB apart, 1024 bytes between 8 depths
__device__ __forceinline__ uint64_t make_desc_mn(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3ffff) >> 4);
    d |= (uint64_t)(kDepth * 128 >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

__device__ __forceinline__ void tmem_load_32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3]), "=&r"(r[4]), "=&r"(r[5]), "=&r"(r[6]), "=&r"(r[7]),
          "=&r"(r[8]), "=&r"(r[9]), "=&r"(r[10]), "=&r"(r[11]), "=&r"(r[12]), "=&r"(r[13]), "=&r"(r[14]), "=&r"(r[15]),
          "=&r"(r[16]), "=&r"(r[17]), "=&r"(r[18]), "=&r"(r[19]), "=&r"(r[20]), "=&r"(r[21]), "=&r"(r[22]), "=&r"(r[23]),
          "=&r"(r[24]), "=&r"(r[25]), "=&r"(r[26]), "=&r"(r[27]), "=&r"(r[28]), "=&r"(r[29]), "=&r"(r[30]), "=&r"(r[31])
        : "r"(taddr) : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// ------------------------------------------------------------------------------------------------ fp32 as three bf16 parts

struct SplitArgs {
    fmb_grouped_t a;
    int feature_tiles, row_tiles, unit_rows;
    int wide_features;                           // weights that may be read four values at a time (grouped_resident.cu)
    int split = 1;                               // linears of few rows: CTAs, a cluster, that share the depth of a tile; one tile each
    int slot_rows = 0;                           // rows that a tile has at most
};

// The tiles of a launch, group by group; of a group all units (entries [first, first + count) of `order`) for the same features
// and output rows, then the next features, then the next output rows. A Walk goes through them in steps: the search
// for the group and the reads of its span happen once per group, not per tile (as much as 2,000 cycles).
struct Walk {
    const int32_t* offsets;
    const int* first_unit;
    int groups, rows, unit_rows, feature_tiles, per_unit, tile_rows;
    int g, local, units, begin, end;             // group, tile of it, its units, its span
    int unit, feature0, row0, first, count;      // the tile
    long long slot;                              // of its unit in the scratch

    __device__ __forceinline__ Walk(const fmb_grouped_t& a, const int* first_unit, int unit_rows, int feature_tiles, int row_tiles, int tile_rows)
        : offsets(a.offsets), first_unit(first_unit), groups(a.groups), rows(a.rows), unit_rows(unit_rows), feature_tiles(feature_tiles),
          per_unit(feature_tiles * row_tiles), tile_rows(tile_rows), g(0), local(0), units(1), begin(0), end(0),
          unit(0), feature0(0), row0(0), first(0), count(0), slot(0) {}

    __device__ __forceinline__ void enter() {
        units = max(1, first_unit[g + 1] - first_unit[g]);
        group_span(offsets, g, rows, begin, end);
    }
    __device__ __forceinline__ void place() {
        const int rest = local / units, skip = local - rest * units, rt = rest / feature_tiles;
        unit = first_unit[g] + skip;
        slot = min(unit_slot(begin, skip, units, unit_rows), unit_slots(rows, unit_rows) - 1);
        row0 = rt * tile_rows;
        feature0 = (rest - rt * feature_tiles) * 128;
        // offsets that are none could make a unit that lies outside its group: it has no entries. (In 64 bits: as the minimum of
        // a 32-bit difference and unit_rows the count came out as end + first, CUDA 12.9.)
        const long long at = begin + (long long)skip * unit_rows, left = end - at;
        first = left > 0 ? (int)at : end;
        count = left <= 0 ? 0 : left < unit_rows ? (int)left : unit_rows;
    }
    __device__ __forceinline__ void start(int t) {
        g = group_of_unit(first_unit, groups, t / per_unit);
        local = t - first_unit[g] * per_unit;
        enter();
        place();
    }
    // n tiles on; the caller has made sure that the launch has them
    __device__ __forceinline__ void step(int n) {
        local += n;
        while (local >= units * per_unit && g + 1 < groups) {
            local -= (first_unit[g + 1] - first_unit[g]) * per_unit;
            do ++g; while (g + 1 < groups && first_unit[g + 1] == first_unit[g]);
            enter();
        }
        place();
    }
    // first tile of its group with these features and output rows
    __device__ __forceinline__ bool leads() const { return unit == first_unit[g]; }
};

// the row that `entry` of the order names; -1 where there is none
template <typename ARGS>
__device__ __forceinline__ int row_at(const ARGS& p, int entry, int end) {
    const int row = entry < end ? __ldg(p.a.order + entry) : -1;
    return (unsigned)row < (unsigned)p.a.rows ? row : -1;
}

// four values from p on, of which `live` (at most four) exist
__device__ __forceinline__ float4 load_quad(const float* p, int live, bool wide) {
    if (wide && live >= 4) return __ldg(reinterpret_cast<const float4*>(p));
    return make_float4(live > 0 ? __ldg(p) : 0.0f, live > 1 ? __ldg(p + 1) : 0.0f, live > 2 ? __ldg(p + 2) : 0.0f, live > 3 ? __ldg(p + 3) : 0.0f);
}

// upper halves of two floats side by side
__device__ __forceinline__ uint32_t upper_halves(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }
__device__ __forceinline__ float without_upper(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// Infinities: all of one is in its upper half, and what it leaves there is no number. So where the products of the upper halves, hi hi,
// are infinite, they alone are the result; the kernels leave out the five others there. (A signalling NaN that has nothing in its upper
// half but the exponent, which no operation makes, counts as an infinity. Made the usual one while it is split, by an addition of -0 to
// every value, it costs the deep products 5 %: 9,000 x 2,048 x 1,024 223 -> 234 us.)
__device__ __forceinline__ bool infinite(float x) { return fabsf(x) == __uint_as_float(0x7f800000u); }

// the three bf16 parts of four consecutive values, at byte `offset` of each part's tile
template <int PART_BYTES>
__device__ __forceinline__ void store_quad(uint8_t* tile, uint32_t offset, float4 q) {
#pragma unroll
    for (int part = 0; part < 3; ++part) {
        *reinterpret_cast<uint2*>(tile + part * PART_BYTES + offset) = make_uint2(upper_halves(q.x, q.y), upper_halves(q.z, q.w));
        if (part < 2) q = make_float4(without_upper(q.x), without_upper(q.y), without_upper(q.z), without_upper(q.w));
    }
}

// byte of quad q of row r in a tile of 128-byte rows with the 128-byte swizzle
__device__ __forceinline__ uint32_t quad_offset(int r, int q) {
    return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + (((q >> 1) ^ (r & 7)) << 4) + (q & 1) * 8);
}

// A tensor map of [groups][rows][columns] with the strides given (in elements), in boxes of 1 x box_rows x box_columns; false
// where TMA does not take the alignment. dims 2: one group.
bool encode_map(CUtensorMap* map, int type, const void* base, int columns, int rows, int groups, long long row_stride,
                long long group_stride, int box_rows, int dims, int box_columns, bool swizzled);

}  // namespace grp
}  // namespace fmb
