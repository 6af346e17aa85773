// Rows by group: a stable counting sort of row numbers by a small key (the species of an atom, the expert of a row).
//
//   count:  a CTA counts the keys of kRowsPerCta consecutive rows
//   scan:   per group, the counts of the CTAs before each CTA, and the total
//   place:  every warp of a CTA owns consecutive rows; the warps' own counts give each its first place per group, and inside
//           32 rows the lanes with the same key find their order by votes; no atomics on results, so the order is the one of
//           the row numbers
//
// Rows whose key is no group come behind all groups. Up to kRowsPerCta rows `place` alone does it: one launch.
// Bound by latency: 8 bytes move per row and the second pass reads keys from L2. A lane asks for its keys all at once and keeps them for
// both passes of `place`; one at a time, each waited for, 1,944 rows took 14 us. A call: 1,944 rows by 2 keys 11 us (one launch of
// one CTA, of which the launch is most), 2,100,003 rows by 128 keys 35 us (three launches; 17 MB, 2.6 us of memory).

#include "fmb_common.cuh"

namespace fmb {

namespace {

constexpr int kWarps = 32, kThreads = kWarps * 32;
constexpr int kKeys = 8;                                  // per lane
constexpr int kRowsPerWarp = 32 * kKeys;
constexpr int kRowsPerCta = kWarps * kRowsPerWarp;

// the groups of this lane's rows begin + 32 i + lane: `groups` stands for "no group", -1 for rows past the end
template <typename K>
__device__ __forceinline__ void load_keys(const K* __restrict__ keys, long long begin, long long rows, int groups, int (&g)[kKeys]) {
    const int lane = threadIdx.x & 31;
    K key[kKeys];
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
        const long long row = begin + 32 * i + lane;
        key[i] = row < rows ? keys[row] : (K)-1;
    }
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
        g[i] = begin + 32 * i + lane >= rows ? -1 : key[i] < 0 || key[i] >= (K)groups ? groups : (int)key[i];
}

// Lanes whose rows have this lane's group, for each of its rows, by a vote per bit of the group's number: 3 instructions a bit,
// where a match instruction holds the SM's one unit for 80 cycles (2.1 M rows: 19 us for the counts alone).
__device__ __forceinline__ void match_groups(const int (&g)[kKeys], int bits, unsigned (&same)[kKeys]) {
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
        const unsigned there = __ballot_sync(0xffffffffu, g[i] >= 0);
        same[i] = g[i] >= 0 ? there : 0;
    }
    for (int b = 0; b < bits; ++b) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i) {
            const bool set = (g[i] >> b) & 1;
            const unsigned with = __ballot_sync(0xffffffffu, set);
            same[i] &= set ? with : ~with;
        }
    }
}

// of the 32 warps' counts of group g: what the warps before lane `w`'s have, and all of them (lane = warp)
__device__ __forceinline__ int warps_before(int mine, int& all) {
    const int lane = threadIdx.x & 31;
    int inclusive = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inclusive, o);
        if (lane >= o) inclusive += up;
    }
    all = __shfl_sync(0xffffffffu, inclusive, 31);
    return inclusive - mine;
}

template <typename K>
__global__ void __launch_bounds__(kThreads)
k_group_count(const K* __restrict__ keys, long long rows, int groups, int32_t* __restrict__ table) {
    __shared__ int counts[FMB_MAX_GROUPS + 1];
    const int width = groups + 1;
    int g[kKeys];
    load_keys(keys, (long long)blockIdx.x * kRowsPerCta + (threadIdx.x >> 5) * kRowsPerWarp, rows, groups, g);
    for (int q = threadIdx.x; q < width; q += kThreads) counts[q] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
        if (g[i] >= 0) atomicAdd(counts + g[i], 1);               // sums of integers: the same in any order
    __syncthreads();
    for (int q = threadIdx.x; q < width; q += kThreads) table[(long long)blockIdx.x * width + q] = counts[q];
}

// table[cta][g] becomes the rows of g in the CTAs before; totals[g]. A CTA takes 32 groups, its 32 warps a share of the
// table's rows each.
__global__ void __launch_bounds__(1024)
k_group_scan(int32_t* __restrict__ table, int32_t* __restrict__ totals, int ctas, int width) {
    __shared__ int part[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.x * 32 + lane;
    const int share = (ctas + 31) / 32, begin = warp * share, end = min(ctas, begin + share);
    int sum = 0;
    if (g < width) {
#pragma unroll 8
        for (int c = begin; c < end; ++c) sum += table[(long long)c * width + g];
    }
    part[warp][lane] = sum;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += part[w][lane];
    if (g >= width) return;
    for (int c0 = begin; c0 < end; c0 += 8) {
        int here[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) here[i] = c0 + i < end ? table[(long long)(c0 + i) * width + g] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (c0 + i < end) table[(long long)(c0 + i) * width + g] = before;
            before += here[i];
        }
    }
    if (warp == 31) totals[g] = before;
}

// starts[g] = sum of starts[0 .. g) for g < width, by the whole CTA
__device__ __forceinline__ void exclusive_starts(int* starts, int width) {
    __shared__ int warp_total[kWarps];
    const int per = (width + kThreads - 1) / kThreads, begin = min(width, (int)threadIdx.x * per), end = min(width, begin + per);
    int sum = 0, all;
    for (int i = begin; i < end; ++i) sum += starts[i];
    int before = warps_before(sum, all);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 31) warp_total[warp] = all;
    __syncthreads();
    int ahead = lane < warp ? warp_total[lane] : 0;
    before += warp_sum(ahead);
    for (int i = begin; i < end; ++i) {
        const int here = starts[i];
        starts[i] = before;
        before += here;
    }
    __syncthreads();
}

// ALONE: the only CTA, which takes its own counts for the totals. The CTA's rows are put in order in shared memory first, so
// that the rows of a group leave in one run.
template <typename K, bool ALONE>
__global__ void __launch_bounds__(kThreads, ALONE ? 1 : 2)
k_group_place(const K* __restrict__ keys, long long rows, int groups, int bits, const int32_t* __restrict__ table,
              const int32_t* __restrict__ totals, int32_t* __restrict__ order, int32_t* __restrict__ offsets) {
    extern __shared__ int counts[];                       // [kWarps][groups + 1], [groups + 1] starts of the CTA, [groups + 1] of all, rows
    const int width = groups + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int* const here = counts + kWarps * width;
    int* const starts = ALONE ? here : here + width;
    int* const sorted = here + 2 * width;                 // row of the CTA | group << 13
    const long long first = (long long)blockIdx.x * kRowsPerCta;
    int g[kKeys], rank[kKeys];
    load_keys(keys, first + warp * kRowsPerWarp, rows, groups, g);
    const int warps = ALONE ? (int)((rows + kRowsPerWarp - 1) / kRowsPerWarp) : kWarps;        // that have rows
    for (int i = threadIdx.x; i < warps * width; i += kThreads) counts[i] = 0;
    if (!ALONE)
        for (int q = threadIdx.x; q < width; q += kThreads) starts[q] = totals[q];
    unsigned same[kKeys];
    match_groups(g, bits, same);
    __syncthreads();
    int* const mine = counts + warp * width;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
        const int before = g[i] >= 0 ? mine[g[i]] : 0, ahead = __popc(same[i] & ((1u << lane) - 1u));
        __syncwarp();
        if (g[i] >= 0 && ahead == 0) mine[g[i]] = before + __popc(same[i]);
        rank[i] = before + ahead;
        __syncwarp();
    }
    __syncthreads();
    for (int q = warp; q < width; q += kWarps) {
        int all;
        const int before = warps_before(lane < warps ? counts[lane * width + q] : 0, all);
        if (lane < warps) counts[lane * width + q] = before;
        if (lane == 0) here[q] = all;
    }
    __syncthreads();
    exclusive_starts(here, width);
    if (!ALONE) exclusive_starts(starts, width);
    if (blockIdx.x == 0)
        for (int q = threadIdx.x; q < width; q += kThreads) offsets[q] = starts[q];
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
        if (g[i] >= 0) sorted[here[g[i]] + mine[g[i]] + rank[i]] = (warp * kRowsPerWarp + 32 * i + lane) | g[i] << 13;
    __syncthreads();
    if (!ALONE) {
        // where the CTA's rows of a group go, less their place among its own
        for (int q = threadIdx.x; q < width; q += kThreads) starts[q] += table[(long long)blockIdx.x * width + q] - here[q];
        __syncthreads();
    }
    const int count = (int)min((long long)kRowsPerCta, rows - first);
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
        const int i = threadIdx.x + j * kThreads, v = i < count ? sorted[i] : 0;
        if (i < count) order[(ALONE ? 0 : starts[v >> 13]) + i] = (int32_t)(first + (v & (kRowsPerCta - 1)));
    }
}

constexpr int place_smem(int width) { return ((kWarps + 2) * width + kRowsPerCta) * 4; }

template <typename K>
int group_rows(const K* keys, long long rows, int groups, int32_t* order, int32_t* offsets, int32_t* scratch, cudaStream_t stream) {
    const int width = groups + 1, ctas = ceil_div(rows, kRowsPerCta);
    const int smem = place_smem(width), bits = 32 - __builtin_clz(groups);
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_group_place<K, true>, place_smem(FMB_MAX_GROUPS + 1)));
    FMB_CUDA_CHECK(opt_in_shared_memory((const void*)k_group_place<K, false>, place_smem(FMB_MAX_GROUPS + 1)));
    if (ctas <= 1) {
        k_group_place<K, true><<<1, kThreads, smem, stream>>>(keys, rows, groups, bits, nullptr, nullptr, order, offsets);
        FMB_LAUNCH_CHECK();
        return FMB_OK;
    }
    int32_t* const totals = scratch + (long long)ctas * width;
    k_group_count<K><<<ctas, kThreads, 0, stream>>>(keys, rows, groups, scratch);
    FMB_LAUNCH_CHECK();
    k_group_scan<<<ceil_div(width, 32), 1024, 0, stream>>>(scratch, totals, ctas, width);
    FMB_LAUNCH_CHECK();
    k_group_place<K, false><<<ctas, kThreads, smem, stream>>>(keys, rows, groups, bits, scratch, totals, order, offsets);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

}  // namespace

}  // namespace fmb

using namespace fmb;

extern "C" FMB_API long long fmb_group_rows_scratch(long long rows, int groups) {
    if (rows <= kRowsPerCta || groups < 1) return 0;
    return ((rows + kRowsPerCta - 1) / kRowsPerCta + 1) * (groups + 1);
}

extern "C" FMB_API int fmb_group_rows(const void* keys, int key_bytes, long long rows, int groups, int32_t* order,
                                      int32_t* offsets, int32_t* scratch, fmb_stream_t stream) {
    FMB_REQUIRE(groups >= 1 && groups <= FMB_MAX_GROUPS, "fmb_group_rows: 1 to FMB_MAX_GROUPS groups");
    FMB_REQUIRE(rows >= 0 && rows < (1ll << 31) - kRowsPerCta, "fmb_group_rows: too many rows");
    FMB_REQUIRE(offsets && (rows == 0 || (keys && order)), "fmb_group_rows: null argument");
    FMB_REQUIRE(scratch || fmb_group_rows_scratch(rows, groups) == 0, "fmb_group_rows: null scratch");
    FMB_REQUIRE(key_bytes == 4 || key_bytes == 8, "fmb_group_rows: keys of 4 or 8 bytes");
    if (key_bytes == 4)
        return group_rows((const int32_t*)keys, rows, groups, order, offsets, scratch, (cudaStream_t)stream);
    return group_rows((const long long*)keys, rows, groups, order, offsets, scratch, (cudaStream_t)stream);
}
