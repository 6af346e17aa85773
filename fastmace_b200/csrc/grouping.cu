// Rows by group: a stable counting sort of row numbers by a small key (the species of an atom, the expert of a row).
//
//   count:  a CTA counts the keys of kRowsPerCta consecutive rows
//   scan:   per group, the counts of the CTAs before each CTA, and the total
//   place:  every warp of a CTA owns consecutive rows; the warps' own counts give each its first place per group, and inside
//           32 rows the lanes with the same key find their order by a match; no atomics on results, so the order is the one of
//           the row numbers
//
// Rows whose key is no group come behind all groups. Up to kRowsPerCta rows `place` alone does it: one launch.
// Bound by latency: 8 bytes move per row and key reads hit L2 the second time.

#include "fmb_common.cuh"

namespace fmb {

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kRowsPerWarp = 1024;
constexpr int kRowsPerCta = kWarps * kRowsPerWarp;

// `groups` stands for "no group"
template <typename K>
__device__ __forceinline__ int group_of(const K* __restrict__ keys, long long row, int groups) {
    const K key = keys[row];
    return key < 0 || key >= (K)groups ? groups : (int)key;
}

// counts[warp][g] of the rows of every warp of this CTA, in shared memory
template <typename K>
__device__ __forceinline__ void count_warp(const K* __restrict__ keys, long long begin, long long end, int groups, int* counts) {
    const int lane = threadIdx.x & 31;
    for (long long row = begin + lane; row - lane < end; row += 32) {
        const int g = row < end ? group_of(keys, row, groups) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, g);
        if (g >= 0 && lane == __ffs(same) - 1) counts[g] += __popc(same);
        __syncwarp();
    }
}

template <typename K>
__global__ void __launch_bounds__(kThreads)
k_group_count(const K* __restrict__ keys, long long rows, int groups, int32_t* __restrict__ table) {
    extern __shared__ int counts[];                       // [kWarps][groups + 1]
    const int width = groups + 1, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < kWarps * width; i += kThreads) counts[i] = 0;
    __syncthreads();
    const long long begin = (long long)blockIdx.x * kRowsPerCta + warp * kRowsPerWarp;
    count_warp(keys, begin, min(rows, begin + kRowsPerWarp), groups, counts + warp * width);
    __syncthreads();
    for (int g = threadIdx.x; g < width; g += kThreads) {
        int sum = 0;
        for (int w = 0; w < kWarps; ++w) sum += counts[w * width + g];
        table[(long long)blockIdx.x * width + g] = sum;
    }
}

// table[cta][g] becomes the rows of g in the CTAs before; totals[g]. A CTA takes 32 groups, its 32 warps a share of the
// table's rows each.
__global__ void __launch_bounds__(1024)
k_group_scan(int32_t* __restrict__ table, int32_t* __restrict__ totals, int ctas, int width) {
    __shared__ int part[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.x * 32 + lane;
    const int share = (ctas + 31) / 32, begin = warp * share, end = min(ctas, begin + share);
    int sum = 0;
    if (g < width)
        for (int c = begin; c < end; ++c) sum += table[(long long)c * width + g];
    part[warp][lane] = sum;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += part[w][lane];
    if (g >= width) return;
    for (int c = begin; c < end; ++c) {
        int32_t* at = table + (long long)c * width + g;
        const int here = *at;
        *at = before;
        before += here;
    }
    if (warp == 31) totals[g] = before;
}

// starts[g] = sum of totals[0 .. g) for g <= width, by the whole CTA; `totals` and `starts` may be the same array
__device__ __forceinline__ void exclusive_starts(const int* totals, int* starts, int width) {
    __shared__ int warp_sum_of[kWarps];
    const int per = (width + kThreads - 1) / kThreads, begin = threadIdx.x * per, end = min(width, begin + per);
    int sum = 0;
    for (int i = begin; i < end; ++i) sum += totals[i];
    int inclusive = sum;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inclusive, o);
        if (lane >= o) inclusive += up;
    }
    if (lane == 31) warp_sum_of[warp] = inclusive;
    __syncthreads();
    int before = inclusive - sum;
    for (int w = 0; w < warp; ++w) before += warp_sum_of[w];
    for (int i = begin; i < end; ++i) {
        const int here = totals[i];
        starts[i] = before;
        before += here;
    }
    __syncthreads();
}

// ALONE: the only CTA, which takes its own counts for the totals
template <typename K, bool ALONE>
__global__ void __launch_bounds__(kThreads)
k_group_place(const K* __restrict__ keys, long long rows, int groups, const int32_t* __restrict__ table,
              const int32_t* __restrict__ totals, int32_t* __restrict__ order, int32_t* __restrict__ offsets) {
    extern __shared__ int counts[];                       // [kWarps][groups + 1], then [groups + 1] starts
    const int width = groups + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int* const starts = counts + kWarps * width;
    for (int i = threadIdx.x; i < kWarps * width; i += kThreads) counts[i] = 0;
    __syncthreads();
    const long long begin = (long long)blockIdx.x * kRowsPerCta + warp * kRowsPerWarp, end = min(rows, begin + kRowsPerWarp);
    count_warp(keys, begin, end, groups, counts + warp * width);
    __syncthreads();
    for (int g = threadIdx.x; g < width; g += kThreads) {
        int sum = 0;
        for (int w = 0; w < kWarps; ++w) {
            const int here = counts[w * width + g];
            counts[w * width + g] = sum;
            sum += here;
        }
        starts[g] = ALONE ? sum : totals[g];
    }
    __syncthreads();
    exclusive_starts(starts, starts, width);
    if (blockIdx.x == 0)
        for (int g = threadIdx.x; g < width; g += kThreads) offsets[g] = starts[g];
    for (int g = threadIdx.x; g < width; g += kThreads) {
        const int first = starts[g] + (ALONE ? 0 : table[(long long)blockIdx.x * width + g]);
        for (int w = 0; w < kWarps; ++w) counts[w * width + g] += first;
    }
    __syncthreads();
    int* const next = counts + warp * width;
    for (long long row = begin + lane; row - lane < end; row += 32) {
        const int g = row < end ? group_of(keys, row, groups) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, g);
        const int rank = __popc(same & ((1u << lane) - 1u));
        const int base = g >= 0 ? next[g] : 0;
        __syncwarp();
        if (g >= 0) {
            order[base + rank] = (int32_t)row;
            if (rank == 0) next[g] = base + __popc(same);
        }
        __syncwarp();
    }
}

template <typename K>
int group_rows(const K* keys, long long rows, int groups, int32_t* order, int32_t* offsets, int32_t* scratch, cudaStream_t stream) {
    const int width = groups + 1, ctas = ceil_div(rows, kRowsPerCta);
    const int smem = (kWarps + 1) * width * (int)sizeof(int);
    if (ctas <= 1) {
        k_group_place<K, true><<<1, kThreads, smem, stream>>>(keys, rows, groups, nullptr, nullptr, order, offsets);
        FMB_LAUNCH_CHECK();
        return FMB_OK;
    }
    int32_t* const totals = scratch + (long long)ctas * width;
    k_group_count<K><<<ctas, kThreads, smem, stream>>>(keys, rows, groups, scratch);
    FMB_LAUNCH_CHECK();
    k_group_scan<<<ceil_div(width, 32), 1024, 0, stream>>>(scratch, totals, ctas, width);
    FMB_LAUNCH_CHECK();
    k_group_place<K, false><<<ctas, kThreads, smem, stream>>>(keys, rows, groups, scratch, totals, order, offsets);
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
