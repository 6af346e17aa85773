// What the kernels of the grouped products share: spans of the groups, units of work.
#pragma once

#include "fmb_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace fmb {
namespace grp {

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// the entries [begin, end) of group g in `order`, whatever offsets holds
__device__ __forceinline__ void group_span(const int32_t* offsets, int g, int rows, int& begin, int& end) {
    begin = min(max(offsets[g], 0), rows);
    end = min(max(offsets[g + 1], begin), rows);
}

// A unit is up to `size` entries of one group. first[g] = units of the groups before g, first[groups] = all; groups without
// rows have `empty` units. By the whole CTA (THREADS threads, a multiple of 32); ends with a barrier.
template <int THREADS>
__device__ __forceinline__ void count_units(const int32_t* offsets, int groups, int rows, int size, int empty, int* first) {
    __shared__ int warp_total[THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (groups + THREADS - 1) / THREADS, from = min(groups, (int)threadIdx.x * per), to = min(groups, from + per);
    int sum = 0;
    for (int g = from; g < to; ++g) {
        int begin, end;
        group_span(offsets, g, rows, begin, end);
        const int units = end > begin ? (end - begin - 1) / size + 1 : empty;
        first[g] = sum;
        sum += units;
    }
    int inclusive = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inclusive, o);
        if (lane >= o) inclusive += up;
    }
    if (lane == 31) warp_total[warp] = inclusive;
    __syncthreads();
    int before = inclusive - sum;
    for (int w = 0; w < warp; ++w) before += warp_total[w];
    for (int g = from; g < to; ++g) first[g] += before;
    if (threadIdx.x == THREADS - 1) first[groups] = before + sum;
    __syncthreads();
}

// Units that `rows` entries can make at most. Offsets that are none can add up to more: what is past this is left out, so that
// buffers of this many units are never left.
__host__ __device__ __forceinline__ long long most_units(int rows, int groups, int size) { return (long long)rows / size + groups; }
__device__ __forceinline__ int units_in_all(const int* first, int groups, int rows, int size) {
    return (int)min((long long)max(0, first[groups]), most_units(rows, groups, size));
}

// Where the sums of unit u of a group's `units` lie, in units: at its first entry's multiple of the size, behind the end of the group
// before. No two are alike: units that begin within one size of each other are the last of a group and one of the next group that is
// not the last, or that group has one unit and is not kept.
__host__ __device__ __forceinline__ long long unit_slot(int begin, int u, int units, int size) {
    return 2ll * (begin / size + u) + (u == units - 1);
}
__host__ __device__ __forceinline__ long long unit_slots(int rows, int size) { return 2ll * (rows / size + 1); }

// the group that unit u belongs to: the last one that begins at or before it
__device__ __forceinline__ int group_of_unit(const int* first, int groups, int u) {
    int low = 0, high = groups - 1;
    while (low < high) {
        const int mid = (low + high + 1) >> 1;
        if (first[mid] <= u) low = mid; else high = mid - 1;
    }
    return low;
}

enum Mode { kLinear = 0, kInputGradient = 1, kWeightGradient = 2 };

// tcgen05 kernels of 16-bit operands, brought by TMA (grouped_tc.cu), and the bytes of scratch that a call with these sizes,
// strides and pointers needs
// exponents, of the weight gradient: x is held in 8 bits (held.cuh), a->x points at the codes
int tma_launch(const fmb_grouped_t* a, Mode mode, cudaStream_t stream, const uint8_t* exponents = nullptr);
long long tma_scratch_bytes(const fmb_grouped_t* a, Mode mode, bool held = false);
// tcgen05 kernel that keeps the split weights in tensor memory (grouped_resident.cu): fp32 linears of a depth of at most 128, rows
// that TMA takes
int resident_launch(const fmb_grouped_t* a, Mode mode, cudaStream_t stream);

// rows that start at multiples of four values, so that they can be read four at a time
inline bool four_at_a_time(const void* base, long long stride, int bytes) {
    return ((uintptr_t)base & (uintptr_t)(4 * bytes - 1)) == 0 && stride % 4 == 0;
}

// all fp32 products, and the floats of scratch they need (grouped_parts.cu)
int parts_launch(const fmb_grouped_t* a, Mode mode, cudaStream_t stream);
long long parts_scratch(const fmb_grouped_t* a, Mode mode);

inline long long most_units(const fmb_grouped_t* a, int unit_rows) { return most_units(a->rows, a->groups, unit_rows); }
// sums of the units of every group that has more than one, from scratch to w
int sum_units(const fmb_grouped_t* a, int unit_rows, cudaStream_t stream);
int sm_count();

// copies into the layouts that TMA takes (grouped_pack.cu)
// (rows, weights: where to, or null; in 32 bits the strides are multiples of four values, else of eight)
int pack(const fmb_grouped_t* a, const void* src, long long stride, int columns, void* rows, void* weights, cudaStream_t stream);
int pack_32(const fmb_grouped_t* a, const void* src, long long stride, int columns, void* rows, void* weights, cudaStream_t stream);
int sort_rows(const fmb_grouped_t* a, void* x, void* y, int32_t* first_block, const uint8_t* exponents, cudaStream_t stream);

}  // namespace grp
}  // namespace fmb
