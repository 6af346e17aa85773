// Copies that put the 16-bit operands of a grouped product into a form that TMA takes at its full rate.
//
//   * rows and weights that do not start at multiples of 16 bytes (odd sizes), into rows that do;
//   * for the weight gradient, the rows of x and y in the order of their groups, every group filled up with zeros to a multiple of
//     64 rows: TMA brings rows that lie side by side at 64 bytes a cycle and SM, rows gathered by number at 30. Each row is read
//     once here and n / 256 or k / 256 times by the products.

#include "grouped.cuh"

#include <algorithm>

namespace fmb {
namespace grp {

namespace {

constexpr int kThreads = 256;

// eight values from src on, of which `live` exist
__device__ __forceinline__ uint4 load_eight(const uint16_t* __restrict__ src, int live, bool wide) {
    if (wide && live >= 8) return __ldg(reinterpret_cast<const uint4*>(src));
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < live ? __ldg(src + i) : 0;
    return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

// a row by one warp; the destination is filled up with zeros to `width`, a multiple of eight
__device__ __forceinline__ void copy_row(uint16_t* __restrict__ dst, const uint16_t* __restrict__ src, int columns, int width, bool wide) {
    const int lane = threadIdx.x & 31;
#pragma unroll 4
    for (int c = 8 * lane; c < width; c += 256) *reinterpret_cast<uint4*>(dst + c) = load_eight(src + c, src ? columns - c : 0, wide);
}

struct RowsArgs {
    const uint16_t* src;
    uint16_t* dst;
    long long src_stride, dst_stride;
    int columns, wide;
};

__global__ void __launch_bounds__(kThreads)
k_pack_rows(RowsArgs a, int rows) {
    for (int r = (blockIdx.x * kThreads + threadIdx.x) >> 5; r < rows; r += gridDim.x * (kThreads / 32))
        copy_row(a.dst + r * a.dst_stride, a.src + r * a.src_stride, a.columns, (int)a.dst_stride, a.wide);
}

// rows of 32-bit values, filled up with zeros to a multiple of four
__global__ void __launch_bounds__(kThreads)
k_pack_rows_32(const float* src, long long stride, int columns, float* dst, int rows) {
    const int lane = threadIdx.x & 31, width = (columns + 3) / 4 * 4;
    for (int r = (blockIdx.x * kThreads + threadIdx.x) >> 5; r < rows; r += gridDim.x * (kThreads / 32))
        for (int c = lane; c < width; c += 32) dst[(long long)r * width + c] = c < columns ? __ldg(src + r * stride + c) : 0.0f;
}

__global__ void __launch_bounds__(kThreads)
k_pack_weights_32(fmb_grouped_t a, float* dst) {
    const int g = blockIdx.y, lane = threadIdx.x & 31, width = (a.n + 3) / 4 * 4;
    int begin, end;
    group_span(a.offsets, g, a.rows, begin, end);
    if (begin == end) return;
    for (int r = (blockIdx.x * kThreads + threadIdx.x) >> 5; r < a.k; r += gridDim.x * (kThreads / 32)) {
        const float* const from = (const float*)a.w + g * a.w_group_stride + r * a.w_row_stride;
        float* const to = dst + ((long long)g * a.k + r) * width;
        for (int c = lane; c < width; c += 32) to[c] = c < a.n ? __ldg(from + c) : 0.0f;
    }
}

// the matrices of the groups that have rows
__global__ void __launch_bounds__(kThreads)
k_pack_weights(fmb_grouped_t a, uint16_t* dst, int width, int wide) {
    const int g = blockIdx.y;
    int begin, end;
    group_span(a.offsets, g, a.rows, begin, end);
    if (begin == end) return;
    const uint16_t* const from = (const uint16_t*)a.w + g * a.w_group_stride;
    uint16_t* const to = dst + (long long)g * a.k * width;
    for (int r = (blockIdx.x * kThreads + threadIdx.x) >> 5; r < a.k; r += gridDim.x * (kThreads / 32))
        copy_row(to + (long long)r * width, from + r * a.w_row_stride, a.n, width, wide);
}

// x and y by groups; first_block[g]: blocks of 64 rows of the groups before g
__global__ void __launch_bounds__(kThreads)
k_sort_rows(fmb_grouped_t a, RowsArgs x, RowsArgs y, int32_t* first_block) {
    extern __shared__ int first[];
    count_units<kThreads>(a.offsets, a.groups, a.rows, 64, 0, first);
    if (blockIdx.x == 0)
        for (int g = threadIdx.x; g <= a.groups; g += kThreads) first_block[g] = first[g];
    const long long total = units_in_all(first, a.groups, a.rows, 64) * 64ll;
    for (long long r = (blockIdx.x * kThreads + threadIdx.x) >> 5; r < total; r += gridDim.x * (kThreads / 32)) {
        const int block = (int)(r >> 6), g = group_of_unit(first, a.groups, block);
        int begin, end;
        group_span(a.offsets, g, a.rows, begin, end);
        const long long entry = begin + (long long)(block - first[g]) * 64 + (r & 63);
        int row = entry < end ? __ldg(a.order + entry) : -1;
        if (row >= a.rows) row = -1;
        copy_row(x.dst + r * x.dst_stride, row >= 0 ? x.src + row * x.src_stride : nullptr, x.columns, (int)x.dst_stride, x.wide);
        copy_row(y.dst + r * y.dst_stride, row >= 0 ? y.src + row * y.src_stride : nullptr, y.columns, (int)y.dst_stride, y.wide);
    }
}

RowsArgs rows_args(const void* src, long long stride, int columns, void* dst) {
    RowsArgs r;
    r.src = (const uint16_t*)src;
    r.dst = (uint16_t*)dst;
    r.src_stride = stride;
    r.dst_stride = (columns + 7) / 8 * 8;
    r.columns = columns;
    r.wide = ((uintptr_t)src & 15) == 0 && stride % 8 == 0;
    return r;
}

}  // namespace

int pack_rows(const void* src, long long stride, int columns, int rows, void* dst, cudaStream_t stream) {
    const int grid = std::min(ceil_div(rows, kThreads / 32), 8 * sm_count());
    k_pack_rows<<<grid, kThreads, 0, stream>>>(rows_args(src, stride, columns, dst), rows);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

int pack_rows_32(const void* src, long long stride, int columns, int rows, void* dst, cudaStream_t stream) {
    const int grid = std::min(ceil_div(rows, kThreads / 32), 8 * sm_count());
    k_pack_rows_32<<<grid, kThreads, 0, stream>>>((const float*)src, stride, columns, (float*)dst, rows);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

int pack_weights_32(const fmb_grouped_t* a, void* dst, cudaStream_t stream) {
    const int grid = std::min(ceil_div(a->k, kThreads / 32), std::max(1, 16 * sm_count() / a->groups));
    k_pack_weights_32<<<dim3(grid, a->groups), kThreads, 0, stream>>>(*a, (float*)dst);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

int pack_weights(const fmb_grouped_t* a, void* dst, cudaStream_t stream) {
    const RowsArgs r = rows_args(a->w, a->w_row_stride, a->n, dst);
    const int grid = std::min(ceil_div(a->k, kThreads / 32), std::max(1, 16 * sm_count() / a->groups));
    k_pack_weights<<<dim3(grid, a->groups), kThreads, 0, stream>>>(*a, r.dst, (int)r.dst_stride, r.wide && a->w_group_stride % 8 == 0);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

int sort_rows(const fmb_grouped_t* a, void* x, void* y, int32_t* first_block, cudaStream_t stream) {
    const int grid = std::min(ceil_div(a->rows + 64ll * a->groups, kThreads / 32), 8 * sm_count());
    k_sort_rows<<<grid, kThreads, (a->groups + 1) * (int)sizeof(int), stream>>>(
        *a, rows_args(a->x, a->x_stride, a->k, x), rows_args(a->y, a->y_stride, a->n, y), first_block);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

}  // namespace grp
}  // namespace fmb
