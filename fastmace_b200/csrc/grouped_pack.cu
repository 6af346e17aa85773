// Copies that put the 16-bit operands of a grouped product into a form that TMA takes at its full rate.
//
//   * rows and weights that do not start at multiples of 16 bytes (odd sizes), into rows that do;
//   * for the weight gradient, the rows of x and y in the order of their groups, every group filled up with zeros to a multiple of
//     64 rows: TMA brings rows that lie side by side at 64 bytes a cycle and SM, rows gathered by number at 30. Each row is read
//     once here and n / 256 or k / 256 times by the products.

#include "held.cuh"

#include <algorithm>

namespace fmb {
namespace grp {

namespace {

constexpr int kThreads = 256;

// eight values from src on, of which `live` exist
__device__ __forceinline__ uint4 load_eight(const uint16_t* __restrict__ src, int live, bool wide) {
    if (wide && live >= 8) return __ldg(reinterpret_cast<const uint4*>(src));
    if (live >= 8) {
        // by words: they begin at the first value, or at the second
        const bool odd = ((uintptr_t)src & 2) != 0;
        const uint32_t* const words = reinterpret_cast<const uint32_t*>(src + odd);
        const uint32_t a = __ldg(words), b = __ldg(words + 1), c = __ldg(words + 2);
        if (!odd) return make_uint4(a, b, c, __ldg(words + 3));
        const uint32_t first = __ldg(src), last = __ldg(src + 7);
        return make_uint4(first | a << 16, a >> 16 | b << 16, b >> 16 | c << 16, c >> 16 | last << 16);
    }
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < live ? __ldg(src + i) : 0;
    return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

// a row by one warp; the destination is filled up with zeros to `width`, a multiple of eight
__device__ __forceinline__ void copy_row(uint16_t* __restrict__ dst, const uint16_t* __restrict__ src, int columns, int width, bool wide) {
    // four loads on their way, also where a row ends before
    for (int c0 = 8 * (threadIdx.x & 31); c0 < width; c0 += 1024) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = load_eight(src + c0 + 256 * j, src ? columns - c0 - 256 * j : 0, wide);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c0 + 256 * j < width) *reinterpret_cast<uint4*>(dst + c0 + 256 * j) = v[j];
    }
}

struct RowsArgs {
    const uint16_t* src;
    uint16_t* dst;
    long long src_stride, dst_stride;
    int columns, wide;
};

// this warp's number among those of its column of the grid, or of the columns from `first` on, and how many they are
__device__ __forceinline__ int warp_of_column(int first) { return ((blockIdx.y - first) * gridDim.x * kThreads + blockIdx.x * kThreads + threadIdx.x) >> 5; }
__device__ __forceinline__ int warps_of_columns(int count) { return count * gridDim.x * (kThreads / 32); }

// Column g < columns of the grid: the matrix of group g, if it has rows; the columns behind: the rows. One launch, of which either part may
// be missing (17 matrices of 1,000 x 515 and 5,003 rows: 13 us, 17 by two launches).
__global__ void __launch_bounds__(kThreads)
k_pack(fmb_grouped_t a, uint16_t* weights, int wide, RowsArgs x, int columns) {
    const int g = blockIdx.y;
    if (g >= columns) {
        for (int r = warp_of_column(columns); r < a.rows; r += warps_of_columns(gridDim.y - columns))
            copy_row(x.dst + r * x.dst_stride, x.src + r * x.src_stride, x.columns, (int)x.dst_stride, x.wide);
        return;
    }
    int begin, end;
    group_span(a.offsets, g, a.rows, begin, end);
    if (begin == end) return;
    const int width = (a.n + 7) / 8 * 8;
    const uint16_t* const from = (const uint16_t*)a.w + g * a.w_group_stride;
    uint16_t* const to = weights + (long long)g * a.k * width;
    for (int r = warp_of_column(g); r < a.k; r += warps_of_columns(1))
        copy_row(to + (long long)r * width, from + r * a.w_row_stride, a.n, width, wide);
}

// the same for 32-bit values, filled up with zeros to a multiple of four
__device__ __forceinline__ void copy_row_32(float* __restrict__ dst, const float* __restrict__ src, int columns) {
    for (int c = threadIdx.x & 31; c < (columns + 3) / 4 * 4; c += 32) dst[c] = c < columns ? __ldg(src + c) : 0.0f;
}

__global__ void __launch_bounds__(kThreads)
k_pack_32(fmb_grouped_t a, float* weights, const float* src, long long stride, int columns_of_row, float* dst, int columns) {
    const int g = blockIdx.y;
    if (g >= columns) {
        const long long width = (columns_of_row + 3) / 4 * 4;
        for (int r = warp_of_column(columns); r < a.rows; r += warps_of_columns(gridDim.y - columns)) copy_row_32(dst + r * width, src + r * stride, columns_of_row);
        return;
    }
    int begin, end;
    group_span(a.offsets, g, a.rows, begin, end);
    if (begin == end) return;
    const long long width = (a.n + 3) / 4 * 4;
    for (int r = warp_of_column(g); r < a.k; r += warps_of_columns(1))
        copy_row_32(weights + ((long long)g * a.k + r) * width, (const float*)a.w + g * a.w_group_stride + r * a.w_row_stride, a.n);
}

// Eight values from column c of a row that is held in 8 bits, in T; what is past the columns is zero.
template <typename T>
__device__ __forceinline__ uint4 held_eight(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, int c, int columns, bool wide) {
    if (c >= columns) return make_uint4(0, 0, 0, 0);
    uint32_t v[2] = {0, 0};
    if (wide) {
        const uint2 eight = __ldg(reinterpret_cast<const uint2*>(codes + c));
        v[0] = eight.x;
        v[1] = eight.y;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < columns) v[i / 4] |= (uint32_t)__ldg(codes + c + i) << (8 * (i % 4));
    }
    const float unit = held::unit_of(__ldg(exponents + c / held::kBlock));
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 two = held::two_values(v[i / 2] >> (16 * (i % 2)));
        out[i] = eight::two_of<T>(two.x * unit, two.y * unit);
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

template <typename T>
__device__ __forceinline__ void release_row(uint16_t* __restrict__ dst, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents,
                                            int columns, int width, bool wide) {
    for (int c0 = 8 * (threadIdx.x & 31); c0 < width; c0 += 1024) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = held_eight<T>(codes, exponents, c0 + 256 * j, codes ? columns : 0, wide);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c0 + 256 * j < width) *reinterpret_cast<uint4*>(dst + c0 + 256 * j) = v[j];
    }
}

// x and y by groups; first_block[g]: blocks of 64 rows of the groups before g. HELD: x is held in 8 bits, and read back in T on its way
template <typename T, bool HELD>
__global__ void __launch_bounds__(kThreads)
k_sort_rows(fmb_grouped_t a, RowsArgs x, RowsArgs y, int32_t* first_block, const uint8_t* __restrict__ exponents) {
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
        if constexpr (HELD)
            release_row<T>(x.dst + r * x.dst_stride, row >= 0 ? (const uint8_t*)x.src + row * (long long)x.columns : nullptr,
                           exponents + row * (long long)held::blocks_of(x.columns), x.columns, (int)x.dst_stride, x.wide);
        else
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

namespace {

// A warp per row of what is copied, as far as there is room; with both, the rows have as many columns of the grid as they need.
dim3 grid_of(const fmb_grouped_t* a, bool rows, bool weights) {
    const int of_rows = std::min(ceil_div(a->rows, kThreads / 32), 8 * sm_count());
    if (!weights) return dim3(of_rows);
    const int x = std::min(ceil_div(a->k, kThreads / 32), std::max(1, 16 * sm_count() / a->groups));
    return dim3(x, a->groups + (rows ? ceil_div(of_rows, x) : 0));
}

}  // namespace

int pack(const fmb_grouped_t* a, const void* src, long long stride, int columns, void* rows, void* weights, cudaStream_t stream) {
    const bool wide = ((uintptr_t)a->w & 15) == 0 && a->w_row_stride % 8 == 0 && a->w_group_stride % 8 == 0;
    const int matrices = weights ? a->groups : 0;
    k_pack<<<grid_of(a, rows, weights), kThreads, 0, stream>>>(
        *a, (uint16_t*)weights, wide, rows_args(src, stride, columns, rows), matrices);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

int pack_32(const fmb_grouped_t* a, const void* src, long long stride, int columns, void* rows, void* weights, cudaStream_t stream) {
    const int matrices = weights ? a->groups : 0;
    k_pack_32<<<grid_of(a, rows, weights), kThreads, 0, stream>>>(
        *a, (float*)weights, (const float*)src, stride, columns, (float*)rows, matrices);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

int sort_rows(const fmb_grouped_t* a, void* x, void* y, int32_t* first_block, const uint8_t* exponents, cudaStream_t stream) {
    const int grid = std::min(ceil_div(a->rows + 64ll * a->groups, kThreads / 32), 8 * sm_count()), smem = (a->groups + 1) * (int)sizeof(int);
    RowsArgs from_x = rows_args(a->x, a->x_stride, a->k, x), from_y = rows_args(a->y, a->y_stride, a->n, y);
    if (exponents) from_x.wide = a->k % 8 == 0 && ((uintptr_t)a->x & 7) == 0;
    if (!exponents) k_sort_rows<uint16_t, false><<<grid, kThreads, smem, stream>>>(*a, from_x, from_y, first_block, nullptr);
    else if (a->type == FMB_TYPE_BF16) k_sort_rows<__nv_bfloat16, true><<<grid, kThreads, smem, stream>>>(*a, from_x, from_y, first_block, exponents);
    else k_sort_rows<__half, true><<<grid, kThreads, smem, stream>>>(*a, from_x, from_y, first_block, exponents);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

}  // namespace grp
}  // namespace fmb
