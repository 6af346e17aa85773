// Entry points of the grouped products (fmb_grouped_linear and the calls beside it): checks, and which kernel runs.
//
// 16-bit operands: grouped_tc.cu. fp32 operands, split into bf16 parts on their way: grouped_parts.cu, and linears of a depth of up to
// 128, whose split weights fit in tensor memory, grouped_resident.cu.

#include "grouped.cuh"

#include <algorithm>

namespace fmb {
namespace grp {

namespace {

// sums of the units of every group that has more than one, in the order of its entries
__global__ void __launch_bounds__(256)
k_sum_units(fmb_grouped_t a, int unit_rows) {
    const int g = blockIdx.y;
    __shared__ int first[2];
    __shared__ float parts[4][64];
    if (threadIdx.x < 32) {
        int before = 0;
        for (int q = threadIdx.x; q < g; q += 32) {
            int begin, end;
            group_span(a.offsets, q, a.rows, begin, end);
            before += end > begin ? (end - begin - 1) / unit_rows + 1 : 1;
        }
        before = warp_sum(before);
        int begin, end;
        group_span(a.offsets, g, a.rows, begin, end);
        if (threadIdx.x == 0) {
            first[0] = before;
            first[1] = end > begin ? (end - begin - 1) / unit_rows + 1 : 1;
        }
    }
    __syncthreads();
    const int units = first[1];
    if (units <= 1 || first[0] + units > most_units(a.rows, a.groups, unit_rows)) return;
    // four threads share a sum: with one each, 49,152 values of 37 units took 11 us for their round trips
    const long long size = (long long)a.k * a.n, i = (long long)blockIdx.x * 64 + (threadIdx.x & 63);
    const int part = threadIdx.x >> 6, from = units * part / 4, to = units * (part + 1) / 4;
    float sum = 0.0f;
    if (i < size) {
        const float* const at = a.scratch + first[0] * size + i;
        for (int u = from; u < to; u += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = u + j < to ? at[(u + j) * size] : 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += v[j];
        }
    }
    parts[part][threadIdx.x & 63] = sum;
    __syncthreads();
    if (part > 0 || i >= size) return;
    sum = (sum + parts[1][threadIdx.x]) + (parts[2][threadIdx.x] + parts[3][threadIdx.x]);
    float* const out = (float*)a.w + g * a.w_group_stride + (i / a.n) * a.w_row_stride + i % a.n;
    *out = a.accumulate ? *out + sum : sum;
}

__global__ void __launch_bounds__(256)
k_zero_weights(fmb_grouped_t a) {
    const long long size = (long long)a.k * a.n;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < size; i += gridDim.x * 256ll)
        ((float*)a.w)[blockIdx.y * a.w_group_stride + (i / a.n) * a.w_row_stride + i % a.n] = 0.0f;
}

int check(const fmb_grouped_t* a) {
    FMB_REQUIRE(a, "grouped product: null argument");
    FMB_REQUIRE(a->type >= FMB_TYPE_F32 && a->type <= FMB_TYPE_F16, "grouped product: type");
    FMB_REQUIRE(a->groups >= 1 && a->groups <= FMB_MAX_GROUPS, "grouped product: 1 to FMB_MAX_GROUPS groups");
    FMB_REQUIRE(a->rows >= 0 && a->k >= 1 && a->n >= 1, "grouped product: sizes");
    FMB_REQUIRE(a->k <= (1 << 20) && a->n <= (1 << 20), "grouped product: more than 2^20 columns");
    FMB_REQUIRE(a->rows <= (1 << 30), "grouped product: more than 2^30 rows");
    FMB_REQUIRE(a->offsets && a->w, "grouped product: null argument");
    FMB_REQUIRE(a->rows == 0 || (a->order && a->x && a->y), "grouped product: null argument");
    FMB_REQUIRE(a->rows <= 1 || (a->x_stride >= a->k && a->y_stride >= a->n), "grouped product: rows overlap");
    return FMB_OK;
}

int run(const fmb_grouped_t* a, Mode mode, cudaStream_t stream) {
    const int rc = check(a);
    if (rc) return rc;
    if (a->rows == 0 && mode != kWeightGradient) return FMB_OK;
    if (a->rows == 0) {
        if (a->accumulate) return FMB_OK;
        k_zero_weights<<<dim3(std::min(ceil_div((long long)a->k * a->n, 256), 4096), a->groups), 256, 0, stream>>>(*a);
        FMB_LAUNCH_CHECK();
        return FMB_OK;
    }
    return a->type == FMB_TYPE_F32 ? parts_launch(a, mode, stream) : tma_launch(a, mode, stream);
}

}  // namespace

int sum_units(const fmb_grouped_t* a, int unit_rows, cudaStream_t stream) {
    k_sum_units<<<dim3(ceil_div((long long)a->k * a->n, 64), a->groups), 256, 0, stream>>>(*a, unit_rows);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 1;
    return sms;
}

}  // namespace grp
}  // namespace fmb

using namespace fmb;
using namespace fmb::grp;

extern "C" FMB_API int fmb_grouped_linear(const fmb_grouped_t* a, fmb_stream_t stream) { return run(a, kLinear, (cudaStream_t)stream); }

extern "C" FMB_API int fmb_grouped_input_gradient(const fmb_grouped_t* a, fmb_stream_t stream) {
    return run(a, kInputGradient, (cudaStream_t)stream);
}

extern "C" FMB_API int fmb_grouped_weight_gradient(const fmb_grouped_t* a, fmb_stream_t stream) {
    return run(a, kWeightGradient, (cudaStream_t)stream);
}

extern "C" FMB_API long long fmb_grouped_scratch(const fmb_grouped_t* a, int which) {
    if (!a || which < 0 || which > 2 || a->groups < 1 || a->k < 1 || a->n < 1 || a->rows < 1) return 0;
    return a->type == FMB_TYPE_F32 ? parts_scratch(a, (Mode)which) : tma_scratch_bytes(a, (Mode)which) / 4;
}
