// Entry points of the grouped products (fmb_grouped_linear and the calls beside it): checks, and which kernel runs.
//
// 16-bit operands: grouped_tc.cu. fp32 operands, split into bf16 parts on their way: grouped_parts.cu, and linears of a depth of up to
// 128, whose split weights fit in tensor memory, grouped_resident.cu.

#include "grouped.cuh"

#include <algorithm>

namespace fmb {
namespace grp {

namespace {

// Sums of the units of every group that has more than one, in the order of its entries. A thread has four values, side by side where
// `wide`; 4 or 16 threads share the units of a value where there are many (49,152 values of 37 units took 11 us with one each, for
// their round trips, and 6 with four). Groups of one unit cost their blocks only, and of those there is a bounded number.
__global__ void __launch_bounds__(256)
k_sum_units(fmb_grouped_t a, int unit_rows, int wide) {
    const int g = blockIdx.y;
    int begin, end;
    group_span(a.offsets, g, a.rows, begin, end);
    const int units = end > begin ? (end - begin - 1) / unit_rows + 1 : 1;
    if (units <= 1) return;
    __shared__ float4 parts[256];
    const int share = units > 64 ? 16 : units > 12 ? 4 : 1, threads = 256 / share;
    const int thread = threadIdx.x % threads, part = threadIdx.x / threads, from = units * part / share, to = units * (part + 1) / share;
    const long long size = (long long)a.k * a.n;
    const int step = wide ? 1 : threads;
    for (long long first = (long long)blockIdx.x * 4 * threads; first < size; first += (long long)gridDim.x * 4 * threads) {
        // this thread's values: i, i + step, ...
        const long long i = first + (wide ? 4 * thread : thread);
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int u = from; u < to; u += 4) {
            float v[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float* const at = a.scratch + unit_slot(begin, u + j, units, unit_rows) * size + i;
                if (wide) {
                    const float4 q = u + j < to && i < size ? *reinterpret_cast<const float4*>(at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    v[j][0] = q.x; v[j][1] = q.y; v[j][2] = q.z; v[j][3] = q.w;
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[j][c] = u + j < to && i + c * step < size ? at[c * step] : 0.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) sum[c] += v[j][c];
        }
        if (share > 1) {
            __syncthreads();                                      // what was here has been read
            parts[threadIdx.x] = make_float4(sum[0], sum[1], sum[2], sum[3]);
            __syncthreads();
            if (part > 0) continue;
            for (int q = 1; q < share; ++q) {
                const float4 v = parts[q * threads + thread];
                sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
            }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const long long one = i + c * step;
            if (one >= size) break;
            float* const out = (float*)a.w + g * a.w_group_stride + (one / a.n) * a.w_row_stride + one % a.n;
            *out = a.accumulate ? *out + sum[c] : sum[c];
        }
    }
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
    const long long size = (long long)a->k * a->n;
    const int wide = size % 4 == 0 && ((uintptr_t)a->scratch & 15) == 0, blocks = std::max(1, 32 * sm_count() / a->groups);
    k_sum_units<<<dim3(std::min(ceil_div(size, 64), blocks), a->groups), 256, 0, stream>>>(*a, unit_rows, wide);
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
