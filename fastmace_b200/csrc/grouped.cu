// Products of a grouped linear and its gradients: one matrix per group of rows (fmb_grouped_linear and the calls beside it).

#include "grouped.cuh"

namespace fmb {

namespace {

using namespace grp;

constexpr int kT = 64, kK = 16, kThreads = 256;

// out[r] = in[r] W[g] (or W[g]^T): a CTA takes 64 rows of a group and 64 columns
template <typename T, bool TRANSPOSED>
__global__ void __launch_bounds__(kThreads)
k_grouped_rows(fmb_grouped_t a) {
    __shared__ float sx[kK][kT + 4], sw[kK][kT + 4];
    __shared__ int32_t row_of[kT];
    const int depth = TRANSPOSED ? a.n : a.k, width = TRANSPOSED ? a.k : a.n;
    const T* const in = (const T*)(TRANSPOSED ? a.y : a.x);
    T* const out = (T*)(TRANSPOSED ? a.x : a.y);
    const long long in_stride = TRANSPOSED ? a.y_stride : a.x_stride, out_stride = TRANSPOSED ? a.x_stride : a.y_stride;
    int unit = blockIdx.x, g = 0, begin = 0, end = 0;
    for (; g <= a.groups; ++g) {
        if (g == a.groups) {
            begin = min(max(a.offsets[g], 0), a.rows);
            end = a.zero_rest ? a.rows : begin;
        } else {
            group_span(a.offsets, g, a.rows, begin, end);
        }
        const int units = (end - begin + kT - 1) / kT;
        if (unit < units) break;
        unit -= units;
    }
    if (g > a.groups) return;
    const int first = begin + unit * kT, col0 = blockIdx.y * kT;
    if (threadIdx.x < kT) {
        const int at = first + threadIdx.x;
        int row = at < end ? a.order[at] : -1;
        if (row >= a.rows) row = -1;
        row_of[threadIdx.x] = row;
    }
    __syncthreads();
    float acc[4][4] = {};
    const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
    if (g < a.groups) {
        const T* const w = (const T*)a.w + (long long)g * a.w_group_stride;
        for (int k0 = 0; k0 < depth; k0 += kK) {
            for (int i = threadIdx.x; i < kT * kK; i += kThreads) {
                const int r = i / kK, k = i % kK;
                const int row = row_of[r];
                sx[k][r] = row >= 0 && k0 + k < depth ? to_float(in[(long long)row * in_stride + k0 + k]) : 0.0f;
                const int kk = TRANSPOSED ? i % kK : i / kT, c = TRANSPOSED ? i / kK : i % kT;
                const bool live = k0 + kk < depth && col0 + c < width;
                const long long at = TRANSPOSED ? (long long)(col0 + c) * a.w_row_stride + k0 + kk
                                                : (long long)(k0 + kk) * a.w_row_stride + col0 + c;
                sw[kk][c] = live ? to_float(w[at]) : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sx[k][tr * 4 + i], sw[k][tc + 16 * j], acc[i][j]);
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row_of[tr * 4 + i];
        if (row < 0) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col0 + tc + 16 * j < width) out[(long long)row * out_stride + col0 + tc + 16 * j] = from_float<T>(acc[i][j]);
    }
}

// dW[g] (+)= sum x[r]^T y[r]: a CTA takes 64 x 64 of a group's matrix
template <typename T>
__global__ void __launch_bounds__(kThreads)
k_grouped_weights(fmb_grouped_t a) {
    __shared__ float sx[kK][kT + 4], sy[kK][kT + 4];
    const int g = blockIdx.z, k0 = blockIdx.x * kT, n0 = blockIdx.y * kT;
    int begin, end;
    group_span(a.offsets, g, a.rows, begin, end);
    float acc[4][4] = {};
    const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
    for (int r0 = begin; r0 < end; r0 += kK) {
        for (int i = threadIdx.x; i < kT * kK; i += kThreads) {
            const int r = i / kT, c = i % kT;
            int row = r0 + r < end ? a.order[r0 + r] : -1;
            if (row >= a.rows) row = -1;
            sx[r][c] = row >= 0 && k0 + c < a.k ? to_float(((const T*)a.x)[(long long)row * a.x_stride + k0 + c]) : 0.0f;
            sy[r][c] = row >= 0 && n0 + c < a.n ? to_float(((const T*)a.y)[(long long)row * a.y_stride + n0 + c]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kK; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sx[r][tr * 4 + i], sy[r][tc + 16 * j], acc[i][j]);
        __syncthreads();
    }
    float* const w = (float*)a.w + (long long)g * a.w_group_stride;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = k0 + tr * 4 + i, n = n0 + tc + 16 * j;
            if (k >= a.k || n >= a.n) continue;
            float* const at = w + (long long)k * a.w_row_stride + n;
            *at = a.accumulate ? *at + acc[i][j] : acc[i][j];
        }
}

int check(const fmb_grouped_t* a, int wide_in, int wide_out) {
    FMB_REQUIRE(a, "grouped product: null argument");
    FMB_REQUIRE(a->type >= FMB_TYPE_F32 && a->type <= FMB_TYPE_F16, "grouped product: type");
    FMB_REQUIRE(a->groups >= 1 && a->groups <= FMB_MAX_GROUPS, "grouped product: 1 to FMB_MAX_GROUPS groups");
    FMB_REQUIRE(a->rows >= 0 && a->k >= 1 && a->n >= 1, "grouped product: sizes");
    FMB_REQUIRE(a->k <= (1 << 20) && a->n <= (1 << 20), "grouped product: more than 2^20 columns");
    FMB_REQUIRE(a->rows <= (1 << 30), "grouped product: more than 2^30 rows");
    FMB_REQUIRE(a->offsets && a->w, "grouped product: null argument");
    FMB_REQUIRE(a->rows == 0 || (a->order && a->x && a->y), "grouped product: null argument");
    FMB_REQUIRE(a->rows <= 1 || (a->x_stride >= a->k && a->y_stride >= a->n), "grouped product: rows overlap");
    (void)wide_in;
    (void)wide_out;
    return FMB_OK;
}

template <bool TRANSPOSED>
int rows_launch(const fmb_grouped_t* a, cudaStream_t stream) {
    const int rc = check(a, 0, 0);
    if (rc) return rc;
    if (a->rows == 0) return FMB_OK;
    const int by_tma = tma_launch(a, TRANSPOSED ? kInputGradient : kLinear, stream);
    if (by_tma != FMB_ERR_UNSUPPORTED) return by_tma;
    const dim3 grid(ceil_div(a->rows, kT) + a->groups + 1, ceil_div(TRANSPOSED ? a->k : a->n, kT));
    if (a->type == FMB_TYPE_F32) k_grouped_rows<float, TRANSPOSED><<<grid, kThreads, 0, stream>>>(*a);
    else if (a->type == FMB_TYPE_BF16) k_grouped_rows<__nv_bfloat16, TRANSPOSED><<<grid, kThreads, 0, stream>>>(*a);
    else k_grouped_rows<__half, TRANSPOSED><<<grid, kThreads, 0, stream>>>(*a);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

}  // namespace

}  // namespace fmb

using namespace fmb;

extern "C" FMB_API int fmb_grouped_linear(const fmb_grouped_t* a, fmb_stream_t stream) {
    return rows_launch<false>(a, (cudaStream_t)stream);
}

extern "C" FMB_API int fmb_grouped_input_gradient(const fmb_grouped_t* a, fmb_stream_t stream) {
    return rows_launch<true>(a, (cudaStream_t)stream);
}

extern "C" FMB_API long long fmb_grouped_scratch(const fmb_grouped_t* a) {
    return a && a->groups >= 1 && a->k >= 1 && a->n >= 1 ? scratch_floats(a) : 0;
}

extern "C" FMB_API int fmb_grouped_weight_gradient(const fmb_grouped_t* a, fmb_stream_t stream_) {
    const int rc = check(a, 0, 0);
    if (rc) return rc;
    cudaStream_t stream = (cudaStream_t)stream_;
    if (a->rows) {
        const int by_tma = tma_launch(a, kWeightGradient, stream);
        if (by_tma != FMB_ERR_UNSUPPORTED) return by_tma;
    }
    const dim3 grid(ceil_div(a->k, kT), ceil_div(a->n, kT), a->groups);
    if (a->type == FMB_TYPE_F32) k_grouped_weights<float><<<grid, kThreads, 0, stream>>>(*a);
    else if (a->type == FMB_TYPE_BF16) k_grouped_weights<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(*a);
    else k_grouped_weights<__half><<<grid, kThreads, 0, stream>>>(*a);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}
