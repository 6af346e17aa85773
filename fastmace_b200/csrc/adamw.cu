// AdamW over a list of tensors in one launch (more only beyond kMaxTensors): weights, gradients and moments pass once.
//
// The list travels as a kernel argument, so nothing is uploaded and a captured step replays by itself; the number of the
// step is a device counter that the last CTA to finish advances. A warp takes a block of 256 values, two float4 per lane and
// array. With moments in 8 bits the block shares a scale per moment: first moments are held as e4m3 of m / s, second
// moments as e4m3 of sqrt(v) / s, s = (largest of the block) / 448. Relative steps of 2^-4 over 2^15 and the root's smaller
// range keep the quotient m / sqrt(v) to a few per cent of itself; a v that is not zero is never held as zero, which would make
// the next quotient m / eps. All arithmetic is in fp32, rounded as written: the moments come out with the same bits
// whatever the compiler contracts, so their 8-bit codes do not depend on it either.
//
// Bound by HBM: 28 bytes a value with fp32 gradients and moments, 16 with 8-bit moments.

#include "fmb_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace fmb {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBlock = FMB_ADAMW_BLOCK;
constexpr int kBlocksPerWarp = 2;
constexpr int kCtaBlocks = kWarps * kBlocksPerWarp;
constexpr int kMaxTensors = 400;

struct Entry {
    float* p;
    const void* g;
    void* copy;
    long long values, block;
    int cta_begin;               // first CTA of this tensor
    int wide;                    // every array of the tensor may be read four values at a time
};

struct Table {
    Entry entry[kMaxTensors];
    int count;
    int advance;                 // the last launch of a step counts it
    int copy_type;
    float decay, lr, b1, c1, b2, c2, eps;
    double beta1, beta2;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    double* state;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename T> __device__ __forceinline__ void load_four(const T* p, float (&out)[4]) {
    if constexpr (sizeof(T) == 4) {
        const float4 q = *reinterpret_cast<const float4*>(p);
        out[0] = q.x; out[1] = q.y; out[2] = q.z; out[3] = q.w;
    } else {
        const uint2 q = *reinterpret_cast<const uint2*>(p);
        const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = to_float(e[i]);
    }
}

__device__ __forceinline__ void decode_four(uint32_t codes, float scale, float (&out)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * i)), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        out[2 * i] = __fmul_rn(f.x, scale);
        out[2 * i + 1] = __fmul_rn(f.y, scale);
    }
}

// largest magnitude of the warp's values; a NaN counts as larger than everything
__device__ __forceinline__ float warp_largest(const float (&a)[4], const float (&b)[4]) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        top = max(top, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
    return __uint_as_float(__reduce_max_sync(0xffffffffu, top));
}

// scale of a block: its largest value becomes 448; blocks of zeros and of the tiniest numbers have a scale all the same
__device__ __forceinline__ float block_scale(float largest) {
    const float s = __fdiv_rn(largest, 448.0f);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

template <bool KEEP>
__device__ __forceinline__ uint32_t encode_four(const float (&x)[4], float scale) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 q = make_float2(__fdiv_rn(x[2 * i], scale), __fdiv_rn(x[2 * i + 1], scale));
        uint32_t two = __nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, __NV_E4M3);
        if constexpr (KEEP) {
            if (x[2 * i] > 0.0f && (two & 0xffu) == 0) two |= 1u;
            if (x[2 * i + 1] > 0.0f && (two >> 8) == 0) two |= 0x100u;
        }
        out |= two << (16 * i);
    }
    return out;
}

template <typename G, bool EIGHT>
__global__ void __launch_bounds__(kThreads)
k_adamw(const __grid_constant__ Table t) {
    __shared__ float corrections[2];
    // the tensor of this CTA: the last one that begins at or before it
    int low = 0, high = t.count - 1;
    while (low < high) {
        const int mid = (low + high + 1) >> 1;
        if (t.entry[mid].cta_begin <= (int)blockIdx.x) low = mid; else high = mid - 1;
    }
    const Entry e = t.entry[low];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        corrections[0] = (float)(1.0 / (1.0 - t.state[1] * t.beta1));
        corrections[1] = (float)(1.0 / sqrt(1.0 - t.state[2] * t.beta2));
    }
    __syncthreads();
    const float step = t.lr * corrections[0], root_scale = corrections[1];
    const G* const grad = (const G*)e.g;
    const long long first = ((long long)(blockIdx.x - e.cta_begin) * kCtaBlocks + warp) * kBlock;
#pragma unroll 1
    for (int b = 0; b < kBlocksPerWarp; ++b) {
        const long long at = first + (long long)b * kWarps * kBlock;
        if (at >= e.values) break;
        const long long block = e.block + at / kBlock, moment = block * kBlock;
        const bool whole = e.wide && at + kBlock <= e.values;
        float p[2][4], g[2][4], m[2][4], v[2][4];
        float ms = 0.0f, vs = 0.0f;
        if constexpr (EIGHT) {
            ms = t.m_scale[block];
            vs = t.v_scale[block];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = h * 128 + lane * 4;
            if constexpr (EIGHT) {
                const uint32_t mc = *reinterpret_cast<const uint32_t*>((const uint8_t*)t.m + moment + i);
                const uint32_t vc = *reinterpret_cast<const uint32_t*>((const uint8_t*)t.v + moment + i);
                decode_four(mc, ms, m[h]);
                decode_four(vc, vs, v[h]);
            } else {
                load_four((const float*)t.m + moment + i, m[h]);
                load_four((const float*)t.v + moment + i, v[h]);
            }
            if (whole) {
                load_four((const float*)e.p + at + i, p[h]);
                load_four(grad + at + i, g[h]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool live = at + i + j < e.values;
                    p[h][j] = live ? e.p[at + i + j] : 0.0f;
                    g[h][j] = live ? to_float(grad[at + i + j]) : 0.0f;
                    if (!live) m[h][j] = v[h][j] = 0.0f;
                }
            }
        }
        float root[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (EIGHT) v[h][j] = __fmul_rn(v[h][j], v[h][j]);
                const float gr = g[h][j];
                m[h][j] = __fadd_rn(__fmul_rn(m[h][j], t.b1), __fmul_rn(gr, t.c1));
                v[h][j] = __fadd_rn(__fmul_rn(v[h][j], t.b2), __fmul_rn(__fmul_rn(gr, t.c2), gr));
                root[h][j] = __fsqrt_rn(v[h][j]);
                p[h][j] = p[h][j] * t.decay - __fdividef(m[h][j] * step, root[h][j] * root_scale + t.eps);
            }
        if constexpr (EIGHT) {
            const float new_ms = block_scale(warp_largest(m[0], m[1])), new_vs = block_scale(warp_largest(root[0], root[1]));
            if (lane == 0) {
                t.m_scale[block] = new_ms;
                t.v_scale[block] = new_vs;
            }
            ms = new_ms;
            vs = new_vs;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = h * 128 + lane * 4;
            if constexpr (EIGHT) {
                *reinterpret_cast<uint32_t*>((uint8_t*)t.m + moment + i) = encode_four<false>(m[h], ms);
                *reinterpret_cast<uint32_t*>((uint8_t*)t.v + moment + i) = encode_four<true>(root[h], vs);
            } else {
                *reinterpret_cast<float4*>((float*)t.m + moment + i) = make_float4(m[h][0], m[h][1], m[h][2], m[h][3]);
                *reinterpret_cast<float4*>((float*)t.v + moment + i) = make_float4(v[h][0], v[h][1], v[h][2], v[h][3]);
            }
            uint32_t half_bits[2] = {0, 0};
            if (e.copy) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    if (t.copy_type == FMB_TYPE_BF16) {
                        const __nv_bfloat162 two = __floats2bfloat162_rn(p[h][2 * q], p[h][2 * q + 1]);
                        half_bits[q] = *reinterpret_cast<const uint32_t*>(&two);
                    } else {
                        const __half2 two = __floats2half2_rn(p[h][2 * q], p[h][2 * q + 1]);
                        half_bits[q] = *reinterpret_cast<const uint32_t*>(&two);
                    }
                }
            }
            if (whole) {
                *reinterpret_cast<float4*>(e.p + at + i) = make_float4(p[h][0], p[h][1], p[h][2], p[h][3]);
                if (e.copy) *reinterpret_cast<uint2*>((uint16_t*)e.copy + at + i) = make_uint2(half_bits[0], half_bits[1]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at + i + j < e.values) {
                        e.p[at + i + j] = p[h][j];
                        if (e.copy) ((uint16_t*)e.copy)[at + i + j] = (uint16_t)(half_bits[j >> 1] >> (16 * (j & 1)));
                    }
            }
        }
    }
    if (!t.advance) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        // every CTA has read the step before it counts itself done
        unsigned* const done = reinterpret_cast<unsigned*>(t.state + 3);
        __threadfence();
        if (atomicAdd(done, 1u) == gridDim.x - 1) {
            *done = 0;
            t.state[0] += 1.0;
            t.state[1] *= t.beta1;
            t.state[2] *= t.beta2;
        }
    }
}

template <typename G>
int launch(const Table& t, int ctas, bool eight, cudaStream_t stream) {
    if (eight) k_adamw<G, true><<<ctas, kThreads, 0, stream>>>(t);
    else k_adamw<G, false><<<ctas, kThreads, 0, stream>>>(t);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

}  // namespace

}  // namespace fmb

using namespace fmb;

extern "C" FMB_API int fmb_adamw_step(const fmb_adamw_t* a, const fmb_adamw_tensor_t* tensors, int count, fmb_stream_t stream) {
    FMB_REQUIRE(a && (count == 0 || tensors) && count >= 0, "fmb_adamw_step: null argument");
    FMB_REQUIRE(a->moment_bits == 32 || a->moment_bits == 8, "fmb_adamw_step: moments of 32 or 8 bits");
    FMB_REQUIRE(a->grad_type >= FMB_TYPE_F32 && a->grad_type <= FMB_TYPE_F16, "fmb_adamw_step: gradient type");
    FMB_REQUIRE(a->m && a->v && a->state, "fmb_adamw_step: null moments or state");
    FMB_REQUIRE(aligned(a->m, 16) && aligned(a->v, 16), "fmb_adamw_step: moments start at a multiple of 16 bytes");
    FMB_REQUIRE(a->moment_bits == 32 || (a->m_scale && a->v_scale), "fmb_adamw_step: 8-bit moments need their scales");
    FMB_REQUIRE(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0, "fmb_adamw_step: betas in [0, 1)");
    const int grad_bytes = a->grad_type == FMB_TYPE_F32 ? 4 : 2;
    int last = -1;
    for (int i = 0; i < count; ++i) {
        if (!tensors[i].g || tensors[i].values == 0) continue;
        FMB_REQUIRE(tensors[i].p && tensors[i].values > 0 && tensors[i].block >= 0, "fmb_adamw_step: bad tensor");
        FMB_REQUIRE(aligned(tensors[i].p, 4) && aligned(tensors[i].g, grad_bytes) && aligned(tensors[i].copy, 2),
                    "fmb_adamw_step: a pointer is not aligned to its type");
        FMB_REQUIRE(!tensors[i].copy || a->copy_type == FMB_TYPE_BF16 || a->copy_type == FMB_TYPE_F16, "fmb_adamw_step: copy type");
        last = i;
    }
    if (last < 0) return FMB_OK;
    Table t;
    t.copy_type = a->copy_type;
    t.decay = (float)(1.0 - a->lr * a->weight_decay);
    t.lr = (float)a->lr;
    t.b1 = (float)a->beta1; t.c1 = (float)(1.0 - a->beta1);
    t.b2 = (float)a->beta2; t.c2 = (float)(1.0 - a->beta2);
    t.eps = (float)a->eps;
    t.beta1 = a->beta1; t.beta2 = a->beta2;
    t.m = a->m; t.v = a->v; t.m_scale = a->m_scale; t.v_scale = a->v_scale; t.state = a->state;
    t.count = 0;
    long long ctas = 0;
    for (int i = 0; i <= last; ++i) {
        const fmb_adamw_tensor_t& s = tensors[i];
        if (!s.g || s.values == 0) continue;
        Entry& e = t.entry[t.count++];
        e.p = s.p; e.g = s.g; e.copy = s.copy; e.values = s.values; e.block = s.block;
        e.cta_begin = (int)ctas;
        e.wide = aligned(s.p, 16) && aligned(s.g, 4 * grad_bytes) && aligned(s.copy, 8);
        ctas += (s.values + (long long)kCtaBlocks * kBlock - 1) / ((long long)kCtaBlocks * kBlock);
        FMB_REQUIRE(ctas < (1ll << 31), "fmb_adamw_step: too many values");
        if (t.count == kMaxTensors || i == last) {
            t.advance = i == last;
            const bool eight = a->moment_bits == 8;
            const int rc = a->grad_type == FMB_TYPE_F32    ? launch<float>(t, (int)ctas, eight, (cudaStream_t)stream)
                           : a->grad_type == FMB_TYPE_BF16 ? launch<__nv_bfloat16>(t, (int)ctas, eight, (cudaStream_t)stream)
                                                           : launch<__half>(t, (int)ctas, eight, (cudaStream_t)stream);
            if (rc) return rc;
            t.count = 0;
            ctas = 0;
        }
    }
    return FMB_OK;
}
