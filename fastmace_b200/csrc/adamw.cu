// AdamW over a list of tensors in one launch (more only beyond kMaxTensors): weights, gradients and moments pass once.
//
// The list travels as a kernel argument, so nothing is uploaded and a captured step replays by itself; the number of the
// step is a device counter that the last CTA to finish advances. A warp takes a block of 256 values, two float4 per lane and
// array. With moments in 8 bits the block shares a scale per moment: first moments are held as e4m3 of m / s, second
// moments as e4m3 of sqrt(v) / s, s = (largest of the block) / 448. Relative steps of 2^-4 over 2^15 and the root's smaller
// range keep the quotient m / sqrt(v) of one step to a few per cent of itself; a v that is not zero is never held as zero, which would
// make the next quotient m / eps. Over many steps that is not enough: with beta2 = 0.999 a root moves by 0.05 % a step downwards and
// codes are 6 to 12 % apart, so that rounded to the nearest a code stays and the value follows its block's largest instead of its own
// gradients. Held at random (Table::random), as the code below or above with the chances that make the expected v the exact one, it follows
// its moving average: the expectation of v is that of fp32 at every step, and its root spreads about that by a sixth, which codes a
// twelfth apart and a memory of 2,000 steps make. The bits are Philox's, of the step, the place of the value and a key, 16 a
// value. First moments move by a tenth a step and are rounded to the nearest. Arithmetic is in fp32, and
// that of the moments is rounded operation by operation, as it is written here: a moment that came out a bit
// apart could take the next code, 2^-4 away, and with the block's largest the scale would follow a step later.
//
// Bound by HBM: 28 bytes a value with fp32 gradients and moments, 16 with 8-bit moments. 200 M values in 32 bits with bf16 copies
// take 910 us (6.6 TB/s, what a copy of as many bytes reaches), 64 M in 8 bits with bf16 gradients and copies 207 (5.0 TB/s: 24 warps'
// conversions and exact quotients an SM keep it at 74 % of its rate), the 43 tensors of a medium model 27 (4.7 M values, 131 MB).

#include "fmb_common.cuh"
#include "philox.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

namespace fmb {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBlock = FMB_ADAMW_BLOCK;
constexpr int kCtaBlocks = 16;
constexpr int kMaxTensors = 400, kFewTensors = 64;        // of a launch: the list is 56 bytes a tensor of kernel arguments

struct Entry {
    float* p;
    const void* g;
    void* copy;
    long long values, block;
    long long first;             // first block of this tensor among those of the launch
    int wide;                    // every array of the tensor may be read four values at a time
};

template <int CAPACITY>
struct Table {
    Entry entry[CAPACITY];
    int count;
    int advance;                 // the last launch of a step counts it
    int copy_type;
    uint32_t random;             // 8 bits: key of the random rounding of second moments
    long long blocks;            // of the launch
    float decay, lr, b1, c1, b2, c2, eps;
    double beta1, beta2;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    double* state;
};

static_assert(sizeof(Entry) == 56 && sizeof(Table<kMaxTensors>) <= 32764, "fits what a kernel takes as arguments");

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename G> __device__ __forceinline__ G zero_of() { return G(0.0f); }

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
    const float s = __fmul_rn(largest, 1.0f / 448.0f);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

// x / scale from the rounded inverse of the scale, the quotient corrected by its residual (Markstein, 1990)
__device__ __forceinline__ float quotient(float x, float scale, float inverse) {
    const float q = __fmul_rn(x, inverse);
    return fmaf(fmaf(-q, scale, x), inverse, q);
}

// code of x / scale for x >= 0: the number of the type below q or the one above, which has the chance (q^2 - below^2) / (above^2 - below^2).
// Below 2^-6 the numbers are 2^-9 apart, as they are between 2^-6 and 2^-5, and q moves there.
__device__ __forceinline__ float either(float q, uint32_t bits) {
    const float u = (float)bits * (1.0f / 65536.0f) + (0.5f / 65536.0f), base = q < 0x1p-6f ? 0x1p-6f : 0.0f;
    const uint32_t cut = __float_as_uint(q + base) & 0xfff00000u;
    const float below = __uint_as_float(cut) - base, above = __uint_as_float(cut + 0x00100000u) - base;
    return u * ((above - below) * (above + below)) < (q - below) * (q + below) ? above : below;
}
__device__ __forceinline__ uint32_t encode_four_either(const float (&x)[4], float scale, float inverse, uint32_t bits_low, uint32_t bits_high) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t bits = i ? bits_high : bits_low;
        const float2 q = make_float2(either(quotient(x[2 * i], scale, inverse), bits & 0xffffu), either(quotient(x[2 * i + 1], scale, inverse), bits >> 16));
        uint32_t two = __nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, __NV_E4M3);
        if (x[2 * i] > 0.0f && (two & 0xffu) == 0) two |= 1u;
        if (x[2 * i + 1] > 0.0f && (two >> 8) == 0) two |= 0x100u;
        out |= two << (16 * i);
    }
    return out;
}

// codes of x / scale; KEEP: what is positive does not become zero
template <bool KEEP>
__device__ __forceinline__ uint32_t encode_four(const float (&x)[4], float scale, float inverse) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 q = make_float2(quotient(x[2 * i], scale, inverse), quotient(x[2 * i + 1], scale, inverse));
        uint32_t two = __nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, __NV_E4M3);
        if constexpr (KEEP) {
            if (x[2 * i] > 0.0f && (two & 0xffu) == 0) two |= 1u;
            if (x[2 * i + 1] > 0.0f && (two >> 8) == 0) two |= 0x100u;
        }
        out |= two << (16 * i);
    }
    return out;
}

// What a warp reads of a block: two times four values per lane of every array, as they are held.
template <typename G, bool EIGHT>
struct Raw {
    using Four = typename std::conditional<sizeof(G) == 4, float4, uint2>::type;
    using Moment = typename std::conditional<EIGHT, uint32_t, float4>::type;
    float4 p[2];
    Four g[2];
    Moment m[2], v[2];
    float m_scale, v_scale;
    int entry;                   // of the table
    long long at;                // first value of the block in its tensor
    bool whole;
};

template <typename G, bool EIGHT, int CAPACITY>
__device__ __forceinline__ void load_block(const Table<CAPACITY>& t, long long b, int& entry, Raw<G, EIGHT>& r) {
    const int lane = threadIdx.x & 31;
    while (entry + 1 < t.count && t.entry[entry + 1].first <= b) ++entry;
    const Entry& e = t.entry[entry];
    r.entry = entry;
    r.at = (b - e.first) * kBlock;
    r.whole = e.wide && r.at + kBlock <= e.values;
    const long long moment = e.block * kBlock + r.at;
    if constexpr (EIGHT) {
        r.m_scale = t.m_scale[e.block + r.at / kBlock];
        r.v_scale = t.v_scale[e.block + r.at / kBlock];
    }
    using Moment = typename Raw<G, EIGHT>::Moment;
    constexpr int kHeld = EIGHT ? 1 : 4;                 // bytes of a moment
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = h * 128 + lane * 4;
        r.m[h] = *reinterpret_cast<const Moment*>((const uint8_t*)t.m + (moment + i) * kHeld);
        r.v[h] = *reinterpret_cast<const Moment*>((const uint8_t*)t.v + (moment + i) * kHeld);
        if (r.whole) {
            r.p[h] = *reinterpret_cast<const float4*>(e.p + r.at + i);
            r.g[h] = *reinterpret_cast<const typename Raw<G, EIGHT>::Four*>((const G*)e.g + r.at + i);
        } else {
            float* const p = reinterpret_cast<float*>(&r.p[h]);
            G* const g = reinterpret_cast<G*>(&r.g[h]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool live = r.at + i + j < e.values;
                p[j] = live ? e.p[r.at + i + j] : 0.0f;
                g[j] = live ? ((const G*)e.g)[r.at + i + j] : zero_of<G>();
            }
        }
    }
}

template <typename G, bool EIGHT, bool RANDOM, int CAPACITY>
__device__ __forceinline__ void step_block(const Table<CAPACITY>& t, const Raw<G, EIGHT>& r, float step, float root_scale, uint32_t number) {
    const int lane = threadIdx.x & 31;
    const Entry& e = t.entry[r.entry];
    const long long block = e.block + r.at / kBlock, moment = block * kBlock;
    float p[2][4], m[2][4], v[2][4], root[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float* const rp = reinterpret_cast<const float*>(&r.p[h]);
        const G* const rg = reinterpret_cast<const G*>(&r.g[h]);
        if constexpr (EIGHT) {
            decode_four(r.m[h], r.m_scale, m[h]);
            decode_four(r.v[h], r.v_scale, v[h]);
        } else {
            const float* const rm = reinterpret_cast<const float*>(&r.m[h]);
            const float* const rv = reinterpret_cast<const float*>(&r.v[h]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                m[h][j] = rm[j];
                v[h][j] = rv[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!r.whole && r.at + h * 128 + lane * 4 + j >= e.values) m[h][j] = v[h][j] = 0.0f;
            if constexpr (EIGHT) v[h][j] = __fmul_rn(v[h][j], v[h][j]);
            const float gr = to_float(rg[j]);
            m[h][j] = __fadd_rn(__fmul_rn(m[h][j], t.b1), __fmul_rn(gr, t.c1));
            v[h][j] = __fadd_rn(__fmul_rn(v[h][j], t.b2), __fmul_rn(__fmul_rn(gr, t.c2), gr));
            root[h][j] = __fsqrt_rn(v[h][j]);
            p[h][j] = rp[j] * t.decay - __fdividef(m[h][j] * step, root[h][j] * root_scale + t.eps);
        }
    }
    float ms = 1.0f, vs = 1.0f, m_inverse = 1.0f, v_inverse = 1.0f;
    if constexpr (EIGHT) {
        ms = block_scale(warp_largest(m[0], m[1]));
        vs = block_scale(warp_largest(root[0], root[1]));
        if (lane == 0) {
            t.m_scale[block] = ms;
            t.v_scale[block] = vs;
        }
        m_inverse = __fdiv_rn(1.0f, ms);
        v_inverse = __fdiv_rn(1.0f, vs);
    }
    uint32_t bits[4];
    if constexpr (RANDOM) {
        const unsigned long long at = block * 32 + lane;
        bits[0] = (uint32_t)at; bits[1] = (uint32_t)(at >> 32); bits[2] = number; bits[3] = 0x61646d77u;
        philox(bits, t.random, 0x6d616365u);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = h * 128 + lane * 4;
        if constexpr (EIGHT) {
            *reinterpret_cast<uint32_t*>((uint8_t*)t.m + moment + i) = encode_four<false>(m[h], ms, m_inverse);
            *reinterpret_cast<uint32_t*>((uint8_t*)t.v + moment + i) =
                RANDOM ? encode_four_either(root[h], vs, v_inverse, bits[2 * h], bits[2 * h + 1]) : encode_four<true>(root[h], vs, v_inverse);
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
        if (r.whole) {
            *reinterpret_cast<float4*>(e.p + r.at + i) = make_float4(p[h][0], p[h][1], p[h][2], p[h][3]);
            if (e.copy) *reinterpret_cast<uint2*>((uint16_t*)e.copy + r.at + i) = make_uint2(half_bits[0], half_bits[1]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r.at + i + j < e.values) {
                    e.p[r.at + i + j] = p[h][j];
                    if (e.copy) ((uint16_t*)e.copy)[r.at + i + j] = (uint16_t)(half_bits[j >> 1] >> (16 * (j & 1)));
                }
        }
    }
}

// Moments in 8 bits: as many CTAs as the device holds, whose warps take blocks in turn, so that the whole GPU is at one place of every
// array; in 32 bits, where a block has twice the bytes to wait for, CTAs of 16 blocks that come and go (200 M values 906 us against
// 990; the other way round 64 M values in 8 bits 220 against 330). With 8 bits a warp asks for its next block before it works on
// the one it has; with 32 the registers that takes cost more warps than it gains (1,070 us). Random rounding takes the issue slots of ten
// rounds and two squares a value: 64 M values 298 us, 202 to the nearest.
template <typename G, bool EIGHT, bool RANDOM, int CAPACITY>
__global__ void __launch_bounds__(kThreads, EIGHT ? 3 : 4)          // 80 registers, 64: what the plain ones take by themselves
k_adamw(const __grid_constant__ Table<CAPACITY> t) {
    __shared__ float corrections[2];
    __shared__ uint32_t steps_before;
    const int warp = threadIdx.x >> 5;
    const long long begin = (long long)blockIdx.x * (EIGHT ? kWarps : kCtaBlocks);
    const long long end = EIGHT ? t.blocks : min(t.blocks, begin + kCtaBlocks), stride = EIGHT ? (long long)gridDim.x * kWarps : kWarps;
    long long b = begin + warp;
    int entry = 0, high = t.count - 1;
    while (entry < high) {
        const int mid = (entry + high + 1) >> 1;
        if (t.entry[mid].first <= b) entry = mid; else high = mid - 1;
    }
    Raw<G, EIGHT> raw;
    if (EIGHT && b < end) load_block<G, EIGHT, CAPACITY>(t, b, entry, raw);
    if (threadIdx.x == 0) {
        corrections[0] = (float)(1.0 / (1.0 - t.state[1] * t.beta1));
        corrections[1] = (float)(1.0 / sqrt(1.0 - t.state[2] * t.beta2));
        if (RANDOM) steps_before = (uint32_t)(unsigned long long)t.state[0];
    }
    __syncthreads();
    const float step = t.lr * corrections[0], root_scale = corrections[1];
    const uint32_t number = RANDOM ? steps_before : 0;
#pragma unroll 1
    for (; b < end; b += stride) {
        if constexpr (EIGHT) {
            Raw<G, EIGHT> next;
            if (b + stride < end) load_block<G, EIGHT, CAPACITY>(t, b + stride, entry, next);
            step_block<G, EIGHT, RANDOM, CAPACITY>(t, raw, step, root_scale, number);
            raw = next;
        } else {
            load_block<G, EIGHT, CAPACITY>(t, b, entry, raw);
            step_block<G, EIGHT, RANDOM, CAPACITY>(t, raw, step, root_scale, number);
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

template <typename G, bool EIGHT, bool RANDOM, int CAPACITY>
int launch(const Table<CAPACITY>& t, cudaStream_t stream) {
    long long ctas = (t.blocks + kCtaBlocks - 1) / kCtaBlocks;
    if (EIGHT) {
        int dev = 0, sms = 0;
        static const int per_sm = [] {
            int n = 0;
            return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_adamw<G, EIGHT, RANDOM, CAPACITY>, kThreads, 0) == cudaSuccess && n > 0 ? n : 1;
        }();
        FMB_CUDA_CHECK(cudaGetDevice(&dev));
        FMB_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        ctas = std::min<long long>((t.blocks + kWarps - 1) / kWarps, (long long)per_sm * sms);
    }
    FMB_REQUIRE(ctas < (1ll << 31), "fmb_adamw_step: too many values");
    k_adamw<G, EIGHT, RANDOM, CAPACITY><<<(unsigned)ctas, kThreads, 0, stream>>>(t);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

template <typename G, int CAPACITY>
int launch(const Table<CAPACITY>& t, bool eight, cudaStream_t stream) {
    if (!eight) return launch<G, false, false, CAPACITY>(t, stream);
    return t.random ? launch<G, true, true, CAPACITY>(t, stream) : launch<G, true, false, CAPACITY>(t, stream);
}

bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

// the tensors up to `last` that have a gradient
template <int CAPACITY>
int step(const fmb_adamw_t* a, const fmb_adamw_tensor_t* tensors, int last, cudaStream_t stream) {
    const int grad_bytes = a->grad_type == FMB_TYPE_F32 ? 4 : 2;
    Table<CAPACITY> t;
    t.copy_type = a->copy_type;
    t.random = (uint32_t)a->random;
    t.decay = (float)(1.0 - a->lr * a->weight_decay);
    t.lr = (float)a->lr;
    t.b1 = (float)a->beta1; t.c1 = (float)(1.0 - a->beta1);
    t.b2 = (float)a->beta2; t.c2 = (float)(1.0 - a->beta2);
    t.eps = (float)a->eps;
    t.beta1 = a->beta1; t.beta2 = a->beta2;
    t.m = a->m; t.v = a->v; t.m_scale = a->m_scale; t.v_scale = a->v_scale; t.state = a->state;
    t.count = 0;
    t.blocks = 0;
    for (int i = 0; i <= last; ++i) {
        const fmb_adamw_tensor_t& s = tensors[i];
        if (!s.g || s.values == 0) continue;
        Entry& e = t.entry[t.count++];
        e.p = s.p; e.g = s.g; e.copy = s.copy; e.values = s.values; e.block = s.block;
        e.first = t.blocks;
        e.wide = aligned(s.p, 16) && aligned(s.g, 4 * grad_bytes) && aligned(s.copy, 8);
        t.blocks += (s.values + kBlock - 1) / kBlock;
        if (t.count == CAPACITY || i == last) {
            t.advance = i == last;
            const bool eight = a->moment_bits == 8;
            const int rc = a->grad_type == FMB_TYPE_F32    ? launch<float, CAPACITY>(t, eight, stream)
                           : a->grad_type == FMB_TYPE_BF16 ? launch<__nv_bfloat16, CAPACITY>(t, eight, stream)
                                                           : launch<__half, CAPACITY>(t, eight, stream);
            if (rc) return rc;
            t.count = 0;
            t.blocks = 0;
        }
    }
    return FMB_OK;
}

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
    FMB_REQUIRE(a->moment_bits == 8 || !a->random, "fmb_adamw_step: random rounding is of 8-bit moments");
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
    return last < kFewTensors ? step<kFewTensors>(a, tensors, last, (cudaStream_t)stream)
                              : step<kMaxTensors>(a, tensors, last, (cudaStream_t)stream);
}
