// Rows between the forward and the backward pass in 8 bits (held.cuh), and the gate of an expert's two matrices with them:
//
//   hold:     codes and exponents of x
//   gate:     u = (a | b), h = silu(a) b, and u held on the way
//   gradient: da = dh b s (1 + a (1 - s)), db = dh a s with s = 1 / (1 + exp(-a)), from held u (or u itself), and h anew
//   release:  x read back
//
// One pass each, bound by memory. A lane has eight neighbouring columns (16 bytes of a 16-bit type), four lanes a block of 32; where rows
// do not start at multiples of eight values it has one column, and a warp a block. The largest of a block is a maximum over those
// lanes, so the codes leave in the pass that reads the values. The arithmetic is in fp32 and every result is rounded once.

#include "held.cuh"

#include <algorithm>

namespace fmb {
namespace held {

namespace {

constexpr int kThreads = 256;

template <typename T, int N> struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack { T v[N]; };

// A CTA's threads by rows: `lanes` (a power of two, whole blocks) for the columns of one, 256 / lanes rows at a time.
struct Grid {
    int lanes, width, columns, parts;            // width: of a part
};

template <typename T, int N>
__device__ __forceinline__ void load(const T* __restrict__ at, int live, float (&x)[N]) {
    if (live >= N) {
        const Pack<T, N> in = *reinterpret_cast<const Pack<T, N>*>(at);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = to_float(in.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i < live ? to_float(at[i]) : 0.0f;
    }
}

template <typename T, int N>
__device__ __forceinline__ void store(T* __restrict__ at, int live, const float (&x)[N]) {
    if (live >= N) {
        Pack<T, N> out;
#pragma unroll
        for (int i = 0; i < N; ++i) out.v[i] = rounded<T>(x[i]);
        *reinterpret_cast<Pack<T, N>*>(at) = out;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < live) at[i] = rounded<T>(x[i]);
    }
}

// Codes of this lane's values and the block's exponent, by all lanes of the warp; `live` of the values exist, the others are zero.
template <typename T, int N>
__device__ __forceinline__ void hold(const float (&x)[N], int live, bool block_exists, uint8_t* __restrict__ codes, uint8_t* __restrict__ exponent) {
    constexpr int kLanes = kBlock / N;
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t bits = __float_as_uint(x[i]) & 0x7fffffffu;
        if (bits < 0x7f800000u) largest = max(largest, bits);
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    // largest = m 2^E: 448 = 1.75 x 2^8 units hold it at e = E - 8 where m <= 1.75
    const int e = min(max((int)((largest + 0x1fffffu) >> 23) - kBias - 8, Units<T>::kLowest), Units<T>::kHighest);
    const float inverse = unit_of(kBias - e), most = e == Units<T>::kHighest ? 240.0f : 448.0f;
    uint32_t out[(N + 3) / 4];
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        float v[2];
        uint32_t nan = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float value = i + j < N ? x[i + j] : 0.0f;
            if ((__float_as_uint(value) & 0x7fffffffu) >= 0x7f800000u) nan |= 0x7fu << (8 * j);
            v[j] = fminf(fmaxf(value * inverse, -most), most);
        }
        const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3) | nan;
        if (i % 4 == 0) out[i / 4] = two; else out[i / 4] |= two << 16;
    }
    if (live >= N && N == 8) {
        *reinterpret_cast<uint2*>(codes) = make_uint2(out[0], out[(N + 3) / 4 - 1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < live) codes[i] = (uint8_t)(out[i / 4] >> (8 * (i % 4)));
    }
    if (block_exists && (threadIdx.x & (kLanes - 1)) == 0) *exponent = (uint8_t)(e + kBias);
}

template <int N>
__device__ __forceinline__ void release(const uint8_t* __restrict__ codes, int live, int byte, float (&x)[N]) {
    const float unit = unit_of(byte);
    uint32_t in[(N + 3) / 4] = {};
    if (live >= N && N == 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(codes);
        in[0] = v.x;
        in[(N + 3) / 4 - 1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < live) in[i / 4] |= (uint32_t)codes[i] << (8 * (i % 4));
    }
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 v = two_values(in[i / 4] >> (8 * (i % 4)));
        x[i] = v.x * unit;
        if (i + 1 < N) x[i + 1] = v.y * unit;
    }
}

// Rows of this thread, the same number for all threads of a CTA, and columns of each: what is past the last has none to load or store.
template <typename F>
__device__ __forceinline__ void walk(const Grid& g, long long rows, int n, F body) {
    const int per_cta = kThreads / g.lanes, part = threadIdx.x & (g.lanes - 1), whole = blocks_of(g.width) * kBlock;
    for (long long r0 = (long long)blockIdx.x * per_cta; r0 < rows; r0 += (long long)gridDim.x * per_cta) {
        const long long r = r0 + threadIdx.x / g.lanes;
        for (int c0 = 0; c0 < whole; c0 += g.lanes * n) {
            const int c = c0 + part * n;
            const bool exists = r < rows && c < whole;
            body(r, c, exists ? g.width - c : 0, exists);
        }
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
k_hold(fmb_held_t a, Grid g) {
    const int blocks = blocks_of(g.width);
    walk(g, (long long)a.rows * g.parts, N, [&](long long r, int c, int live, bool exists) {
        const long long row = g.parts == 2 ? r >> 1 : r;
        const int first = g.parts == 2 && (r & 1) ? g.width : 0;
        float v[N];
        load<T, N>((const T*)a.x + row * a.x_stride + first + c, live, v);
        hold<T, N>(v, live, exists, a.codes + row * a.columns + first + c, a.exponents + r * blocks + c / kBlock);
    });
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
k_release(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, int rows, int columns, T* __restrict__ out,
          long long stride, Grid g) {
    const int blocks = blocks_of(g.width);
    walk(g, (long long)rows * g.parts, N, [&](long long r, int c, int live, bool exists) {
        if (!exists) return;
        const long long row = g.parts == 2 ? r >> 1 : r;
        const int first = g.parts == 2 && (r & 1) ? g.width : 0;
        float v[N];
        release<N>(codes + row * columns + first + c, live, exponents[r * blocks + c / kBlock], v);
        store<T, N>(out + row * stride + first + c, live, v);
    });
}

// 1 / (1 + exp(-x)): in float32 to its last bits; where results have 16 bits, by the fast exponential and division
template <typename T> __device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }
template <> __device__ __forceinline__ float sigmoid<float>(float x) { return 1.0f / (1.0f + expf(-x)); }

template <typename T, int N, bool HOLD>
__global__ void __launch_bounds__(kThreads)
k_gate(fmb_held_t a, Grid g) {
    const int blocks = blocks_of(g.width);
    walk(g, a.rows, N, [&](long long r, int c, int live, bool exists) {
        const T* const u = (const T*)a.x + r * a.x_stride + c;
        float x[N], y[N], h[N];
        load<T, N>(u, live, x);
        load<T, N>(u + g.width, live, y);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = x[i] * sigmoid<T>(x[i]) * y[i];
        store<T, N>((T*)a.h + r * a.h_stride + c, live, h);
        if (HOLD) {
            uint8_t* const codes = a.codes + r * a.columns + c;
            uint8_t* const exponents = a.exponents + 2 * r * blocks + c / kBlock;
            hold<T, N>(x, live, exists, codes, exponents);
            hold<T, N>(y, live, exists, codes + g.width, exponents + blocks);
        }
    });
}

template <typename T, int N, bool HELD>
__global__ void __launch_bounds__(kThreads)
k_gate_gradient(fmb_held_t a, Grid g) {
    const int blocks = blocks_of(g.width);
    walk(g, a.rows, N, [&](long long r, int c, int live, bool exists) {
        if (!exists) return;
        float x[N], y[N], dh[N], h[N];
        load<T, N>((const T*)a.dh + r * a.dh_stride + c, live, dh);
        if (HELD) {
            const uint8_t* const codes = a.codes + r * a.columns + c;
            const uint8_t* const exponents = a.exponents + 2 * r * blocks + c / kBlock;
            release<N>(codes, live, exponents[0], x);
            release<N>(codes + g.width, live, exponents[blocks], y);
        } else {
            const T* const u = (const T*)a.x + r * a.x_stride + c;
            load<T, N>(u, live, x);
            load<T, N>(u + g.width, live, y);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float s = sigmoid<T>(x[i]), silu = x[i] * s;
            h[i] = silu * y[i];
            y[i] = dh[i] * y[i] * s * (1.0f + x[i] * (1.0f - s));
            x[i] = dh[i] * silu;
        }
        T* const du = (T*)a.du + r * a.du_stride + c;
        store<T, N>(du, live, y);
        store<T, N>(du + g.width, live, x);
        if (a.h) store<T, N>((T*)a.h + r * a.h_stride + c, live, h);
    });
}

bool by_eight(const void* base, long long stride, int bytes) {
    return ((uintptr_t)base & (uintptr_t)(std::min(16, 8 * bytes) - 1)) == 0 && stride % 8 == 0;
}

Grid grid_of(int columns, int parts, int n) {
    Grid g;
    g.columns = columns;
    g.parts = parts;
    g.width = columns / parts;
    g.lanes = kBlock / n;
    while (g.lanes < kThreads && g.lanes * n < g.width) g.lanes *= 2;
    return g;
}

unsigned ctas(const Grid& g, long long rows) { return (unsigned)std::min<long long>((rows + kThreads / g.lanes - 1) / (kThreads / g.lanes), 1 << 20); }

struct Launch {
    const fmb_held_t& a;
    bool wide;
    cudaStream_t stream;

    template <typename T, int N>
    void go(int what) const {
        const Grid g = grid_of(a.columns, what == 0 ? a.parts : 2, N);
        const long long rows = (long long)a.rows * (what == 0 ? a.parts : 1);
        if (what == 0) k_hold<T, N><<<ctas(g, rows), kThreads, 0, stream>>>(a, g);
        else if (what == 1 && a.codes) k_gate<T, N, true><<<ctas(g, rows), kThreads, 0, stream>>>(a, g);
        else if (what == 1) k_gate<T, N, false><<<ctas(g, rows), kThreads, 0, stream>>>(a, g);
        else if (a.codes) k_gate_gradient<T, N, true><<<ctas(g, rows), kThreads, 0, stream>>>(a, g);
        else k_gate_gradient<T, N, false><<<ctas(g, rows), kThreads, 0, stream>>>(a, g);
    }
    template <typename T> void typed(int what) const { wide ? go<T, 8>(what) : go<T, 1>(what); }

    int operator()(int what) const {
        if (a.type == FMB_TYPE_F32) typed<float>(what);
        else if (a.type == FMB_TYPE_BF16) typed<__nv_bfloat16>(what);
        else typed<__half>(what);
        FMB_LAUNCH_CHECK();
        return FMB_OK;
    }
};

int check(const fmb_held_t* a, int parts) {
    FMB_REQUIRE(a, "held rows: null argument");
    FMB_REQUIRE(a->type >= FMB_TYPE_F32 && a->type <= FMB_TYPE_F16, "held rows: type");
    FMB_REQUIRE(a->rows >= 0 && a->rows <= (1 << 30), "held rows: more than 2^30 rows");
    FMB_REQUIRE(a->columns >= 1 && a->columns <= (1 << 20), "held rows: 1 to 2^20 columns");
    FMB_REQUIRE((a->parts == 1 || a->parts == 2) && a->columns % a->parts == 0 && (!parts || a->parts == parts), "held rows: parts");
    FMB_REQUIRE(!a->codes == !a->exponents, "held rows: codes and exponents belong together");
    return FMB_OK;
}

// whether every matrix that is there can be taken eight values at a time
bool wide(const fmb_held_t& a) {
    const int bytes = a.type == FMB_TYPE_F32 ? 4 : 2;
    auto fits = [&](const void* base, long long stride) { return !base || by_eight(base, stride, bytes); };
    return a.columns / a.parts % 8 == 0 && fits(a.x, a.x_stride) && fits(a.h, a.h_stride) && fits(a.dh, a.dh_stride) && fits(a.du, a.du_stride) &&
           ((uintptr_t)a.codes & 7) == 0;
}

template <typename T>
void release_typed(const uint8_t* codes, const uint8_t* exponents, int rows, int columns, int parts, void* out, long long stride, cudaStream_t stream) {
    const bool eight = columns / parts % 8 == 0 && by_eight(out, stride, sizeof(T)) && ((uintptr_t)codes & 7) == 0;
    const Grid g = grid_of(columns, parts, eight ? 8 : 1);
    const long long all = (long long)rows * parts;
    if (eight) k_release<T, 8><<<ctas(g, all), kThreads, 0, stream>>>(codes, exponents, rows, columns, (T*)out, stride, g);
    else k_release<T, 1><<<ctas(g, all), kThreads, 0, stream>>>(codes, exponents, rows, columns, (T*)out, stride, g);
}

}  // namespace

int release(int type, const uint8_t* codes, const uint8_t* exponents, int rows, int columns, int parts, void* out, long long row_stride,
            cudaStream_t stream) {
    if (type == FMB_TYPE_F32) release_typed<float>(codes, exponents, rows, columns, parts, out, row_stride, stream);
    else if (type == FMB_TYPE_BF16) release_typed<__nv_bfloat16>(codes, exponents, rows, columns, parts, out, row_stride, stream);
    else release_typed<__half>(codes, exponents, rows, columns, parts, out, row_stride, stream);
    FMB_LAUNCH_CHECK();
    return FMB_OK;
}

}  // namespace held
}  // namespace fmb

using namespace fmb;
using namespace fmb::held;

extern "C" FMB_API int fmb_hold_rows(const fmb_held_t* a, fmb_stream_t stream) {
    const int rc = check(a, 0);
    if (rc || a->rows == 0) return rc;
    FMB_REQUIRE(a->x && a->codes, "fmb_hold_rows: null argument");
    FMB_REQUIRE(a->rows == 1 || a->x_stride >= a->columns, "fmb_hold_rows: rows overlap");
    fmb_held_t own = *a;
    own.h = own.du = nullptr;
    own.dh = nullptr;
    return Launch{own, wide(own), (cudaStream_t)stream}(0);
}

extern "C" FMB_API int fmb_release_rows(const fmb_held_t* a, fmb_stream_t stream) {
    const int rc = check(a, 0);
    if (rc || a->rows == 0) return rc;
    FMB_REQUIRE(a->h && a->codes, "fmb_release_rows: null argument");
    FMB_REQUIRE(a->rows == 1 || a->h_stride >= a->columns, "fmb_release_rows: rows overlap");
    return release(a->type, a->codes, a->exponents, a->rows, a->columns, a->parts, a->h, a->h_stride, (cudaStream_t)stream);
}

extern "C" FMB_API int fmb_gated_rows(const fmb_held_t* a, fmb_stream_t stream) {
    const int rc = check(a, 2);
    if (rc || a->rows == 0) return rc;
    FMB_REQUIRE(a->x && a->h, "fmb_gated_rows: null argument");
    FMB_REQUIRE(a->rows == 1 || (a->x_stride >= a->columns && a->h_stride >= a->columns / 2), "fmb_gated_rows: rows overlap");
    fmb_held_t own = *a;
    own.du = nullptr;
    own.dh = nullptr;
    return Launch{own, wide(own), (cudaStream_t)stream}(1);
}

extern "C" FMB_API int fmb_gated_rows_gradient(const fmb_held_t* a, fmb_stream_t stream) {
    const int rc = check(a, 2);
    if (rc || a->rows == 0) return rc;
    FMB_REQUIRE((a->codes || a->x) && a->dh && a->du, "fmb_gated_rows_gradient: null argument");
    FMB_REQUIRE(!(a->codes && a->x), "fmb_gated_rows_gradient: rows or what is held of them, not both");
    FMB_REQUIRE(a->rows == 1 || ((!a->x || a->x_stride >= a->columns) && a->dh_stride >= a->columns / 2 && a->du_stride >= a->columns &&
                                 (!a->h || a->h_stride >= a->columns / 2)), "fmb_gated_rows_gradient: rows overlap");
    return Launch{*a, wide(*a), (cudaStream_t)stream}(2);
}
