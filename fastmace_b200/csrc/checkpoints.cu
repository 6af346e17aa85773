// Rows between the forward and the backward pass in 8 bits (held.cuh), and the gate of an expert's two matrices with them:
//
//   hold:     codes and exponents of x
//   gate:     u = (a | b), h = silu(a) b, and u held on the way
//   gradient: da = dh b s (1 + a (1 - s)), db = dh a s with s = 1 / (1 + exp(-a)), from held u (or u itself), and h anew
//   release:  x read back
//
// One pass each, bound by memory. A lane has eight neighbouring columns (16 bytes of a 16-bit type), four lanes a block of 32; where rows
// do not start at multiples of eight values a lane has one column of each of four blocks, and a warp a block, so that it reads and writes
// side by side with the others. The largest of a block is a maximum over those lanes, so the codes leave in the pass that reads the
// values. The arithmetic is in fp32 and every result is rounded once.

#include "held.cuh"

#include <algorithm>
#include <type_traits>

namespace fmb {
namespace held {

namespace {

constexpr int kThreads = 256;

template <typename T, int N> struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack { T v[N]; };

// A CTA's threads by rows: `lanes` (a power of two, whole blocks) for the columns of one, 256 / lanes rows at a time.
struct Grid {
    int lanes, width, columns, parts;            // width: of a part
};

// A lane's N values as they are in memory, two to a word where they have 16 bits, so that what is on its way takes few registers
template <typename T, int N> struct Raw {
    static constexpr int kWords = (N * (int)sizeof(T) + 3) / 4;
    uint32_t v[kWords];
};

template <typename T, int N>
__device__ __forceinline__ Raw<T, N> load(const T* __restrict__ at, int live) {
    using R = Raw<T, N>;
    R in = {};
    if constexpr (N == 8) {
        if (live >= N) {
#pragma unroll
            for (int i = 0; i < R::kWords; i += 4) {
                const uint4 four = __ldg(reinterpret_cast<const uint4*>(at) + i / 4);
                in.v[i] = four.x; in.v[i + 1] = four.y; in.v[i + 2] = four.z; in.v[i + 3] = four.w;
            }
            return in;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i >= live) break;
        if constexpr (sizeof(T) == 4) in.v[i] = __ldg(reinterpret_cast<const uint32_t*>(at) + i);
        else in.v[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(at) + i) << (16 * (i % 2));
    }
    return in;
}

template <typename T, int N>
__device__ __forceinline__ void unpack(const Raw<T, N>& in, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t w = in.v[i * sizeof(T) / 4];
        if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) x[i] = __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
        else x[i] = __half2float(__ushort_as_half((uint16_t)(i % 2 ? w >> 16 : w & 0xffffu)));
    }
}

// the largest of |x|, as the bits of a float; NaN and infinities are larger than what is finite
template <typename T, int N>
__device__ __forceinline__ uint32_t largest_of(const Raw<T, N>& in) {
    uint32_t largest = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) largest = max(largest, in.v[i] & 0x7fffffffu);
        return largest;
    } else {
#pragma unroll
        for (int i = 0; i < Raw<T, N>::kWords; ++i) largest = __vmaxu2(largest, in.v[i] & 0x7fff7fffu);
        largest = max(largest >> 16, largest & 0xffffu);
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return largest << 16;
        else return __float_as_uint(__half2float(__ushort_as_half((uint16_t)largest)));
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
__device__ __forceinline__ void hold(const Raw<T, N>& raw, const float (&x)[N], int live, bool block_exists, uint8_t* __restrict__ codes,
                                     uint8_t* __restrict__ exponent) {
    constexpr int kLanes = kBlock / N;
    constexpr uint32_t kInfinity = 0x7f800000u;
    auto over_block = [](uint32_t v) {
        if constexpr (kLanes == 32) {
            return __reduce_max_sync(0xffffffffu, v);
        } else {
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
            return v;
        }
    };
    // largest = m 2^E: 448 = 1.75 x 2^8 units hold it at e = E - 8 where m <= 1.75
    auto exponent_of = [](uint32_t largest) { return min(max((int)((largest + 0x1fffffu) >> 23) - kBias - 8, Units<T>::kLowest), Units<T>::kHighest); };
    uint32_t largest = over_block(largest_of<T, N>(raw));
    int e = exponent_of(largest);
    uint32_t out[(N + 3) / 4];
    auto put = [&](int i, uint32_t two) {
        if (i % 4 == 0) out[i / 4] = two; else out[i / 4] |= two << 16;
    };
    // What is not finite does not count for the unit and is NaN; in the highest unit codes end at 240. Neither is met often.
    if (__any_sync(0xffffffffu, e == Units<T>::kHighest)) {
        largest = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t bits = __float_as_uint(x[i]) & 0x7fffffffu;
            if (bits < kInfinity) largest = max(largest, bits);
        }
        e = exponent_of(over_block(largest));
        const float inverse = unit_of(kBias - e), most = e == Units<T>::kHighest ? 240.0f : 448.0f;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float y = i + 1 < N ? x[i + 1 < N ? i + 1 : i] : 0.0f;
            uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(fminf(fmaxf(x[i] * inverse, -most), most), fminf(fmaxf(y * inverse, -most), most)), __NV_SATFINITE, __NV_E4M3);
            if ((__float_as_uint(x[i]) & 0x7fffffffu) >= kInfinity) two |= 0x7f;
            if ((__float_as_uint(y) & 0x7fffffffu) >= kInfinity) two |= 0x7f00;
            put(i, two);
        }
    } else {
        const float inverse = unit_of(kBias - e);
#pragma unroll
        for (int i = 0; i < N; i += 2)
            put(i, __nv_cvt_float2_to_fp8x2(make_float2(x[i] * inverse, i + 1 < N ? x[i + 1 < N ? i + 1 : i] * inverse : 0.0f), __NV_SATFINITE, __NV_E4M3));
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

// a lane's codes, and its values of them
template <int N> struct Codes {
    uint32_t v[(N + 3) / 4], byte;
};

template <int N>
__device__ __forceinline__ Codes<N> load_codes(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponent, int live) {
    Codes<N> in = {};
    if (live <= 0) return in;
    in.byte = __ldg(exponent);
    if (live >= N && N == 8) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(codes));
        in.v[0] = v.x;
        in.v[(N + 3) / 4 - 1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < live) in.v[i / 4] |= (uint32_t)__ldg(codes + i) << (8 * (i % 4));
    }
    return in;
}

template <int N>
__device__ __forceinline__ void release(const Codes<N>& in, float (&x)[N]) {
    const float unit = unit_of(in.byte);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 v = two_values(in.v[i / 4] >> (8 * (i % 4)));
        x[i] = v.x * unit;
        if (i + 1 < N) x[i + 1 < N ? i + 1 : i] = v.y * unit;
    }
}

// Places of a thread, whose loads are on their way together: N neighbouring columns of two rows, or one column of four blocks of a row
template <int N> constexpr int kPlaces = N == 1 ? 4 : 2;

struct Place {
    long long row;
    int column, live;                            // columns that exist from there on
    bool exists;                                 // the block does
};

// The same number of rounds for all threads of a CTA; what is past the last row or block has nothing to load or store.
template <int N, typename F>
__device__ __forceinline__ void walk(const Grid& g, long long rows, F body) {
    constexpr int kOfRow = N == 1 ? kPlaces<N> : 1, kRowsAtOnce = kPlaces<N> / kOfRow;
    const int per_cta = kThreads / g.lanes, whole = blocks_of(g.width) * kBlock;
    const int part = threadIdx.x & (g.lanes - 1), first = N == 1 ? part / 32 * 32 * kOfRow + part % 32 : part * N;
    for (long long r0 = (long long)blockIdx.x * per_cta * kRowsAtOnce; r0 < rows; r0 += (long long)gridDim.x * per_cta * kRowsAtOnce) {
        const long long r = r0 + threadIdx.x / g.lanes;
        for (int c0 = 0; c0 < whole; c0 += g.lanes * N * kOfRow) {
            if (N == 1 && c0 + first - part % 32 >= whole) continue;             // (the same for a warp)
            Place at[kPlaces<N>];
#pragma unroll
            for (int q = 0; q < kPlaces<N>; ++q) {
                at[q].row = r + (N == 1 ? 0 : q * per_cta);
                at[q].column = c0 + first + (N == 1 ? q * kBlock : 0);
                at[q].exists = at[q].row < rows && at[q].column < whole;
                at[q].live = at[q].exists ? g.width - at[q].column : 0;
            }
            body(at);
        }
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
k_hold(fmb_held_t a, Grid g) {
    const int blocks = blocks_of(g.width);
    walk<N>(g, (long long)a.rows * g.parts, [&](const Place (&at)[kPlaces<N>]) {
        auto row = [&](const Place& p) { return g.parts == 2 ? p.row >> 1 : p.row; };
        auto column = [&](const Place& p) { return (g.parts == 2 && (p.row & 1) ? g.width : 0) + p.column; };
        Raw<T, N> raw[kPlaces<N>];
#pragma unroll
        for (int q = 0; q < kPlaces<N>; ++q) raw[q] = load<T, N>((const T*)a.x + row(at[q]) * a.x_stride + column(at[q]), at[q].live);
#pragma unroll
        for (int q = 0; q < kPlaces<N>; ++q) {
            float x[N];
            unpack<T, N>(raw[q], x);
            hold<T, N>(raw[q], x, at[q].live, at[q].exists, a.codes + row(at[q]) * a.columns + column(at[q]), a.exponents + at[q].row * blocks + at[q].column / kBlock);
        }
    });
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
k_release(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, int rows, int columns, T* __restrict__ out,
          long long stride, Grid g) {
    const int blocks = blocks_of(g.width);
    walk<N>(g, (long long)rows * g.parts, [&](const Place (&at)[kPlaces<N>]) {
        auto row = [&](const Place& p) { return g.parts == 2 ? p.row >> 1 : p.row; };
        auto column = [&](const Place& p) { return (g.parts == 2 && (p.row & 1) ? g.width : 0) + p.column; };
        Codes<N> in[kPlaces<N>];
#pragma unroll
        for (int q = 0; q < kPlaces<N>; ++q)
            in[q] = load_codes<N>(codes + row(at[q]) * columns + column(at[q]), exponents + at[q].row * blocks + at[q].column / kBlock, at[q].live);
#pragma unroll
        for (int q = 0; q < kPlaces<N>; ++q) {
            float x[N];
            release<N>(in[q], x);
            store<T, N>(out + row(at[q]) * stride + column(at[q]), at[q].live, x);
        }
    });
}

// 1 / (1 + exp(-x)): in float32 to its last bits; where results have 16 bits, by the approximate exponential and reciprocal (2 and 1 ulp, and
// |x| 2^-24 for x log2 e)
template <typename T> __device__ __forceinline__ float sigmoid(float x) {
    float power, s;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(power) : "f"(x * -1.44269504088896341f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + power));
    return s;
}
template <> __device__ __forceinline__ float sigmoid<float>(float x) { return 1.0f / (1.0f + expf(-x)); }

template <typename T, int N, bool HOLD>
__global__ void __launch_bounds__(kThreads)
k_gate(fmb_held_t a, Grid g) {
    const int blocks = blocks_of(g.width);
    walk<N>(g, a.rows, [&](const Place (&at)[kPlaces<N>]) {
        Raw<T, N> raw[kPlaces<N>][2];
#pragma unroll
        for (int q = 0; q < kPlaces<N>; ++q) {
            const T* const u = (const T*)a.x + at[q].row * a.x_stride + at[q].column;
            raw[q][0] = load<T, N>(u, at[q].live);
            raw[q][1] = load<T, N>(u + g.width, at[q].live);
        }
#pragma unroll
        for (int q = 0; q < kPlaces<N>; ++q) {
            float x[N], y[N], h[N];
            unpack<T, N>(raw[q][0], x);
            unpack<T, N>(raw[q][1], y);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = x[i] * sigmoid<T>(x[i]) * y[i];
            store<T, N>((T*)a.h + at[q].row * a.h_stride + at[q].column, at[q].live, h);
            if (HOLD) {
                uint8_t* const codes = a.codes + at[q].row * a.columns + at[q].column;
                uint8_t* const exponents = a.exponents + 2 * at[q].row * blocks + at[q].column / kBlock;
                hold<T, N>(raw[q][0], x, at[q].live, at[q].exists, codes, exponents);
                hold<T, N>(raw[q][1], y, at[q].live, at[q].exists, codes + g.width, exponents + blocks);
            }
        }
    });
}

template <typename T, int N, bool HELD>
__global__ void __launch_bounds__(kThreads)
k_gate_gradient(fmb_held_t a, Grid g) {
    const int blocks = blocks_of(g.width);
    walk<N>(g, a.rows, [&](const Place (&at)[kPlaces<N>]) {
        Raw<T, N> dh_raw[kPlaces<N>], raw[kPlaces<N>][2];
        Codes<N> codes[kPlaces<N>][2];
#pragma unroll
        for (int q = 0; q < kPlaces<N>; ++q) {
            dh_raw[q] = load<T, N>((const T*)a.dh + at[q].row * a.dh_stride + at[q].column, at[q].live);
            if (HELD) {
                const uint8_t* const from = a.codes + at[q].row * a.columns + at[q].column;
                const uint8_t* const exponents = a.exponents + 2 * at[q].row * blocks + at[q].column / kBlock;
                codes[q][0] = load_codes<N>(from, exponents, at[q].live);
                codes[q][1] = load_codes<N>(from + g.width, exponents + blocks, at[q].live);
            } else {
                const T* const u = (const T*)a.x + at[q].row * a.x_stride + at[q].column;
                raw[q][0] = load<T, N>(u, at[q].live);
                raw[q][1] = load<T, N>(u + g.width, at[q].live);
            }
        }
#pragma unroll
        for (int q = 0; q < kPlaces<N>; ++q) {
            float x[N], y[N], dh[N], h[N];
            unpack<T, N>(dh_raw[q], dh);
            if (HELD) {
                release<N>(codes[q][0], x);
                release<N>(codes[q][1], y);
            } else {
                unpack<T, N>(raw[q][0], x);
                unpack<T, N>(raw[q][1], y);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float s = sigmoid<T>(x[i]), silu = x[i] * s;
                h[i] = silu * y[i];
                y[i] = dh[i] * y[i] * s * (1.0f + x[i] * (1.0f - s));
                x[i] = dh[i] * silu;
            }
            T* const du = (T*)a.du + at[q].row * a.du_stride + at[q].column;
            store<T, N>(du, at[q].live, y);
            store<T, N>(du + g.width, at[q].live, x);
            if (a.h) store<T, N>((T*)a.h + at[q].row * a.h_stride + at[q].column, at[q].live, h);
        }
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
    const int columns_of_lane = n == 1 ? kPlaces<1> : n;
    while (g.lanes < kThreads && g.lanes * columns_of_lane < g.width) g.lanes *= 2;
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
