// Rows between the forward and the backward pass in 8 bits (held.cuh), and the gate of an expert's two matrices with them:
//
//   hold:     codes and exponents of x
//   gate:     u = (a | b), h = silu(a) b, and u held on the way
//   gradient: da = dh b s (1 + a (1 - s)), db = dh a s with s = 1 / (1 + exp(-a)), from held u (or u itself), and h anew
//   release:  x read back
//
// One pass each, bound by memory. A lane has eight neighbouring columns of two rows, 16 bytes of a 16-bit type, four lanes a block of 32;
// where rows do not start at multiples of eight values (not WIDE) it takes them by the words and halves that they lie in (a column a
// lane, side by side with the others, takes four times the instructions: 20,000 rows of 2 x 1,001 in 80 us). The largest of
// a block is a maximum over its lanes, so the codes leave in the pass that reads the values. The arithmetic is in fp32 and
// every result is rounded once.

#include "eight.cuh"
#include "held.cuh"

#include <algorithm>
#include <type_traits>

namespace fmb {
namespace held {

namespace {

using namespace eight;

constexpr int kThreads = 256;

constexpr int kLanes = kBlock / kEach;

// A CTA's threads by rows: `lanes` (a power of two, whole blocks) for the columns of one, 256 / lanes rows at a time.
struct Grid {
    int lanes, width, columns, parts;            // width: of a part
};

// eight codes, by words, halves and bytes as they lie
template <bool WIDE>
__device__ __forceinline__ void store_codes(uint8_t* __restrict__ at, int live, uint32_t low, uint32_t high) {
    const unsigned from = (unsigned)(uintptr_t)at & 3;
    if (live >= kEach && WIDE) {
        *reinterpret_cast<uint2*>(at) = make_uint2(low, high);
    } else if (live >= kEach && from == 0) {
        reinterpret_cast<uint32_t*>(at)[0] = low;
        reinterpret_cast<uint32_t*>(at)[1] = high;
    } else if (live >= kEach) {
        // up to the next word; a word; what is left
        const unsigned before = 4 - from;        // bytes, 1 to 3
        if (before & 1) at[0] = (uint8_t)low;
        if (before & 2) *reinterpret_cast<uint16_t*>(at + (before & 1)) = (uint16_t)(low >> (8 * (before & 1)));
        *reinterpret_cast<uint32_t*>(at + before) = __funnelshift_r(low, high, 8 * before);
        const uint32_t rest = high >> (8 * before);               // 4 - before bytes
        if (from & 2) *reinterpret_cast<uint16_t*>(at + before + 4) = (uint16_t)rest;
        if (from & 1) at[before + 4 + (from & 2)] = (uint8_t)(rest >> (8 * (from & 2)));
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i < live) at[i] = (uint8_t)((i < 4 ? low : high) >> (8 * (i % 4)));
    }
}

// the largest of |x|, as the bits of a float; NaN and infinities are larger than what is finite
template <typename T>
__device__ __forceinline__ uint32_t largest_of(const Raw<T>& in) {
    uint32_t largest = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) largest = max(largest, in.v[i] & 0x7fffffffu);
        return largest;
    } else {
#pragma unroll
        for (int i = 0; i < Raw<T>::kWords; ++i) largest = __vmaxu2(largest, in.v[i] & 0x7fff7fffu);
        largest = max(largest >> 16, largest & 0xffffu);
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return largest << 16;
        else return __float_as_uint(__half2float(__ushort_as_half((uint16_t)largest)));
    }
}

// Codes of this lane's values and the block's exponent, by all lanes of the warp; `live` of the values exist, the others are zero.
template <typename T, bool WIDE>
__device__ __forceinline__ void hold(const Raw<T>& raw, const float (&x)[kEach], int live, bool block_exists, uint8_t* __restrict__ codes,
                                     uint8_t* __restrict__ exponent) {
    constexpr uint32_t kInfinity = 0x7f800000u;
    auto over_block = [](uint32_t v) {
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    };
    // largest = m 2^E: 448 = 1.75 x 2^8 units hold it at e = E - 8 where m <= 1.75
    auto exponent_of = [](uint32_t largest) { return min(max((int)((largest + 0x1fffffu) >> 23) - kBias - 8, Units<T>::kLowest), Units<T>::kHighest); };
    uint32_t largest = over_block(largest_of<T>(raw));
    int e = exponent_of(largest);
    uint32_t two[kEach / 2];
    // What is not finite does not count for the unit and is NaN; in the highest unit codes end at 240. Neither is met often.
    if (__any_sync(0xffffffffu, e == Units<T>::kHighest)) {
        largest = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t bits = __float_as_uint(x[i]) & 0x7fffffffu;
            if (bits < kInfinity) largest = max(largest, bits);
        }
        e = exponent_of(over_block(largest));
        const float inverse = unit_of(kBias - e), most = e == Units<T>::kHighest ? 240.0f : 448.0f;
#pragma unroll
        for (int i = 0; i < kEach; i += 2) {
            two[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(fminf(fmaxf(x[i] * inverse, -most), most), fminf(fmaxf(x[i + 1] * inverse, -most), most)),
                                                  __NV_SATFINITE, __NV_E4M3);
            if ((__float_as_uint(x[i]) & 0x7fffffffu) >= kInfinity) two[i / 2] |= 0x7f;
            if ((__float_as_uint(x[i + 1]) & 0x7fffffffu) >= kInfinity) two[i / 2] |= 0x7f00;
        }
    } else {
        const float inverse = unit_of(kBias - e);
#pragma unroll
        for (int i = 0; i < kEach; i += 2) two[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(x[i] * inverse, x[i + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
    }
    store_codes<WIDE>(codes, live, two[0] | two[1] << 16, two[2] | two[3] << 16);
    if (block_exists && (threadIdx.x & (kLanes - 1)) == 0) *exponent = (uint8_t)(e + kBias);
}

// a lane's codes, and its values of them
struct Codes {
    uint32_t low, high, byte;
};

template <bool WIDE>
__device__ __forceinline__ Codes load_codes(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponent, int live) {
    Codes in = {};
    if (live <= 0) return in;
    in.byte = __ldg(exponent);
    if (live >= kEach && WIDE) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(codes));
        in.low = v.x;
        in.high = v.y;
    } else if (live >= kEach) {
        // the words that they lie in: the outer two hold bytes of them, so they are there
        const unsigned from = (unsigned)(uintptr_t)codes & 3;
        const uint32_t* const words = reinterpret_cast<const uint32_t*>(codes - from);
        const uint32_t a = __ldg(words), b = __ldg(words + 1), c = from ? __ldg(words + 2) : 0u;
        in.low = __funnelshift_r(a, b, 8 * from);
        in.high = __funnelshift_r(b, c, 8 * from);
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i < live) (i < 4 ? in.low : in.high) |= (uint32_t)__ldg(codes + i) << (8 * (i % 4));
    }
    return in;
}

__device__ __forceinline__ void release(const Codes& in, float (&x)[kEach]) {
    const float unit = unit_of(in.byte);
#pragma unroll
    for (int i = 0; i < kEach; i += 2) {
        const float2 v = two_values((i < 4 ? in.low : in.high) >> (8 * (i % 4)));
        x[i] = v.x * unit;
        x[i + 1] = v.y * unit;
    }
}

// Places of a thread, whose loads are on their way together: kEach neighbouring columns of two rows
constexpr int kPlaces = 2;

struct Place {
    long long row;
    int column, live;                            // columns that exist from there on
    bool exists;                                 // the block does
};

// The same number of rounds for all threads of a CTA; what is past the last row or block has nothing to load or store.
template <typename F>
__device__ __forceinline__ void walk(const Grid& g, long long rows, F body) {
    const int per_cta = kThreads / g.lanes, whole = blocks_of(g.width) * kBlock, first = (threadIdx.x & (g.lanes - 1)) * kEach;
    for (long long r0 = (long long)blockIdx.x * per_cta * kPlaces; r0 < rows; r0 += (long long)gridDim.x * per_cta * kPlaces) {
        const long long r = r0 + threadIdx.x / g.lanes;
        for (int c0 = 0; c0 < whole; c0 += g.lanes * kEach) {
            Place at[kPlaces];
#pragma unroll
            for (int q = 0; q < kPlaces; ++q) {
                at[q].row = r + q * per_cta;
                at[q].column = c0 + first;
                at[q].exists = at[q].row < rows && at[q].column < whole;
                at[q].live = at[q].exists ? g.width - at[q].column : 0;
            }
            body(at);
        }
    }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
k_hold(fmb_held_t a, Grid g) {
    const int blocks = blocks_of(g.width);
    walk(g, (long long)a.rows * g.parts, [&](const Place (&at)[kPlaces]) {
        auto row = [&](const Place& p) { return g.parts == 2 ? p.row >> 1 : p.row; };
        auto column = [&](const Place& p) { return (g.parts == 2 && (p.row & 1) ? g.width : 0) + p.column; };
        Raw<T> raw[kPlaces];
#pragma unroll
        for (int q = 0; q < kPlaces; ++q) raw[q] = load<T, WIDE>((const T*)a.x + row(at[q]) * a.x_stride + column(at[q]), at[q].live);
#pragma unroll
        for (int q = 0; q < kPlaces; ++q) {
            float x[kEach];
            unpack<T>(raw[q], x);
            hold<T, WIDE>(raw[q], x, at[q].live, at[q].exists, a.codes + row(at[q]) * a.columns + column(at[q]), a.exponents + at[q].row * blocks + at[q].column / kBlock);
        }
    });
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
k_release(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, int rows, int columns, T* __restrict__ out,
          long long stride, Grid g) {
    const int blocks = blocks_of(g.width);
    walk(g, (long long)rows * g.parts, [&](const Place (&at)[kPlaces]) {
        auto row = [&](const Place& p) { return g.parts == 2 ? p.row >> 1 : p.row; };
        auto column = [&](const Place& p) { return (g.parts == 2 && (p.row & 1) ? g.width : 0) + p.column; };
        Codes in[kPlaces];
#pragma unroll
        for (int q = 0; q < kPlaces; ++q)
            in[q] = load_codes<WIDE>(codes + row(at[q]) * columns + column(at[q]), exponents + at[q].row * blocks + at[q].column / kBlock, at[q].live);
#pragma unroll
        for (int q = 0; q < kPlaces; ++q) {
            float x[kEach];
            release(in[q], x);
            store<T, WIDE>(out + row(at[q]) * stride + column(at[q]), at[q].live, x);
        }
    });
}

// 1 / (1 + exp(-x)): in float32 to its last bits; where results have 16 bits, by the approximate exponential and reciprocal (2 and 1 ulp, and
// |x| 2^-24 for x log2 e; below 2^-126, for x under -87.3, it is zero, and x times it less than 2e-36 off)
template <typename T> __device__ __forceinline__ float sigmoid(float x) {
    float power, s;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(power) : "f"(x * -1.44269504088896341f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + power));
    return s;
}
template <> __device__ __forceinline__ float sigmoid<float>(float x) { return 1.0f / (1.0f + expf(-x)); }

template <typename T, bool WIDE, bool HOLD>
__global__ void __launch_bounds__(kThreads)
k_gate(fmb_held_t a, Grid g) {
    const int blocks = blocks_of(g.width);
    walk(g, a.rows, [&](const Place (&at)[kPlaces]) {
        Raw<T> raw[kPlaces][2];
#pragma unroll
        for (int q = 0; q < kPlaces; ++q) {
            const T* const u = (const T*)a.x + at[q].row * a.x_stride + at[q].column;
            raw[q][0] = load<T, WIDE>(u, at[q].live);
            raw[q][1] = load<T, WIDE>(u + g.width, at[q].live);
        }
#pragma unroll
        for (int q = 0; q < kPlaces; ++q) {
            float x[kEach], y[kEach], h[kEach];
            unpack<T>(raw[q][0], x);
            unpack<T>(raw[q][1], y);
#pragma unroll
            for (int i = 0; i < kEach; ++i) h[i] = x[i] * sigmoid<T>(x[i]) * y[i];
            store<T, WIDE>((T*)a.h + at[q].row * a.h_stride + at[q].column, at[q].live, h);
            if (HOLD) {
                uint8_t* const codes = a.codes + at[q].row * a.columns + at[q].column;
                uint8_t* const exponents = a.exponents + 2 * at[q].row * blocks + at[q].column / kBlock;
                hold<T, WIDE>(raw[q][0], x, at[q].live, at[q].exists, codes, exponents);
                hold<T, WIDE>(raw[q][1], y, at[q].live, at[q].exists, codes + g.width, exponents + blocks);
            }
        }
    });
}

template <typename T, bool WIDE, bool HELD>
__global__ void __launch_bounds__(kThreads)
k_gate_gradient(fmb_held_t a, Grid g) {
    const int blocks = blocks_of(g.width);
    walk(g, a.rows, [&](const Place (&at)[kPlaces]) {
        Raw<T> dh_raw[kPlaces], raw[kPlaces][2];
        Codes codes[kPlaces][2];
#pragma unroll
        for (int q = 0; q < kPlaces; ++q) {
            dh_raw[q] = load<T, WIDE>((const T*)a.dh + at[q].row * a.dh_stride + at[q].column, at[q].live);
            if (HELD) {
                const uint8_t* const from = a.codes + at[q].row * a.columns + at[q].column;
                const uint8_t* const exponents = a.exponents + 2 * at[q].row * blocks + at[q].column / kBlock;
                codes[q][0] = load_codes<WIDE>(from, exponents, at[q].live);
                codes[q][1] = load_codes<WIDE>(from + g.width, exponents + blocks, at[q].live);
            } else {
                const T* const u = (const T*)a.x + at[q].row * a.x_stride + at[q].column;
                raw[q][0] = load<T, WIDE>(u, at[q].live);
                raw[q][1] = load<T, WIDE>(u + g.width, at[q].live);
            }
        }
#pragma unroll
        for (int q = 0; q < kPlaces; ++q) {
            float x[kEach], y[kEach], dh[kEach], h[kEach];
            unpack<T>(dh_raw[q], dh);
            if (HELD) {
                release(codes[q][0], x);
                release(codes[q][1], y);
            } else {
                unpack<T>(raw[q][0], x);
                unpack<T>(raw[q][1], y);
            }
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const float s = sigmoid<T>(x[i]), silu = x[i] * s;
                h[i] = silu * y[i];
                y[i] = dh[i] * y[i] * s * (1.0f + x[i] * (1.0f - s));
                x[i] = dh[i] * silu;
            }
            T* const du = (T*)a.du + at[q].row * a.du_stride + at[q].column;
            store<T, WIDE>(du, at[q].live, y);
            store<T, WIDE>(du + g.width, at[q].live, x);
            if (a.h) store<T, WIDE>((T*)a.h + at[q].row * a.h_stride + at[q].column, at[q].live, h);
        }
    });
}

bool by_eight(const void* base, long long stride, int bytes) {
    return ((uintptr_t)base & (uintptr_t)(std::min(16, 8 * bytes) - 1)) == 0 && stride % 8 == 0;
}

Grid grid_of(int columns, int parts) {
    Grid g;
    g.columns = columns;
    g.parts = parts;
    g.width = columns / parts;
    g.lanes = kLanes;
    while (g.lanes < kThreads && g.lanes * kEach < g.width) g.lanes *= 2;
    return g;
}

unsigned ctas(const Grid& g, long long rows) {
    const int rows_at_once = kThreads / g.lanes * kPlaces;
    return (unsigned)std::min<long long>((rows + rows_at_once - 1) / rows_at_once, 1 << 20);
}

struct Launch {
    const fmb_held_t& a;
    bool wide;
    cudaStream_t stream;

    template <typename T, bool WIDE>
    void go(int what) const {
        const Grid g = grid_of(a.columns, what == 0 ? a.parts : 2);
        const long long rows = (long long)a.rows * (what == 0 ? a.parts : 1);
        if (what == 0) k_hold<T, WIDE><<<ctas(g, rows), kThreads, 0, stream>>>(a, g);
        else if (what == 1 && a.codes) k_gate<T, WIDE, true><<<ctas(g, rows), kThreads, 0, stream>>>(a, g);
        else if (what == 1) k_gate<T, WIDE, false><<<ctas(g, rows), kThreads, 0, stream>>>(a, g);
        else if (a.codes) k_gate_gradient<T, WIDE, true><<<ctas(g, rows), kThreads, 0, stream>>>(a, g);
        else k_gate_gradient<T, WIDE, false><<<ctas(g, rows), kThreads, 0, stream>>>(a, g);
    }
    template <typename T> void typed(int what) const { wide ? go<T, true>(what) : go<T, false>(what); }

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
    const Grid g = grid_of(columns, parts);
    const long long all = (long long)rows * parts;
    if (eight) k_release<T, true><<<ctas(g, all), kThreads, 0, stream>>>(codes, exponents, rows, columns, (T*)out, stride, g);
    else k_release<T, false><<<ctas(g, all), kThreads, 0, stream>>>(codes, exponents, rows, columns, (T*)out, stride, g);
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
