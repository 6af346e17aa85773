// Eight neighbouring values of a row by a lane: sixteen bytes at a time where rows start at multiples of eight values (WIDE), else by the words
// and halves that they lie in.
#pragma once

#include "grouped.cuh"

#include <type_traits>

namespace fmb {
namespace eight {

constexpr int kEach = 8;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T rounded(float x) { return grp::from_float<T>(x); }
template <> __device__ __forceinline__ float rounded<float>(float x) { return x; }

template <typename T> __device__ __forceinline__ uint32_t two_of(float x, float y);
template <> __device__ __forceinline__ uint32_t two_of<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t two_of<__half>(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A lane's values as they are in memory, two to a word where they have 16 bits, so that what is on its way takes few registers
template <typename T> struct Raw {
    static constexpr int kWords = kEach * (int)sizeof(T) / 4;
    uint32_t v[kWords];
};

template <typename T, bool WIDE>
__device__ __forceinline__ Raw<T> load(const T* __restrict__ at, int live) {
    Raw<T> in = {};
    if (live >= kEach) {
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < Raw<T>::kWords; i += 4) {
                const uint4 four = __ldg(reinterpret_cast<const uint4*>(at) + i / 4);
                in.v[i] = four.x; in.v[i + 1] = four.y; in.v[i + 2] = four.z; in.v[i + 3] = four.w;
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) in.v[i] = __ldg(reinterpret_cast<const uint32_t*>(at) + i);
        } else if ((uintptr_t)at & 2) {
            // three words between two halves
            const uint32_t* const words = reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint16_t*>(at) + 1);
            const uint32_t first = __ldg(reinterpret_cast<const uint16_t*>(at)), last = __ldg(reinterpret_cast<const uint16_t*>(at) + 7);
            const uint32_t a = __ldg(words), b = __ldg(words + 1), c = __ldg(words + 2);
            in.v[0] = first | a << 16;
            in.v[1] = __funnelshift_r(a, b, 16);
            in.v[2] = __funnelshift_r(b, c, 16);
            in.v[3] = c >> 16 | last << 16;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) in.v[i] = __ldg(reinterpret_cast<const uint32_t*>(at) + i);
        }
        return in;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if (i >= live) break;
        if constexpr (sizeof(T) == 4) in.v[i] = __ldg(reinterpret_cast<const uint32_t*>(at) + i);
        else in.v[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(at) + i) << (16 * (i % 2));
    }
    return in;
}

template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& in, float (&x)[kEach]) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const uint32_t w = in.v[i * sizeof(T) / 4];
        if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) x[i] = __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
        else x[i] = __half2float(__ushort_as_half((uint16_t)(i % 2 ? w >> 16 : w & 0xffffu)));
    }
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store(T* __restrict__ at, int live, const float (&x)[kEach]) {
    uint32_t v[Raw<T>::kWords];
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = __float_as_uint(x[i]);
        else v[i] = two_of<T>(x[2 * i], x[2 * i + 1]);
    }
    if (live >= kEach) {
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < Raw<T>::kWords; i += 4) *(reinterpret_cast<uint4*>(at) + i / 4) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else if (sizeof(T) == 2 && (uintptr_t)at & 2) {
            uint16_t* const halves = reinterpret_cast<uint16_t*>(at);
            uint32_t* const words = reinterpret_cast<uint32_t*>(halves + 1);
            halves[0] = (uint16_t)v[0];
#pragma unroll
            for (int i = 0; i < 3; ++i) words[i] = __funnelshift_r(v[i], v[i + 1 < Raw<T>::kWords ? i + 1 : i], 16);
            halves[7] = (uint16_t)(v[3] >> 16);
        } else {
#pragma unroll
            for (int i = 0; i < Raw<T>::kWords; ++i) reinterpret_cast<uint32_t*>(at)[i] = v[i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if (i >= live) break;
        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(at)[i] = v[i];
        else reinterpret_cast<uint16_t*>(at)[i] = (uint16_t)(v[i / 2] >> (16 * (i % 2)));
    }
}

}  // namespace eight
}  // namespace fmb
