// Rows held in 8 bits: e4m3 codes in units of a power of two per 32 columns, the exponent plus 127 in a byte.
//
// The unit is the smallest power of two with |x| <= 448 units in the block, 448 being the largest code. A power of two, so that a code
// read back is exact in the rows' own type: 4 bits of fraction at exponents that the type has. Two limits keep them there: units
// are no smaller than 2^-117 (float16: 2^-15), so that the smallest code, 2^-9 units, is a number of the type and no bfloat16 is
// subnormal; and in the highest unit, 2^120 (2^8), codes end at 240, since 256 units would be past the type's largest number. What is
// not finite is held as NaN, and does not count for the unit.
#pragma once

#include "eight.cuh"

#include <cuda_fp8.h>

namespace fmb {
namespace held {

constexpr int kBlock = FMB_HELD_BLOCK;
constexpr int kBias = 127;

__host__ __device__ __forceinline__ constexpr int blocks_of(int columns) { return (columns + kBlock - 1) / kBlock; }

template <typename T> struct Units { static constexpr int kLowest = -117, kHighest = 120; };
template <> struct Units<__half> { static constexpr int kLowest = -15, kHighest = 8; };

// 2^(byte - 127) for bytes from 1 to 254
__device__ __forceinline__ float unit_of(int byte) { return __uint_as_float((uint32_t)byte << 23); }

// two codes, the first in the lower byte
__device__ __forceinline__ float2 two_values(uint32_t codes) {
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3)));
}

// rows read back, [rows][columns], row_stride apart (checkpoints.cu)
int release(int type, const uint8_t* codes, const uint8_t* exponents, int rows, int columns, int parts, void* out, long long row_stride,
            cudaStream_t stream);

}  // namespace held
}  // namespace fmb
