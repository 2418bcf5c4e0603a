// trb_fp4.cuh -- microscaled 4-bit floating point as the kernels of this library store it.
//
// A row of k values is k / 2 bytes of e2m1 codes (sign, two bits of exponent, one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4,
// 6), the even k in the low four bits, and one e8m0 byte b, 2^(b - 127) or NaN for 255, for every 32 values.  The
// scales of a row begin at a multiple of 16 bytes, so that 16 of them, those of 512 values, are one load.
#pragma once

#include "trb_common.cuh"

namespace trb {
namespace fp4 {

constexpr int kBlock = 32;
// Bytes from one row's scales to the next one's.
__host__ __device__ constexpr int scale_pitch(int k) { return (k / kBlock + 15) & ~15; }

}  // namespace fp4
}  // namespace trb
