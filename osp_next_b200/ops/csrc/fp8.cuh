// The block-128 fp8 format shared by the quantiser (fp8_quant.cu) and the product (fp8_gemm.cu).
//
// A matrix [R, K] is stored as e4m3 codes [R, Kp] (Kp = K rounded up to 128, zero-padded) and
// one power-of-two scale per block of 128 along K (for 1 row, or for 128 rows of a weight),
// held as the byte e = log2(scale) + 127.  The scale is the smallest 2^k, k >= -126, with
// max|x| / 2^k <= 448 (the largest e4m3 value), so the scaling is exact in fp32 and the
// tensor core can apply it itself (block-scaled tcgen05.mma).
//
// Scale bytes lie as the tensor core wants them in TMEM: chunks of 128 rows x 4 blocks
// (512 bytes), chunk [r / 128][kb / 4], in it [r % 32][r % 128 / 32][kb % 4].  One
// tcgen05.cp then moves a chunk, and block kb is byte kb % 4 of every word.  Bytes of rows
// past R and blocks past K / 128 are zero.
#pragma once
#include <cuda_fp8.h>
#include <stdint.h>
#include <string>   // error messages: numbers go in as std::to_string, which needs no stream locale

namespace osp {
namespace fp8 {

constexpr int kBlock = 128;
constexpr int kChunkBytes = 512;
constexpr uint32_t kInfBits = 0x7F800000u;

// Scale byte of a block whose largest magnitude has the (finite, sign-less) fp32 bits `amax`:
// exponent of amax - 8, one more when its mantissa is above 1.75 (448 = 1.75 * 2^8).
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  const int e = (int)((amax + 0x1FFFFFu) >> 23) - 8;
  return (uint32_t)max(e, 1);
}
// 2^(127 - byte), the factor that brings a block into e4m3 range (byte <= 247).
__device__ __forceinline__ float inv_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Byte offset of the scale of (row r, block kb) in the packed scales; kgroups = ceil(K / 512).
__device__ __forceinline__ long scale_offset(long r, int kb, int kgroups) {
  const int i = (int)(r & 127);
  return ((r >> 7) * kgroups + (kb >> 2)) * kChunkBytes + (i & 31) * 16 + (i >> 5) * 4 + (kb & 3);
}

// Two values -> two e4m3 codes (a in the low byte), round to nearest even.
__device__ __forceinline__ uint32_t cvt2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t cvt4(float a, float b, float c, float d) {
  return cvt2(a, b) | (cvt2(c, d) << 16);
}

}  // namespace fp8
}  // namespace osp
