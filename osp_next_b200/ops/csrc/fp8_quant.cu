// Block-128 fp8 quantisation (format: fp8.cuh) of a matrix x [R, K] in bf16, fp16 or fp32.
//
//   fp8_quantize_rows    1 x 128 blocks along K: codes [R, Kp], one warp per row and 512 columns
//   fp8_quantize_tiles   128 x 128 tiles: codes of x (blocks 1 x 128), of x^T (blocks 1 x 128
//                        along R, for the weight gradient), or both from one read; or one
//                        scale per tile (weights), whose codes then serve both orientations
//
// Both are bound by memory: 2 or 4 bytes read and 1 (+ 1/128) written per element and side.  Measured
// against the copy rate of 6551 GB/s: rows of 80640 x 5120 bf16 in 181 us (1.04, part of the codes
// still in L2), 20160 x 13824 bf16 both ways in 206 us (0.83), tiles of an fp32 8960 x 1536 weight both ways
// in 16.3 us (0.77).
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"
#include "launch.h"

namespace osp {
namespace fp8 {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

// The larger of two magnitudes given as fp32 bits.  Maxima are first taken so that a NaN wins
// (SEE_NAN), which shows with infinities as a result >= kInfBits; a block that has one turns its
// infinities into NaN and takes its maxima again so that NaN loses.
template <bool SEE_NAN> __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
  if constexpr (SEE_NAN) return max(a, b);
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}

// N 32-bit words from any address that is a multiple of the element size: the aligned 16-byte groups
// that hold them (each holds some of them, so none lies outside the allocation), shifted into
// place.  Rows whose stride is not a multiple of 16 bytes read this way; element by element
// they took several times as long.
template <int N> __device__ __forceinline__ void load_shifted(const void* p, uint32_t* out) {
  const uint32_t o = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
  const uint4* g = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15));
  uint32_t w[N + 4];
#pragma unroll
  for (int i = 0; i <= N / 4; ++i) {
    const uint4 u = i < N / 4 || o ? g[i] : make_uint4(0, 0, 0, 0);
    w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
  }
#pragma unroll
  for (int i = 0; i < N + 2; ++i) w[i] = o & 8u ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < N + 1; ++i) w[i] = o & 4u ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = o & 2u ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
}

// 8 consecutive elements of a row as they are in memory (16 bytes of a 16-bit type, 32 of fp32);
// maxima of 16-bit types are taken two at a time in packed registers.
template <typename T> struct Piece {
  uint4 r;
  __device__ __forceinline__ void load(const T* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void load_anywhere(const T* p) { load_shifted<4>(p, reinterpret_cast<uint32_t*>(&r)); }
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load_some(const T* p, int n) {
    uint16_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = i < n ? reinterpret_cast<const uint16_t*>(p)[i] : 0;
    r = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                   h[6] | (uint32_t)h[7] << 16);
  }
  // infinities become NaN (e4m3 has none, and a silent 448 would hide an overflow)
  __device__ __forceinline__ void spoil_inf() {
    constexpr uint32_t kInf = std::is_same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
    uint32_t* u = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((u[i] & 0x7FFFu) == kInf) u[i] |= 1u;
      if (((u[i] >> 16) & 0x7FFFu) == kInf) u[i] |= 0x10000u;
    }
  }
  // keeps the packed form live here: unpacked copies are not carried from one use to the next
  __device__ __forceinline__ void pin() { asm volatile("" : "+r"(r.x), "+r"(r.y), "+r"(r.z), "+r"(r.w)); }
  __device__ __forceinline__ uint32_t reg(int i) const { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }
  __device__ __forceinline__ static float wide(uint32_t u, int half) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return __uint_as_float(half ? u & 0xFFFF0000u : u << 16);
    } else {
      const uint32_t h = half ? u >> 16 : u & 0xFFFFu;
      return __half2float(__ushort_as_half((unsigned short)h));
    }
  }
  __device__ __forceinline__ float get(int j) const { return wide(reg(j >> 1), j & 1); }
  // the larger magnitudes of two registers (their signs are of no meaning)
  template <bool SEE_NAN> __device__ __forceinline__ static uint32_t top(uint32_t a, uint32_t b) {
    uint32_t m;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      if constexpr (SEE_NAN) asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
      else asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    } else {
      if constexpr (SEE_NAN) asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
      else asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    }
    return m;
  }
  __device__ __forceinline__ static uint32_t bits(uint32_t packed, int half) {
    return __float_as_uint(wide(packed, half)) & 0x7FFFFFFFu;
  }
  template <bool SEE_NAN> __device__ __forceinline__ uint32_t packed_max() const {
    return top<SEE_NAN>(top<SEE_NAN>(r.x, r.y), top<SEE_NAN>(r.z, r.w));
  }
  template <bool SEE_NAN> __device__ __forceinline__ uint32_t max_bits() const {
    const uint32_t m = packed_max<SEE_NAN>();
    return larger<SEE_NAN>(bits(m, 0), bits(m, 1));
  }
};
template <> struct Piece<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void load_anywhere(const float* p) { load_shifted<8>(p, reinterpret_cast<uint32_t*>(v)); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
  __device__ __forceinline__ void load_some(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
  }
  __device__ __forceinline__ void spoil_inf() {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (isinf(v[i])) v[i] = __uint_as_float(0x7FFFFFFFu);
  }
  __device__ __forceinline__ void pin() {}
  __device__ __forceinline__ float get(int j) const { return v[j]; }
  template <bool SEE_NAN> __device__ __forceinline__ uint32_t max_bits() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = larger<SEE_NAN>(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
  }
};
// The piece at column c of a row of K; zeros from column K on.
template <typename T, bool VEC>
__device__ __forceinline__ void load_piece(Piece<T>& o, const T* row, int c, int K) {
  if (c + 8 <= K) {
    if constexpr (VEC) o.load(row + c);
    else o.load_anywhere(row + c);
  } else {
    o.load_some(row + c, K - c);
  }
}
// ---------------------------------------------------------------------------- rows
// A lane owns 16 consecutive columns, so 8 lanes own a block (3 shuffles for its maximum), a
// lane's codes are one 16-byte store and a warp's four scales one 4-byte word.  A warp takes two
// such runs of 512 columns, with the loads of both in flight.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* x, long ld, uint8_t* q, uint8_t* scale, int R,
                                                            int K, int Kp, int kgroups, long total) {
  grid_dependency_wait();
  allow_dependents();
  const int lane = threadIdx.x & 31;
  const long w0 = ((long)blockIdx.x * 8 + (threadIdx.x >> 5)) * 2;
  if (w0 >= total) return;
  Piece<T> v[2][2];
  long row[2];
  int kg[2];
  row[0] = w0 / kgroups;
  kg[0] = (int)(w0 - row[0] * kgroups);
  const bool wraps = kg[0] + 1 == kgroups;
  row[1] = w0 + 1 < total ? row[0] + wraps : (long)1 << 40;      // past the end: nothing to write
  kg[1] = wraps ? 0 : kg[0] + 1;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int c = kg[u] * 512 + lane * 16;
    if (row[u] < R) {
      load_piece<T, VEC>(v[u][0], x + row[u] * ld, c, K);
      load_piece<T, VEC>(v[u][1], x + row[u] * ld, c + 8, K);
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (row[u] == (long)1 << 40) return;
    uint32_t* word = reinterpret_cast<uint32_t*>(scale + scale_offset(row[u], 4 * kg[u], kgroups));
    if (row[u] >= R) {
      if (lane == 0) *word = 0;
      continue;
    }
    const int c = kg[u] * 512 + lane * 16;
    uint32_t amax = max(v[u][0].template max_bits<true>(), v[u][1].template max_bits<true>());
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (__any_sync(0xffffffffu, amax >= kInfBits)) {
      v[u][0].spoil_inf();
      v[u][1].spoil_inf();
      amax = larger<false>(v[u][0].template max_bits<false>(), v[u][1].template max_bits<false>());
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) amax = larger<false>(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (amax >= kInfBits) amax = 0;              // nothing finite
    }
    const uint32_t byte = scale_byte(amax);
    const float inv = inv_scale(byte);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = v[u][i >> 1].get((i & 1) * 4 + j) * inv;
      o[i] = cvt4(y[0], y[1], y[2], y[3]);
    }
    if (c < Kp) *reinterpret_cast<uint4*>(q + row[u] * Kp + c) = make_uint4(o[0], o[1], o[2], o[3]);
    uint32_t mine = c < Kp ? byte << (8 * (lane >> 3)) : 0u;
    mine |= __shfl_xor_sync(0xffffffffu, mine, 8);
    mine |= __shfl_xor_sync(0xffffffffu, mine, 16);
    if (lane == 0) *word = mine;
  }
}

// ---------------------------------------------------------------------------- tiles
// One CTA per 128 x 128 tile; a thread holds 8 rows x 8 columns, a warp 32 x 64 (4 x 8
// threads), so that row loads are 128-byte segments, row codes 64-byte and column codes
// 32-byte ones without a pass through shared memory.  16-bit inputs stay packed in registers
// (32 for a thread) and their maxima are taken two at a time; all 8 loads are in flight at once.
// Maxima meet in shared memory, one thread per row and column forms its scale, and every
// thread reads back the 16 factors that it needs.
// SUMS: also the sums of x over the tile's 128 rows, part [R / 128, K] (a bias gradient's first
// step, without another read of x).
template <typename T, bool VEC, bool TILE_SCALE, bool ROWS, bool COLS, bool SUMS>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2)
quantize_tiles_kernel(const T* x, long ld, uint8_t* q, uint8_t* scale, uint8_t* qt, uint8_t* scale_t, float* part,
                      int R, int K, int Kp, int Rp) {
  __shared__ uint32_t top[2][4][128];              // [0]: rows over 2 warps, [1]: columns over 4
  __shared__ __align__(16) float factor[2][128];
  __shared__ float sums[SUMS ? 4 : 1][128];
  grid_dependency_wait();
  allow_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wr = warp >> 1, wc = warp & 1;
  const int rl = wr * 32 + (lane >> 3) * 8;        // first row of this thread in the tile
  const int cl = wc * 64 + (lane & 7) * 8;         // first column
  const int kb = blockIdx.x, rb = blockIdx.y;
  const long r0 = (long)rb * 128 + rl;
  const int c0 = kb * 128 + cl;
  const bool inner = (rb + 1) * 128L <= R && (kb + 1) * 128 <= K;      // a whole tile
  Piece<T> v[8];
  if (inner) {
    const T* p = x + r0 * ld + c0;
#pragma unroll
    for (int i = 0; i < 8; ++i, p += ld) {
      if constexpr (VEC) v[i].load(p);
      else v[i].load_anywhere(p);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (r0 + i < R) load_piece<T, VEC>(v[i], x + (r0 + i) * ld, c0, K);
      else v[i].zero();
    }
  }
  // maxima of the thread's rows (over 8 columns) and columns (over 8 rows), then over the warp
  auto gather = [&](auto see) {
    constexpr bool SEE = decltype(see)::value;
    using P = Piece<T>;
    uint32_t seen = 0;
    if constexpr (TILE_SCALE) {
#pragma unroll
      for (int i = 0; i < 8; ++i) seen = larger<SEE>(seen, v[i].template max_bits<SEE>());
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) seen = larger<SEE>(seen, __shfl_xor_sync(0xffffffffu, seen, o));
      if (lane == 0) top[0][0][warp] = seen;
    } else if constexpr (sizeof(T) == 2) {
      if constexpr (ROWS) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const uint32_t a = v[i].template packed_max<SEE>(), b = v[i + 1].template packed_max<SEE>();
          // the two rows side by side
          uint32_t m = P::template top<SEE>(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) m = P::template top<SEE>(m, __shfl_xor_sync(0xffffffffu, m, o));
          const uint32_t m0 = P::bits(m, 0), m1 = P::bits(m, 1);
          seen = max(seen, max(m0, m1));
          if ((lane & 7) == 0) *reinterpret_cast<uint2*>(&top[0][wc][rl + i]) = make_uint2(m0, m1);
        }
      }
      if constexpr (COLS) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t m = P::template top<SEE>(v[0].reg(k), v[1].reg(k));
#pragma unroll
          for (int i = 2; i < 8; ++i) m = P::template top<SEE>(m, v[i].reg(k));
#pragma unroll
          for (int o = 8; o < 32; o <<= 1) m = P::template top<SEE>(m, __shfl_xor_sync(0xffffffffu, m, o));
          const uint32_t m0 = P::bits(m, 0), m1 = P::bits(m, 1);
          seen = max(seen, max(m0, m1));
          if (lane < 8) *reinterpret_cast<uint2*>(&top[1][wr][cl + 2 * k]) = make_uint2(m0, m1);
        }
      }
    } else {
      if constexpr (ROWS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t m = v[i].template max_bits<SEE>();
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) m = larger<SEE>(m, __shfl_xor_sync(0xffffffffu, m, o));
          seen = max(seen, m);
          if ((lane & 7) == 0) top[0][wc][rl + i] = m;
        }
      }
      if constexpr (COLS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t m = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) m = larger<SEE>(m, __float_as_uint(v[i].get(j)) & 0x7FFFFFFFu);
#pragma unroll
          for (int o = 8; o < 32; o <<= 1) m = larger<SEE>(m, __shfl_xor_sync(0xffffffffu, m, o));
          seen = max(seen, m);
          if (lane < 8) top[1][wr][cl + j] = m;
        }
      }
    }
    return seen;
  };
  const uint32_t seen = gather(std::true_type());
  if constexpr (SUMS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].pin();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) a += v[i].get(j);
      a += __shfl_xor_sync(0xffffffffu, a, 8);
      a += __shfl_xor_sync(0xffffffffu, a, 16);
      if (lane < 8) sums[wr][cl + j] = a;
    }
  }
  if (__syncthreads_or(seen >= kInfBits)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].spoil_inf();
    gather(std::false_type());
    __syncthreads();
  }
  // one thread per row (the first 128) and per column: its scale byte, and zeros for what the
  // last chunk of four blocks lacks
  {
    const int side = tid >> 7, i = tid & 127;
    if ((side == 0 && ROWS) || (side == 1 && COLS)) {
      uint32_t m;
      if constexpr (TILE_SCALE) {
        m = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) m = larger<false>(m, top[0][0][w]);
      } else {
        m = larger<false>(top[side][0][i], top[side][1][i]);
        if (side == 1) m = larger<false>(m, larger<false>(top[1][2][i], top[1][3][i]));
      }
      if (m >= kInfBits) m = 0;                    // nothing finite
      const uint32_t byte = scale_byte(m);
      factor[side][i] = inv_scale(byte);
      const int blk = side ? rb : kb, blocks = side ? gridDim.y : gridDim.x;
      const long line = side ? kb * 128L + i : rb * 128L + i;
      uint8_t* s = (side ? scale_t : scale) + scale_offset(line, blk, (blocks + 3) >> 2);
      *s = line < (side ? K : R) ? (uint8_t)byte : 0;
      if (blk == blocks - 1)
        for (int j = 1; j < 4 - (blk & 3); ++j) s[j] = 0;
    }
    if constexpr (SUMS) {
      if (side == 1 && kb * 128 + i < K)
        part[(long)rb * K + kb * 128 + i] = sums[0][i] + sums[1][i] + sums[2][i] + sums[3][i];
    }
  }
  __syncthreads();
  if constexpr (ROWS) {
    float f[8];
    *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(&factor[0][rl]);
    *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(&factor[0][rl + 4]);
    uint8_t* p = q + r0 * Kp + c0;
#pragma unroll
    for (int i = 0; i < 8; ++i, p += Kp) {
      v[i].pin();
      uint2 o;
      o.x = cvt4(v[i].get(0) * f[i], v[i].get(1) * f[i], v[i].get(2) * f[i], v[i].get(3) * f[i]);
      o.y = cvt4(v[i].get(4) * f[i], v[i].get(5) * f[i], v[i].get(6) * f[i], v[i].get(7) * f[i]);
      if (inner || r0 + i < R) *reinterpret_cast<uint2*>(p) = o;
    }
  }
  if constexpr (COLS) {
    float f[8];
    *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(&factor[1][cl]);
    *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(&factor[1][cl + 4]);
    uint8_t* p = qt + (long)c0 * Rp + r0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].pin();
#pragma unroll
    for (int j = 0; j < 8; ++j, p += Rp) {
      uint2 o;
      o.x = cvt4(v[0].get(j) * f[j], v[1].get(j) * f[j], v[2].get(j) * f[j], v[3].get(j) * f[j]);
      o.y = cvt4(v[4].get(j) * f[j], v[5].get(j) * f[j], v[6].get(j) * f[j], v[7].get(j) * f[j]);
      if (inner || c0 + j < K) *reinterpret_cast<uint2*>(p) = o;
    }
  }
}

}  // namespace fp8

// Codes and packed scales of a [rows, cols] matrix on x's device.
static void alloc_side(const at::Tensor& x, int64_t rows, int64_t cols, at::Tensor& q, at::Tensor& s) {
  q = at::empty({rows, (cols + 127) / 128 * 128}, x.options().dtype(at::kFloat8_e4m3fn));
  s = at::empty({(rows + 127) / 128, (cols + 511) / 512, 32, 4, 4}, x.options().dtype(at::kByte));
}

template <typename T>
static void quantize_t(const at::Tensor& x, uint8_t* q, uint8_t* s, uint8_t* qt, uint8_t* st, float* part,
                       bool tile_scale, cudaStream_t stream) {
  const int R = (int)x.size(0), K = (int)x.size(1);
  const int Kp = (K + 127) / 128 * 128, Rp = (R + 127) / 128 * 128;
  const long ld = x.stride(0);
  const T* xp = reinterpret_cast<const T*>(x.data_ptr());
  const bool vec = reinterpret_cast<uintptr_t>(xp) % 16 == 0 && (ld * (long)sizeof(T)) % 16 == 0;
  if (!tile_scale && qt == nullptr) {
    const int kgroups = (K + 511) / 512;
    const long total = (long)Rp * kgroups;
    const unsigned grid = (unsigned)((total + 15) / 16);
    launch_kernel(vec ? fp8::quantize_rows_kernel<T, true> : fp8::quantize_rows_kernel<T, false>, grid, 256, 0, 1,
                  stream, xp, ld, q, s, R, K, Kp, kgroups, total);
    return;
  }
  const dim3 grid(Kp / 128, Rp / 128);
  TORCH_CHECK(grid.y <= 65535, "fp8_quantize: more than 8388480 rows");
#define OSP_TILES(VEC, TS, RO, CO, SU) \
  launch_kernel(fp8::quantize_tiles_kernel<T, VEC, TS, RO, CO, SU>, grid, 256, 0, 1, stream, xp, ld, q, s, qt, st, \
                part, R, K, Kp, Rp)
#define OSP_TILES_SIDES(VEC, TS)                             \
  do {                                                       \
    if (part) OSP_TILES(VEC, false, true, true, true);       \
    else if (q && qt) OSP_TILES(VEC, TS, true, true, false); \
    else if (q) OSP_TILES(VEC, TS, true, false, false);      \
    else OSP_TILES(VEC, TS, false, true, false);             \
  } while (0)
  if (vec) {
    if (tile_scale) OSP_TILES_SIDES(true, true);
    else OSP_TILES_SIDES(true, false);
  } else {
    if (tile_scale) OSP_TILES_SIDES(false, true);
    else OSP_TILES_SIDES(false, false);
  }
#undef OSP_TILES_SIDES
#undef OSP_TILES
}

// Codes and scales of x [R, K] (`rows`) and / or of its transpose (`cols`); any strides.  Sides
// that were not asked for come back undefined.  `sums` (both sides, blocks of one row): also the
// column sums of x over each 128 rows, fp32 [ceil(R / 128), K].
std::vector<at::Tensor> fp8_quantize(const at::Tensor& x_, bool tile_scale, bool rows, bool cols, bool sums) {
  TORCH_CHECK(x_.is_cuda() && x_.dim() == 2, "fp8_quantize: x [R, K] on the GPU");
  at::Tensor x = x_;
  const int64_t R = x.size(0), K = x.size(1);
  TORCH_CHECK(R < (int64_t(1) << 31) - 128 && K < (int64_t(1) << 31) - 512, "fp8_quantize: sizes below 2^31");
  c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(!sums || (rows && cols && !tile_scale), "fp8_quantize: column sums go with both sides");
  std::vector<at::Tensor> out(5);
  if (rows) alloc_side(x, R, K, out[0], out[1]);
  if (cols) alloc_side(x, K, R, out[2], out[3]);
  if (sums) out[4] = at::empty({(R + 127) / 128, K}, x.options().dtype(at::kFloat));
  if (R == 0 || K == 0) return out;
  bool swap = false;
  if (K > 1 && x.stride(1) != 1) {
    if (sums || (R > 1 && x.stride(0) != 1)) {
      x = x.contiguous();
    } else {                        // a transposed view: its rows are the columns of what is stored
      x = x.t();
      swap = true;
    }
  }
  auto ptr = [&](int i) { return out[i].defined() ? reinterpret_cast<uint8_t*>(out[i].data_ptr()) : nullptr; };
  uint8_t *q = ptr(swap ? 2 : 0), *s = ptr(swap ? 3 : 1), *qt = ptr(swap ? 0 : 2), *st = ptr(swap ? 1 : 3);
  float* part = sums ? out[4].data_ptr<float>() : nullptr;
  auto stream = c10::cuda::getCurrentCUDAStream();
  switch (x.scalar_type()) {
    case at::kBFloat16: quantize_t<__nv_bfloat16>(x, q, s, qt, st, part, tile_scale, stream); break;
    case at::kHalf: quantize_t<__half>(x, q, s, qt, st, part, tile_scale, stream); break;
    case at::kFloat: quantize_t<float>(x, q, s, qt, st, part, tile_scale, stream); break;
    default: TORCH_CHECK(false, "fp8_quantize: x bf16, fp16 or fp32");
  }
  return out;
}

}  // namespace osp
