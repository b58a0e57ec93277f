// Block-128 fp8 quantisation (format: fp8.cuh) of a matrix x [R, K] in bf16, fp16 or fp32.
//
//   fp8_quantize_rows    1 x 128 blocks along K: codes [R, Kp], one warp per row and 512 columns
//   fp8_quantize_tiles   128 x 128 tiles: codes of x (blocks 1 x 128), of x^T (blocks 1 x 128
//                        along R, for the weight gradient), or both from one read; or one
//                        scale per tile (weights), whose codes then serve both orientations
//
// Both are bound by memory: 2 or 4 bytes read and 1 (+ 1/128) written per element and side.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "fp8.cuh"

namespace osp {
namespace fp8 {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

// 8 consecutive elements of a row from column c; zeros from column K on.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int c, int K, float* v) {
  if (VEC && c + 8 <= K) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(row + c));
      const float4 b = __ldg(reinterpret_cast<const float4*>(row + c) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + c));
      const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f(h[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? to_f(row[c + i]) : 0.f;
  }
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = abs_bits(v);
  return b >= kInfBits ? 0u : b;
}

// ---------------------------------------------------------------------------- rows
// A lane owns 16 consecutive columns, so 8 lanes own a block (3 shuffles for its maximum), a
// lane's codes are one 16-byte store and a warp's four scales one 4-byte word.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, long ld, uint8_t* __restrict__ q,
                                                            uint8_t* __restrict__ scale, int R, int K, int Kp,
                                                            int kgroups, long total) {
  const int lane = threadIdx.x & 31;
  const long w = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= total) return;
  const long r = w / kgroups;
  const int kg = (int)(w - r * kgroups);
  uint32_t* word = reinterpret_cast<uint32_t*>(scale + scale_offset(r, 4 * kg, kgroups));
  if (r >= R) {
    if (lane == 0) *word = 0;
    return;
  }
  const int c = kg * 512 + lane * 16;
  float v[16];
  load8<T, VEC>(x + r * ld, c, K, v);
  load8<T, VEC>(x + r * ld, c + 8, K, v + 8);
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) amax = max(amax, abs_bits(v[i]));
  const bool bad = __any_sync(0xffffffffu, amax >= kInfBits);
  if (bad) {
    amax = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = max(amax, finite_bits(v[i]));
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const uint32_t byte = scale_byte(amax);
  const float inv = inv_scale(byte);
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] *= inv;
  if (bad) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = nan_if_inf(v[i]);
  }
  uint4 o;
  o.x = cvt4(v[0], v[1], v[2], v[3]);
  o.y = cvt4(v[4], v[5], v[6], v[7]);
  o.z = cvt4(v[8], v[9], v[10], v[11]);
  o.w = cvt4(v[12], v[13], v[14], v[15]);
  if (c < Kp) *reinterpret_cast<uint4*>(q + r * Kp + c) = o;
  uint32_t mine = c < Kp ? byte << (8 * (lane >> 3)) : 0u;
  mine |= __shfl_xor_sync(0xffffffffu, mine, 8);
  mine |= __shfl_xor_sync(0xffffffffu, mine, 16);
  if (lane == 0) *word = mine;
}

// ---------------------------------------------------------------------------- tiles
// One CTA per 128 x 128 tile; a thread holds 8 rows x 8 columns, a warp 32 x 64 (4 x 8
// threads), so that row loads are 128-byte segments, row codes 64-byte and column codes
// 32-byte ones without a pass through shared memory.
template <typename T, bool VEC, bool TILE_SCALE, bool ROWS, bool COLS>
__global__ void __launch_bounds__(256) quantize_tiles_kernel(const T* __restrict__ x, long ld,
                                                             uint8_t* __restrict__ q, uint8_t* __restrict__ scale,
                                                             uint8_t* __restrict__ qt, uint8_t* __restrict__ scale_t,
                                                             int R, int K, int Kp, int Rp) {
  __shared__ uint32_t rmax[2][128];
  __shared__ uint32_t cmax[4][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wr = warp >> 1, wc = warp & 1;
  const int rl = wr * 32 + (lane >> 3) * 8;        // first row of this thread in the tile
  const int cl = wc * 64 + (lane & 7) * 8;         // first column
  const int kb = blockIdx.x, rb = blockIdx.y;
  const long r0 = (long)rb * 128 + rl;
  const int c0 = kb * 128 + cl;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (r0 + i < R) {
      load8<T, VEC>(x + (r0 + i) * ld, c0, K, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[i][j]));
  const bool bad = __syncthreads_or(top >= kInfBits);
  uint32_t ra[8], ca[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) ra[i] = ca[i] = 0;
  if (!bad) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t b = abs_bits(v[i][j]);
        ra[i] = max(ra[i], b);
        ca[j] = max(ca[j], b);
      }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t b = finite_bits(v[i][j]);
        ra[i] = max(ra[i], b);
        ca[j] = max(ca[j], b);
      }
  }
  uint32_t rbyte[8], cbyte[8];
  if constexpr (TILE_SCALE) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, ra[i]);
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) rmax[0][warp] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, rmax[0][i]);
    m = scale_byte(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) rbyte[i] = cbyte[i] = m;
  } else {
    if constexpr (ROWS) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) ra[i] = max(ra[i], __shfl_xor_sync(0xffffffffu, ra[i], o));
      if ((lane & 7) == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) rmax[wc][rl + i] = ra[i];
      }
    }
    if constexpr (COLS) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int o = 8; o < 32; o <<= 1) ca[j] = max(ca[j], __shfl_xor_sync(0xffffffffu, ca[j], o));
      if (lane < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) cmax[wr][cl + j] = ca[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (ROWS) rbyte[i] = scale_byte(max(rmax[0][rl + i], rmax[1][rl + i]));
      if constexpr (COLS)
        cbyte[i] = scale_byte(max(max(cmax[0][cl + i], cmax[1][cl + i]), max(cmax[2][cl + i], cmax[3][cl + i])));
    }
  }
  if (bad) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = nan_if_inf(v[i][j]);
  }
  // scale bytes: 128 rows of this tile's block, and zeros for what the last chunk lacks
  if constexpr (ROWS) {
    const int kgroups = (gridDim.x + 3) >> 2;
    if ((lane & 7) == 0 && wc == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint8_t* s = scale + scale_offset(r0 + i, kb, kgroups);
        *s = r0 + i < R ? (uint8_t)rbyte[i] : 0;
        if (kb == gridDim.x - 1)
          for (int j = 1; j < 4 - (kb & 3); ++j) s[j] = 0;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float inv = inv_scale(rbyte[i]);
      uint2 o;
      o.x = cvt4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
      o.y = cvt4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
      if (r0 + i < R) *reinterpret_cast<uint2*>(q + (r0 + i) * Kp + c0) = o;
    }
  }
  if constexpr (COLS) {
    const int rgroups = (gridDim.y + 3) >> 2;
    if (lane < 8 && wr == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint8_t* s = scale_t + scale_offset(c0 + j, rb, rgroups);
        *s = c0 + j < K ? (uint8_t)cbyte[j] : 0;
        if (rb == gridDim.y - 1)
          for (int i = 1; i < 4 - (rb & 3); ++i) s[i] = 0;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float inv = inv_scale(cbyte[j]);
      uint2 o;
      o.x = cvt4(v[0][j] * inv, v[1][j] * inv, v[2][j] * inv, v[3][j] * inv);
      o.y = cvt4(v[4][j] * inv, v[5][j] * inv, v[6][j] * inv, v[7][j] * inv);
      if (c0 + j < K) *reinterpret_cast<uint2*>(qt + (long)(c0 + j) * Rp + r0) = o;
    }
  }
}

}  // namespace fp8

static void check_side(const at::Tensor& x, const at::Tensor& q, const at::Tensor& s, int64_t rows, int64_t cols) {
  const int64_t cp = (cols + 127) / 128 * 128;
  TORCH_CHECK(q.is_cuda() && q.get_device() == x.get_device() && q.scalar_type() == at::kFloat8_e4m3fn &&
              q.is_contiguous() && q.dim() == 2 && q.size(0) == rows && q.size(1) == cp,
              "fp8_quantize: codes e4m3 [", std::to_string(rows), ", ", std::to_string(cp), "]");
  TORCH_CHECK(s.is_cuda() && s.get_device() == x.get_device() && s.scalar_type() == at::kByte && s.is_contiguous() &&
              s.numel() == (rows + 127) / 128 * ((cols + 511) / 512) * 512, "fp8_quantize: packed scales");
}

template <typename T>
static void quantize_t(const at::Tensor& x, uint8_t* q, uint8_t* s, uint8_t* qt, uint8_t* st, bool tile_scale,
                       cudaStream_t stream) {
  const int R = (int)x.size(0), K = (int)x.size(1);
  const int Kp = (K + 127) / 128 * 128, Rp = (R + 127) / 128 * 128;
  const long ld = x.stride(0);
  const T* xp = reinterpret_cast<const T*>(x.data_ptr());
  const bool vec = reinterpret_cast<uintptr_t>(xp) % 16 == 0 && (ld * (long)sizeof(T)) % 16 == 0;
  if (!tile_scale && qt == nullptr) {
    const int kgroups = (K + 511) / 512;
    const long total = (long)Rp * kgroups;
    const unsigned grid = (unsigned)((total + 7) / 8);
    if (vec) fp8::quantize_rows_kernel<T, true><<<grid, 256, 0, stream>>>(xp, ld, q, s, R, K, Kp, kgroups, total);
    else fp8::quantize_rows_kernel<T, false><<<grid, 256, 0, stream>>>(xp, ld, q, s, R, K, Kp, kgroups, total);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    return;
  }
  const dim3 grid(Kp / 128, Rp / 128);
  TORCH_CHECK(grid.y <= 65535, "fp8_quantize: more than 8388480 rows");
#define OSP_TILES(VEC, TS, RO, CO) \
  fp8::quantize_tiles_kernel<T, VEC, TS, RO, CO><<<grid, 256, 0, stream>>>(xp, ld, q, s, qt, st, R, K, Kp, Rp)
#define OSP_TILES_SIDES(VEC, TS)                      \
  do {                                                \
    if (q && qt) OSP_TILES(VEC, TS, true, true);      \
    else if (q) OSP_TILES(VEC, TS, true, false);      \
    else OSP_TILES(VEC, TS, false, true);             \
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
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// x [R, K] (rows contiguous, any row stride) -> q [R, Kp], s and / or those of x^T, qt [K, Rp], st
void fp8_quantize(const at::Tensor& x, const c10::optional<at::Tensor>& q, const c10::optional<at::Tensor>& s,
                  const c10::optional<at::Tensor>& qt, const c10::optional<at::Tensor>& st, bool tile_scale) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && (x.size(1) <= 1 || x.stride(1) == 1), "fp8_quantize: x [R, K] on the GPU, rows contiguous");
  const int64_t R = x.size(0), K = x.size(1);
  TORCH_CHECK(R < (int64_t(1) << 31) - 128 && K < (int64_t(1) << 31) - 512, "fp8_quantize: sizes below 2^31");
  TORCH_CHECK(q.has_value() == s.has_value() && qt.has_value() == st.has_value() && (q.has_value() || qt.has_value()),
              "fp8_quantize: codes and scales of at least one side");
  if (q.has_value()) check_side(x, *q, *s, R, K);
  if (qt.has_value()) check_side(x, *qt, *st, K, R);
  if (R == 0 || K == 0) return;
  c10::cuda::CUDAGuard guard(x.device());
  auto stream = c10::cuda::getCurrentCUDAStream();
  auto ptr = [](const c10::optional<at::Tensor>& t) {
    return t.has_value() ? reinterpret_cast<uint8_t*>(t->data_ptr()) : nullptr;
  };
  switch (x.scalar_type()) {
    case at::kBFloat16: quantize_t<__nv_bfloat16>(x, ptr(q), ptr(s), ptr(qt), ptr(st), tile_scale, stream); break;
    case at::kHalf: quantize_t<__half>(x, ptr(q), ptr(s), ptr(qt), ptr(st), tile_scale, stream); break;
    case at::kFloat: quantize_t<float>(x, ptr(q), ptr(s), ptr(qt), ptr(st), tile_scale, stream); break;
    default: TORCH_CHECK(false, "fp8_quantize: x bf16, fp16 or fp32");
  }
}

}  // namespace osp
