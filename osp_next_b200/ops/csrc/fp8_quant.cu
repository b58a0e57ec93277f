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
#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"

namespace osp {
namespace fp8 {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

// 8 consecutive elements of a row as they are in memory (16 bytes of a 16-bit type, 32 of fp32).
// `top` takes the larger magnitudes of two such pieces element by element, packed two to a
// register for 16-bit types (NaN wins, so that it is seen in the result); `bits(j)` is the
// magnitude of element j as fp32 bits.
template <typename T> struct Piece {
  uint4 r;
  __device__ __forceinline__ void load(const T* p) { r = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load_some(const T* p, int n) {
    uint16_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = i < n ? reinterpret_cast<const uint16_t*>(p)[i] : 0;
    r = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                   h[6] | (uint32_t)h[7] << 16);
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
  // packed magnitudes of two registers
  __device__ __forceinline__ static uint32_t top(uint32_t a, uint32_t b) {
    using P = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>::type;
    const P m = __hmax2_nan(__habs2(*reinterpret_cast<P*>(&a)), __habs2(*reinterpret_cast<P*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  __device__ __forceinline__ static uint32_t bits(uint32_t packed, int half) {
    return __float_as_uint(wide(packed, half)) & 0x7FFFFFFFu;
  }
  __device__ __forceinline__ uint32_t max_bits() const {
    const uint32_t m = top(top(r.x, r.y), top(r.z, r.w));
    return max(bits(m, 0), bits(m, 1));
  }
};
template <> struct Piece<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
  __device__ __forceinline__ void load_some(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
  }
  __device__ __forceinline__ void pin() {}
  __device__ __forceinline__ float get(int j) const { return v[j]; }
  __device__ __forceinline__ uint32_t max_bits() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
  }
};
// The piece at column c of a row of K; zeros from column K on.
template <typename T, bool VEC>
__device__ __forceinline__ void load_piece(Piece<T>& o, const T* row, int c, int K) {
  if (VEC && c + 8 <= K) o.load(row + c);
  else o.load_some(row + c, K - c);
}
template <typename T>
__device__ __forceinline__ uint32_t finite_max_bits(const Piece<T>& p) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = __float_as_uint(p.get(j)) & 0x7FFFFFFFu;
    m = max(m, b >= kInfBits ? 0u : b);
  }
  return m;
}

// ---------------------------------------------------------------------------- rows
// A lane owns 16 consecutive columns, so 8 lanes own a block (3 shuffles for its maximum), a
// lane's codes are one 16-byte store and a warp's four scales one 4-byte word.  A warp takes two
// such runs of 512 columns, with the loads of both in flight.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, long ld, uint8_t* __restrict__ q,
                                                            uint8_t* __restrict__ scale, int R, int K, int Kp,
                                                            int kgroups, long total) {
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
    uint32_t amax = max(v[u][0].max_bits(), v[u][1].max_bits());
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const bool bad = __any_sync(0xffffffffu, amax >= kInfBits);
    if (bad) {
      amax = max(finite_max_bits(v[u][0]), finite_max_bits(v[u][1]));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    const uint32_t byte = scale_byte(amax);
    const float inv = inv_scale(byte);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = v[u][i >> 1].get((i & 1) * 4 + j) * inv;
        if (bad) y[j] = nan_if_inf(y[j]);
      }
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
template <typename T, bool VEC, bool TILE_SCALE, bool ROWS, bool COLS>
__global__ void __launch_bounds__(256, 2)
quantize_tiles_kernel(const T* __restrict__ x, long ld, uint8_t* __restrict__ q, uint8_t* __restrict__ scale,
                      uint8_t* __restrict__ qt, uint8_t* __restrict__ scale_t, int R, int K, int Kp, int Rp) {
  __shared__ uint32_t rmax[2][128];
  __shared__ uint32_t cmax[4][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wr = warp >> 1, wc = warp & 1;
  const int rl = wr * 32 + (lane >> 3) * 8;        // first row of this thread in the tile
  const int cl = wc * 64 + (lane & 7) * 8;         // first column
  const int kb = blockIdx.x, rb = blockIdx.y;
  const long r0 = (long)rb * 128 + rl;
  const int c0 = kb * 128 + cl;
  Piece<T> v[8];
  if (VEC && (rb + 1) * 128L <= R && (kb + 1) * 128 <= K) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].load(x + (r0 + i) * ld + c0);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (r0 + i < R) load_piece<T, VEC>(v[i], x + (r0 + i) * ld, c0, K);
      else v[i].zero();
    }
  }
  // maxima of the thread's rows (over 8 columns) and columns (over 8 rows), then over the warp
  uint32_t ra[8], ca[8];
  auto gather = [&](bool finite) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ra[i] = finite ? finite_max_bits(v[i]) : v[i].max_bits();
      ca[i] = 0;
    }
    if constexpr (COLS && !TILE_SCALE) {
      if (sizeof(T) == 2 && !finite) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t m = Piece<T>::top(v[0].reg(k), v[1].reg(k));
#pragma unroll
            for (int i = 2; i < 8; ++i) m = Piece<T>::top(m, v[i].reg(k));
#pragma unroll
            for (int o = 8; o < 32; o <<= 1) m = Piece<T>::top(m, __shfl_xor_sync(0xffffffffu, m, o));
            ca[2 * k] = Piece<T>::bits(m, 0);
            ca[2 * k + 1] = Piece<T>::bits(m, 1);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t b = __float_as_uint(v[i].get(j)) & 0x7FFFFFFFu;
            ca[j] = max(ca[j], finite && b >= kInfBits ? 0u : b);
          }
#pragma unroll
          for (int o = 8; o < 32; o <<= 1) ca[j] = max(ca[j], __shfl_xor_sync(0xffffffffu, ca[j], o));
        }
      }
      if (lane < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) cmax[wr][cl + j] = ca[j];
      }
    }
    if constexpr (TILE_SCALE) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, ra[i]);
      m = __reduce_max_sync(0xffffffffu, m);
      if (lane == 0) rmax[0][warp] = m;
      ra[0] = m;
    } else if constexpr (ROWS) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) ra[i] = max(ra[i], __shfl_xor_sync(0xffffffffu, ra[i], o));
      if ((lane & 7) == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) rmax[wc][rl + i] = ra[i];
      }
    }
  };
  gather(false);
  bool over = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) over |= ra[i] >= kInfBits;
  const bool bad = __syncthreads_or(over);
  if (bad) {                                       // maxima of what is finite
    gather(true);
    __syncthreads();
  }
  uint32_t tile_byte = 0;
  if constexpr (TILE_SCALE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) tile_byte = max(tile_byte, rmax[0][i]);
    tile_byte = scale_byte(tile_byte);
  }
  auto value = [&](int i, int j, float inv) {
    const float y = v[i].get(j) * inv;
    return bad ? nan_if_inf(y) : y;
  };
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i].pin();
  // scale bytes: 128 rows of this tile's block, and zeros for what the last chunk lacks
  if constexpr (ROWS) {
    const int kgroups = (gridDim.x + 3) >> 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t byte = TILE_SCALE ? tile_byte : scale_byte(max(rmax[0][rl + i], rmax[1][rl + i]));
      if ((lane & 7) == 0 && wc == 0) {
        uint8_t* s = scale + scale_offset(r0 + i, kb, kgroups);
        *s = r0 + i < R ? (uint8_t)byte : 0;
        if (kb == gridDim.x - 1)
          for (int j = 1; j < 4 - (kb & 3); ++j) s[j] = 0;
      }
      const float inv = inv_scale(byte);
      uint2 o;
      o.x = cvt4(value(i, 0, inv), value(i, 1, inv), value(i, 2, inv), value(i, 3, inv));
      o.y = cvt4(value(i, 4, inv), value(i, 5, inv), value(i, 6, inv), value(i, 7, inv));
      if (r0 + i < R) *reinterpret_cast<uint2*>(q + (r0 + i) * Kp + c0) = o;
    }
  }
  if constexpr (COLS) {
    const int rgroups = (gridDim.y + 3) >> 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].pin();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t byte = TILE_SCALE ? tile_byte
                                       : scale_byte(max(max(cmax[0][cl + j], cmax[1][cl + j]),
                                                        max(cmax[2][cl + j], cmax[3][cl + j])));
      if (lane < 8 && wr == 0) {
        uint8_t* s = scale_t + scale_offset(c0 + j, rb, rgroups);
        *s = c0 + j < K ? (uint8_t)byte : 0;
        if (rb == gridDim.y - 1)
          for (int i = 1; i < 4 - (rb & 3); ++i) s[i] = 0;
      }
      const float inv = inv_scale(byte);
      uint2 o;
      o.x = cvt4(value(0, j, inv), value(1, j, inv), value(2, j, inv), value(3, j, inv));
      o.y = cvt4(value(4, j, inv), value(5, j, inv), value(6, j, inv), value(7, j, inv));
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
    const unsigned grid = (unsigned)((total + 15) / 16);
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
