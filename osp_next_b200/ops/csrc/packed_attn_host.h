// Host checks and tensor maps of the packed attention launchers.
#pragma once
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAStream.h>

#include "packed_attn.cuh"
#include "tma_host.h"

namespace osp {
namespace pa {

struct Shape {
  int Nq, Nk, Hq, Hkv, D, G;
};

// `t` [N, H, D] as TMA can read it: itself where its last dim is contiguous and rows and heads lie at
// multiples of 16 bytes (none of them broadcast), else a copy.
static inline at::Tensor tma_rows(const at::Tensor& t) {
  if (t.dim() != 3 || t.numel() == 0) return t;
  const bool fits = t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                    (t.size(1) == 1 || (t.stride(1) > 0 && t.stride(1) % 8 == 0)) &&
                    (t.size(0) == 1 || (t.stride(0) > 0 && t.stride(0) % 8 == 0));
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

// A [N, H, D] tensor that TMA can read as it lies.
static inline void check_operand(const at::Tensor& x, const at::Tensor& q, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.device() == q.device(), what, ": CUDA tensors on one device");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 && x.dim() == 3, what, ": bf16 [tokens, heads, head_dim]");
  TORCH_CHECK(x.size(0) < (1ll << 31) && x.size(1) < 65536, what, ": too many rows or heads");
  TORCH_CHECK(x.numel() == 0 || (x.stride(2) == 1 && (x.size(1) == 1 || (x.stride(1) > 0 && x.stride(1) % 8 == 0)) &&
              (x.size(0) == 1 || (x.stride(0) > 0 && x.stride(0) % 8 == 0)) &&
              reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0),
              what, ": rows and heads at multiples of 16 bytes, last dim contiguous");
}

static inline Shape check_shapes(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const char* what) {
  check_operand(q, q, what);
  check_operand(k, q, what);
  check_operand(v, q, what);
  Shape s;
  s.Nq = (int)q.size(0);
  s.Nk = (int)k.size(0);
  s.Hq = (int)q.size(1);
  s.Hkv = (int)k.size(1);
  s.D = (int)q.size(2);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(2) == s.D, what, ": k and v [tokens, key heads, head_dim]");
  TORCH_CHECK(s.D % 8 == 0 && s.D <= 128, what, ": head_dim a multiple of 8 up to 128");
  TORCH_CHECK(s.Hkv > 0 && s.Hq % s.Hkv == 0 && s.Hq / s.Hkv <= kRows, what,
              ": query heads a multiple of key heads, at most 128 to one");
  s.G = s.Hq / s.Hkv;
  return s;
}

// A work list; its memory is not given away before the work that is now on this stream is done.
static inline void check_list(const at::Tensor& t, int width, const at::Tensor& q, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == q.device() && t.scalar_type() == at::kInt && t.is_contiguous() &&
              t.dim() == 2 && t.size(1) == width, what);
  if (t.numel() > 0) t.record_stream(c10::cuda::getCurrentCUDAStream(q.get_device()).unwrap());
}

// [N, H, D] as a 3-D tensor (D, H, N) with boxes of 64 elements x heads x positions (128B swizzle);
// elements from D on and rows from N on read as zeros.  A tensor without rows is never read: its map
// is of `other`.
static inline CUtensorMap tile_map(const at::Tensor& x, const at::Tensor& other, int D, int heads, int positions) {
  const at::Tensor& t = x.numel() > 0 ? x : other;
  const uint64_t hs = t.size(1) == 1 ? (uint64_t)D : (uint64_t)t.stride(1);
  const uint64_t rs = t.size(0) == 1 ? hs * t.size(1) : (uint64_t)t.stride(0);
  uint64_t dims[3] = {(uint64_t)D, (uint64_t)t.size(1), (uint64_t)t.size(0)};
  uint64_t strides[2] = {hs, rs};
  uint32_t box[3] = {64, (uint32_t)heads, (uint32_t)positions};
  return make_tmap_bf16(t.data_ptr(), 3, dims, strides, box);
}

}  // namespace pa
}  // namespace osp
