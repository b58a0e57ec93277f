// Rotary positions of q and k in one launch: interleaved or half layout, part of the head, positions of
// one or several axes, cosines and sines from a table (rotary_table in ops/rotary.py evaluates it in 64
// bits, scaled for long contexts or not).
//
//   pair i of a head: (a, b) -> (a c - b s, a s + b c),  (c, s) = table[pos[axis(i)], i]
//   pairs: elements (2 i, 2 i + 1) interleaved, (i, i + R / 2) half layout; elements from R on are copied
//
// Bound by memory: each value is read and written once, and the R / 2 pairs of a token's table row
// serve all heads of q and k.  A warp takes one token: its lanes hold the cosines and sines of the
// vector pieces that they own in registers and pass over the heads, so that a table entry is read once
// per token and not once per head, with four heads' loads in flight.  The inverse (gradients) turns by -s.
// 80640 tokens x 80 heads of 128 in bf16: 492 us, 6.8 TB/s (one head at a time 570); 14039 x 20 in fp32,
// half of each head: 53 us, 5.4 TB/s (67).
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <string>

#include "common.cuh"
#include "tma_host.h"

namespace osp {
namespace rotary {

struct Tensor {
  const void* in;
  void* out;                   // [n, heads, D], contiguous
  long row, head;              // strides of `in` in elements
  int heads;
};

struct Args {
  Tensor t[2];
  const void* pos;             // [n, axes], int32 or int64
  int pos64;
  const float2* table;         // [positions, R / 2]
  long n;
  int axes, positions;
  int D, R;
  int end[4];                  // axis a owns pairs end[a - 1] .. end[a] - 1
  float sign;                  // 1, or -1 for the inverse
  int* err;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec { T v[V]; };

// V values and their fp32 form; 16-bit ones two at a time (one conversion instruction each way).
template <int V>
__device__ __forceinline__ void widen(const Vec<float, V>& x, float* f) {
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = x.v[j];
}
template <int V>
__device__ __forceinline__ void widen(const Vec<__half, V>& x, float* f) {
  if constexpr (V == 1) {
    f[0] = __half2float(x.v[0]);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&x.v[j]));
      f[j] = p.x;
      f[j + 1] = p.y;
    }
  }
}
template <int V>
__device__ __forceinline__ void widen(const Vec<__nv_bfloat16, V>& x, float* f) {
  if constexpr (V == 1) {
    f[0] = __bfloat162float(x.v[0]);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x.v[j]));
      f[j] = p.x;
      f[j + 1] = p.y;
    }
  }
}
template <int V>
__device__ __forceinline__ void narrow(Vec<float, V>& x, const float* f) {
#pragma unroll
  for (int j = 0; j < V; ++j) x.v[j] = f[j];
}
template <int V>
__device__ __forceinline__ void narrow(Vec<__half, V>& x, const float* f) {
  if constexpr (V == 1) {
    x.v[0] = __float2half_rn(f[0]);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) *reinterpret_cast<__half2*>(&x.v[j]) = __floats2half2_rn(f[j], f[j + 1]);
  }
}
template <int V>
__device__ __forceinline__ void narrow(Vec<__nv_bfloat16, V>& x, const float* f) {
  if constexpr (V == 1) {
    x.v[0] = __float2bfloat16(f[0]);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) *reinterpret_cast<__nv_bfloat162*>(&x.v[j]) = __floats2bfloat162_rn(f[j], f[j + 1]);
  }
}

// kHeads pieces (and, in the half layout, their partners `far` elements on), `step` elements apart,
// all loads in flight before the first is used.
template <typename T, int V, bool kHalf, int kHeads>
__device__ __forceinline__ void turn_pieces(const T* src, T* dst, long in_step, int out_step, int far, bool turn,
                                            const float2* cs) {
  Vec<T, V> a[kHeads], b[kHeads];
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    a[u] = *reinterpret_cast<const Vec<T, V>*>(src + u * in_step);
    if (kHalf && turn) b[u] = *reinterpret_cast<const Vec<T, V>*>(src + u * in_step + far);
  }
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    if (turn) {
      float fa[V], fb[V], x[V], y[V];
      widen<V>(a[u], fa);
      if constexpr (kHalf) {
        widen<V>(b[u], fb);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x[j] = fa[j] * cs[j].x - fb[j] * cs[j].y;
          y[j] = fa[j] * cs[j].y + fb[j] * cs[j].x;
        }
        narrow<V>(b[u], y);
        *reinterpret_cast<Vec<T, V>*>(dst + u * out_step + far) = b[u];
      } else {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          x[j] = fa[j] * cs[j / 2].x - fa[j + 1] * cs[j / 2].y;
          x[j + 1] = fa[j] * cs[j / 2].y + fa[j + 1] * cs[j / 2].x;
        }
      }
      narrow<V>(a[u], x);
    }
    *reinterpret_cast<Vec<T, V>*>(dst + u * out_step) = a[u];
  }
}

// Entry i of the positions, -1 where it lies outside the table; 64-bit ones are compared as they are.
__device__ __forceinline__ int position(const Args& a, long i) {
  const long long p = a.pos64 ? static_cast<const long long*>(a.pos)[i] : static_cast<const int*>(a.pos)[i];
  return p >= 0 && p < a.positions ? (int)p : -1;
}

// Cosine and sine of pair i; at: the token's places on the axes.
__device__ __forceinline__ float2 pair_of(const Args& a, const int (&at)[4], int i) {
  int p = at[0];
#pragma unroll
  for (int axis = 1; axis < 4; ++axis)
    if (axis < a.axes && i >= a.end[axis - 1]) p = at[axis];
  const float2 cs = a.table[(long)p * (a.R / 2) + i];
  return make_float2(cs.x, cs.y * a.sign);
}

// One piece = V elements of a pair's first half and V of its second (half layout), or V elements
// (V / 2 pairs, interleaved; also the copied elements).  Pieces of a head: half layout R / 2 / V and
// (D - R) / V to copy, interleaved D / V.
// Four heads of fp32 in flight are held to 64 registers, four blocks an SM (14039 x 20 in fp32, half of each
// head: 53 us; in the 78 that they take otherwise 58).
template <typename T, int V, bool kHalf, int kPieces, int kHeads>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && kHeads == 4 ? 4 : 1)
rotate(const Args args) {
  const long token = (long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (token >= args.n) return;
  const int lane = threadIdx.x % 32;
  const int R = args.R, D = args.D;
  const int turned = kHalf ? R / 2 / V : R / V;
  const int pieces = turned + (D - R) / V;
  const int mine = lane < args.axes ? position(args, token * args.axes + lane) : 0;
  if (__any_sync(0xffffffffu, mine < 0)) {   // no such position on some axis: a token of NaN and an error for the host
#pragma unroll 1
    for (int w = 0; w < 2; ++w) {
      const long size = (long)args.t[w].heads * D;
      T* dst = reinterpret_cast<T*>(args.t[w].out) + token * size;
      Vec<T, 1> nan;
      const float value = NAN;
      narrow<1>(nan, &value);
      for (long i = lane; i < size; i += 32) dst[i] = nan.v[0];
    }
    if (lane == 0) record_error(args.err, kErrRotaryPosition);
    return;
  }
  int at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) at[i] = __shfl_sync(0xffffffffu, mine, i);
  // heads are dealt so that a warp is full: `per` lanes to a head, 32 / per heads at a time
  int per = 1;
  while (per < pieces && per < 32) per <<= 1;
  const int sub = lane % per, group = lane / per, groups = 32 / per;
  float2 cs[kPieces][V];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int p = sub + k * per;
    if (p < turned) {
#pragma unroll
      for (int j = 0; j < (kHalf ? V : V / 2); ++j)
        cs[k][j] = pair_of(args, at, p * (kHalf ? V : V / 2) + j);
    }
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const Tensor& t = args.t[w];
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int p = sub + k * per;
      if (p >= pieces) continue;
      const bool turn = p < turned;
      const int o = turn ? p * V : R + (p - turned) * V;     // this piece's place in the head
      const T* src = reinterpret_cast<const T*>(t.in) + token * t.row + group * t.head + o;
      T* dst = reinterpret_cast<T*>(t.out) + (token * t.heads + group) * D + o;
      const long in_step = groups * t.head;
      const int out_step = groups * D;
      int h = group;
      for (; h + (kHeads - 1) * groups < t.heads; h += kHeads * groups) {
        turn_pieces<T, V, kHalf, kHeads>(src, dst, in_step, out_step, R / 2, turn, cs[k]);
        src += kHeads * in_step;
        dst += kHeads * out_step;
      }
      for (; h < t.heads; h += groups) {
        turn_pieces<T, V, kHalf, 1>(src, dst, in_step, out_step, R / 2, turn, cs[k]);
        src += in_step;
        dst += out_step;
      }
    }
  }
}

template <typename T, int V, bool kHalf>
static void launch(const Args& a, cudaStream_t stream) {
  const unsigned blocks = (unsigned)((a.n + 7) / 8);
  const int turned = kHalf ? a.R / 2 / V : a.R / V;
  const int pieces = turned + (a.D - a.R) / V;
  if (pieces <= 32) rotate<T, V, kHalf, 1, 4><<<blocks, 256, 0, stream>>>(a);
  else if (pieces <= 64) rotate<T, V, kHalf, 2, 2><<<blocks, 256, 0, stream>>>(a);
  else rotate<T, V, kHalf, 8, 1><<<blocks, 256, 0, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <typename T>
static void launch_type(const Args& a, bool half, int vec, cudaStream_t stream) {
  constexpr int W = 16 / sizeof(T);
  if (half) {
    if (vec == W) launch<T, W, true>(a, stream);
    else if (vec == 2) launch<T, 2, true>(a, stream);
    else launch<T, 1, true>(a, stream);
  } else {
    if (vec == W) launch<T, W, false>(a, stream);
    else launch<T, 2, false>(a, stream);
  }
}

}  // namespace rotary

// Rotated copies of q [..., n, Hq, D] and, if given, k [..., n, Hk, D].  pos [n] or [n, axes]; table fp32
// [positions, R / 2, 2]; sections: pairs of each axis (their sum R / 2), or empty for one axis.
std::vector<at::Tensor> rotary_apply(const at::Tensor& q, const c10::optional<at::Tensor>& k, const at::Tensor& pos_,
                                     const at::Tensor& table_, const std::vector<int64_t>& sections, bool half,
                                     bool inverse) {
  using namespace rotary;
  const char* what = "rotary: ";
  TORCH_CHECK(q.is_cuda() && q.dim() >= 3 && table_.dim() == 3, what, "CUDA q [..., tokens, heads, head_dim]");
  const int64_t tokens = q.size(-3), D = q.size(-1), R = 2 * table_.size(1);
  int64_t lead = 1;
  for (int64_t i = 0; i + 3 < q.dim(); ++i) lead *= q.size(i);
  const int64_t n = lead * tokens, axes = std::max<int64_t>(1, (int64_t)sections.size());
  TORCH_CHECK(pos_.device() == q.device() && at::isIntegralType(pos_.scalar_type(), false) &&
              (pos_.dim() == 1 || pos_.dim() == 2) && pos_.size(0) == tokens &&
              (pos_.dim() == 1 ? axes == 1 : pos_.size(1) == axes) && axes <= 4,
              what, "whole positions [tokens] or [tokens, axes], 1 to 4 axes");
  TORCH_CHECK(table_.device() == q.device() && table_.scalar_type() == at::kFloat && table_.size(2) == 2 &&
              table_.size(0) < (1ll << 31), what, "table fp32 [positions, pairs, 2]");
  TORCH_CHECK(R <= D && D <= 256 && D % 2 == 0, what, "table of ", std::to_string(R / 2), " pairs for a head dim of ",
              std::to_string(D), " (even, at most 256)");
  TORCH_CHECK(n < (1ll << 31), what, "too many tokens");
  c10::cuda::CUDAGuard guard(q.device());
  // types whose values fit 32 bits are read as int32
  const at::ScalarType pt = pos_.scalar_type();
  const bool narrow = pt == at::kInt || pt == at::kShort || pt == at::kChar || pt == at::kByte || pt == at::kUInt16;
  at::Tensor pos = pos_.to(narrow ? at::kInt : at::kLong).contiguous();
  if (lead > 1) pos = pos.view({tokens, axes}).repeat({lead, 1});
  const at::Tensor table = table_.contiguous();
  Args a{};
  std::vector<at::Tensor> in, out;
  const int size = (int)q.element_size(), wide = 16 / size;
  in.push_back(q);
  if (k.has_value()) in.push_back(*k);
  // every piece lies in the turned or in the copied part
  int fit = wide;
  while (fit > 1 && ((half ? R / 2 : R) % fit || (D - R) % fit)) fit >>= 1;
  int vec = fit;
  for (size_t i = 0; i < in.size(); ++i) {
    const at::Tensor& x = in[i];
    TORCH_CHECK(x.device() == q.device() && x.scalar_type() == q.scalar_type() && x.dim() == q.dim() &&
                x.size(-1) == D, what, "q and k [..., tokens, heads, head_dim] of one type");
    for (int64_t j = 0; j + 2 < q.dim(); ++j)
      TORCH_CHECK(x.size(j) == q.size(j), what, "q and k of as many tokens");
    out.push_back(at::empty(x.sizes(), x.options()));
    if (x.dim() != 3) in[i] = x.reshape({n, x.size(-2), D});
    auto fits = [&](const at::Tensor& t, int v) {
      return t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % (v * size) == 0 && t.stride(0) % v == 0 &&
             t.stride(1) % v == 0;
    };
    if (in[i].numel() > 0) {
      if (in[i].stride(2) != 1) in[i] = in[i].contiguous();
      // pairs at odd addresses: one aligned copy
      if (!half && !fits(in[i], 2)) in[i] = in[i].clone(at::MemoryFormat::Contiguous);
      while (vec > 1 && !fits(in[i], vec)) vec >>= 1;
    }
    a.t[i] = {in[i].data_ptr(), out[i].data_ptr(), in[i].stride(0), in[i].stride(1), (int)in[i].size(1)};
  }
  int64_t end = 0;
  for (int64_t i = 0; i < axes; ++i) {
    const int64_t pairs = sections.empty() ? R / 2 : sections[i];
    TORCH_CHECK(pairs >= 0, what, "sections from 0 on");
    a.end[i] = (int)(end += pairs);
  }
  TORCH_CHECK(end == R / 2, what, "sections of ", std::to_string(end), " pairs, table of ", std::to_string(R / 2));
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf || q.scalar_type() == at::kFloat, what,
              "bf16, fp16 or fp32");
  if (n == 0 || D == 0) {
    for (size_t i = 0; i < in.size(); ++i) out[i].copy_(q.dim() == 3 ? in[i] : in[i].view(out[i].sizes()));
    return out;
  }
  vec = vec == wide ? wide : vec >= 2 ? 2 : 1;
  a.pos = pos.data_ptr();
  a.pos64 = narrow ? 0 : 1;
  a.table = reinterpret_cast<const float2*>(table.data_ptr<float>());
  TORCH_CHECK(reinterpret_cast<uintptr_t>(a.table) % 8 == 0, what, "table at a multiple of 8 bytes");
  a.n = n;
  a.axes = (int)axes;
  a.positions = (int)table.size(0);
  a.D = (int)D;
  a.R = (int)R;
  a.sign = inverse ? -1.0f : 1.0f;
  a.err = error_word(q.get_device());
  auto stream = c10::cuda::getCurrentCUDAStream();
  switch (q.scalar_type()) {
    case at::kBFloat16: launch_type<__nv_bfloat16>(a, half, vec, stream); break;
    case at::kHalf: launch_type<__half>(a, half, vec, stream); break;
    default: launch_type<float>(a, half, vec, stream);
  }
  return out;
}

}  // namespace osp
