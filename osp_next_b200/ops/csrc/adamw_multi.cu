// AdamW over a list of tensors in one launch per 480 of them (the framework's per-tensor kernel
// is adamw in misc.cu), with the moments in fp32 or in 8 bits.
//
//   g' = g grad_scale;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit moments: each run of 128 elements of a tensor has one power-of-two scale per moment
// (byte e = log2 + 127, the smallest that brings the largest magnitude into range).  m is e4m3;
// v is the top byte of an IEEE half without its sign (5 exponent bits, 3 mantissa bits,
// largest value 61440, 255 = NaN): the square needs twice the exponent range and no sign.
// Both are rounded stochastically: at b2 = 0.999 a step changes v by a thousandth, far below
// half a step of 3 mantissa bits (3 to 6 %), so nearest rounding would never let v move; with
// probability in proportion to the remainder the stored averages stay unbiased.  A positive v
// is never stored as 0, which would divide the next m by eps alone.  The update itself uses
// the unrounded moments.
//
// It has to move 16 bytes per element with fp32 p and g and 8-bit moments (28 with fp32 ones); 177M
// elements in 820 tensors take 498 us, 0.87 of the copy rate, held up by some 64 instructions
// per element.  A warp takes 128 elements at a time, so the block maximum is one warp reduction
// and each of its loads and stores is one contiguous segment.  The list travels in the kernel's
// parameters (up to 32 KB): no table is copied or kept between calls.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <cmath>

#include "common.cuh"
#include "fp8.cuh"
#include "launch.h"

namespace osp {
namespace adamw8 {

constexpr int kCap = 480;                 // tensors per launch: 480 x 64 B + constants < 32764 B
constexpr int kSmallCap = 64;
constexpr int kGroups = 512;              // steps of the table from a chunk to its tensor
constexpr int kChunkBlocks = 32;          // 128-element runs per CTA (8 warps x 4)
constexpr uint32_t kMix1 = 0x6A09E667u, kMix2 = 0xBB67AE85u, kMix3 = 0x3C6EF373u;   // fractions of sqrt 2, 3, 5

// c1 = 1 - b1, c2 = 1 - b2, keep = 1 - lr wd, rate = lr / (1 - b1^t), inv_bc2s = 1 / sqrt(1 - b2^t): formed in
// 64 bits on the host (1 - fp32(0.999) alone would be off by a 75000th).
struct Consts {
  float b1, b2, c1, c2, eps, keep, rate, inv_bc2s, gscale;
};
template <int CAP>
struct Args {
  void* p[CAP];
  const void* g[CAP];
  void* m[CAP];
  void* v[CAP];
  uint8_t* ms[CAP];
  uint8_t* vs[CAP];
  int64_t n[CAP];
  int chunk_end[CAP];                     // chunks of tensors 0..i
  uint32_t key[CAP];
  uint16_t group[kGroups + 1];            // tensor of chunk g << shift; the last tensor from the end on
  int shift;
  int tensors;
  Consts c;
};
static_assert(sizeof(Args<kCap>) <= 32764, "kernel parameters");

__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x = (x ^ (x >> 16)) * kMix1;
  x = (x ^ (x >> 15)) * kMix2;
  return x ^ (x >> 16);
}

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 ld4(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void st4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void st4(__nv_bfloat16* p, float4 v) {
  uint2 u;
  u.x = pack_bf16x2(v.x, v.y);
  u.y = pack_bf16x2(v.z, v.w);
  *reinterpret_cast<uint2*>(p) = u;
}
__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

// Four elements, of which `left` (1..4) exist; `wide`: aligned for one vector access.
template <typename T>
__device__ __forceinline__ void load(const T* p, bool wide, int left, float* o) {
  if (wide && left >= 4) {
    const float4 f = ld4(p);
    o[0] = f.x; o[1] = f.y; o[2] = f.z; o[3] = f.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = j < left ? ld1(p + j) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store(T* p, bool wide, int left, const float* o) {
  if (wide && left >= 4) {
    st4(p, make_float4(o[0], o[1], o[2], o[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) st1(p + j, o[j]);
  }
}
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, bool wide, int left) {
  if (wide && left >= 4) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t u = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) u |= (uint32_t)p[j] << (8 * j);
  return u;
}
__device__ __forceinline__ void store_codes(uint8_t* p, bool wide, int left, uint32_t u) {
  if (wide && left >= 4) {
    *reinterpret_cast<uint32_t*>(p) = u;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) p[j] = (uint8_t)(u >> (8 * j));
}

__device__ __forceinline__ void decode_m(uint32_t u, uint32_t byte, float* o) {
  const float s = __uint_as_float(byte << 23);
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u & 0xFFFF), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u >> 16), __NV_E4M3);
  const float2 fa = __half22float2(__half2(a)), fb = __half22float2(__half2(b));
  o[0] = fa.x * s; o[1] = fa.y * s; o[2] = fb.x * s; o[3] = fb.y * s;
}
__device__ __forceinline__ void decode_v(uint32_t u, uint32_t byte, float* o) {
  const float s = __uint_as_float(byte << 23);
  const uint32_t lo = __byte_perm(u, 0, 0x4140) << 7, hi = __byte_perm(u, 0, 0x4342) << 7;
  const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  o[0] = fa.x * s; o[1] = fa.y * s; o[2] = fb.x * s; o[3] = fb.y * s;
}

// Stochastic rounding of a scaled magnitude a on its fp32 bits: add 20 random bits (16 and
// four zeros) below the three mantissa bits kept, then cut.  Below the least normal 2^-E the
// kept bits of a + 2^-E have the subnormal step; its pattern less one exponent exceeds that of
// a exactly there, so a maximum chooses between the two.  Returned with the eight bits that
// matter on top; the exponent offset, a multiple of half a byte's range, is left to one XOR on
// four packed codes (0x40 for m, 0x80 for v).
__device__ __forceinline__ uint32_t round_bits(float a, float least, uint32_t r16) {
  const uint32_t t = __viaddmax_u32(__float_as_uint(a + least), 0u - (1u << 23), __float_as_uint(a));
  return (r16 * 16u + t) << 4;
}
__device__ __forceinline__ uint32_t pack_top(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
// Largest magnitude of four as fp32 bits (NaN wins).
__device__ __forceinline__ uint32_t top4(const float* x) {
  float t;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(t) : "f"(x[0]), "f"(x[1]), "f"(x[2]));
  asm("max.NaN.abs.f32 %0, %0, %1, %1;" : "+f"(t) : "f"(x[3]));
  return __float_as_uint(t);
}
// Scale byte of a block of v: 61440 = 1.875 * 2^15.
__device__ __forceinline__ uint32_t scale_byte_v(uint32_t vmax) {
  return (uint32_t)max((int)((vmax + 0x0FFFFFu) >> 23) - 15, 1);
}

// sqrt and division of the update by the hardware approximations (relative errors of a few
// 2^-23, on a term that is lr times a number near 1); the precise forms cost some 30
// instructions per element, which is what bounded the 8-bit step.
__device__ __forceinline__ float sqrt_fast(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float stepped(float p, float m, float v, const Consts& c) {
  return p * c.keep - c.rate * __fdividef(m, sqrt_fast(v) * c.inv_bc2s + c.eps);
}

__device__ __forceinline__ void update32(float* pv, const float* gv, float* mv, float* vv, const Consts& c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float gj = gv[j] * c.gscale;
    mv[j] = c.b1 * mv[j] + c.c1 * gj;
    vv[j] = c.b2 * vv[j] + c.c2 * gj * gj;
    pv[j] = stepped(pv[j], mv[j], vv[j], c);
  }
}

// One block of 128 over a warp: codes mu, vu of four elements per lane and the block's scale
// bytes mb, vb in, their new values out; p updated.  `i`: index of the lane's first element.
__device__ __forceinline__ void update8(float* pv, const float* gv, uint32_t& mu, uint32_t& vu, uint32_t& mb,
                                        uint32_t& vb, uint32_t i, uint32_t key, const Consts& c) {
  float mv[4], vv[4];
  decode_m(mu, mb, mv);
  decode_v(vu, vb, vv);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // written with explicit roundings (no contraction), so that the stored codes are
    // reproducible from the formula
    const float gj = __fmul_rn(gv[j], c.gscale);
    mv[j] = __fadd_rn(__fmul_rn(mv[j], c.b1), __fmul_rn(gj, c.c1));
    vv[j] = __fadd_rn(__fmul_rn(vv[j], c.b2), __fmul_rn(__fmul_rn(gj, gj), c.c2));
    pv[j] = stepped(pv[j], mv[j], vv[j], c);
  }
  uint32_t mtop = __reduce_max_sync(0xffffffffu, top4(mv));
  uint32_t vtop = __reduce_max_sync(0xffffffffu, top4(vv));
  const bool bad = max(mtop, vtop) >= fp8::kInfBits;
  if (bad) {                                         // whole warp: maxima of what is finite
    mtop = vtop = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = __float_as_uint(mv[j]) & 0x7FFFFFFFu, y = __float_as_uint(vv[j]) & 0x7FFFFFFFu;
      mtop = max(mtop, x >= fp8::kInfBits ? 0u : x);
      vtop = max(vtop, y >= fp8::kInfBits ? 0u : y);
    }
    mtop = __reduce_max_sync(0xffffffffu, mtop);
    vtop = __reduce_max_sync(0xffffffffu, vtop);
  }
  mb = fp8::scale_byte(mtop);
  vb = scale_byte_v(vtop);
  const float minv = fp8::inv_scale(mb), vinv = fp8::inv_scale(vb);
  uint32_t um[4], uv[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t r = mix(i + j + key);
    const uint32_t m7 = round_bits(fabsf(mv[j]) * minv, 0.015625f, __byte_perm(r, 0, 0x4410));        // 2^-6
    um[j] = (m7 & 0x7FFFFFFFu) | (__float_as_uint(mv[j]) & 0x80000000u);
    uv[j] = round_bits(vv[j] * vinv, 6.103515625e-05f, __byte_perm(r, 0, 0x4432));                    // 2^-14
  }
  mu = pack_top(um[0], um[1], um[2], um[3]) ^ 0x40404040u;
  vu = pack_top(uv[0], uv[1], uv[2], uv[3]) ^ 0x80808080u;
  if ((vu - 0x01010101u) & ~vu & 0x80808080u) {      // some code is 0: a positive v takes 1
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (vv[j] > 0.f && ((vu >> (8 * j)) & 0xFFu) == 0) vu |= 1u << (8 * j);
  }
  if (bad) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!isfinite(mv[j])) mu |= 0x7Fu << (8 * j);
      if (!isfinite(vv[j])) vu |= 0xFFu << (8 * j);
    }
  }
}

// One tensor as a kernel sees it, and the state of one block of it in a lane's registers.
template <typename PT, typename GT> struct View {
  PT* p;
  const GT* g;
  void *m, *v;
  uint8_t *ms, *vs;
  int64_t n;
  uint32_t key;
  bool wide;                              // every pointer allows vectors of four elements
};
template <typename PT, typename GT, bool STATE8> struct Lane {
  float p[4], g[4];
  float m[STATE8 ? 1 : 4], v[STATE8 ? 1 : 4];
  uint32_t mu, vu, mb, vb;

  __device__ __forceinline__ void read(const View<PT, GT>& t, int64_t blk, int lane, bool wide, int left) {
    const int64_t i = blk * 128 + lane * 4;
    load(t.p + i, wide, left, p);
    load(t.g + i, wide, left, g);
    if constexpr (STATE8) {
      mu = load_codes(static_cast<const uint8_t*>(t.m) + i, wide, left);
      vu = load_codes(static_cast<const uint8_t*>(t.v) + i, wide, left);
      mb = t.ms[blk];
      vb = t.vs[blk];
    } else {
      load(static_cast<const float*>(t.m) + i, wide, left, m);
      load(static_cast<const float*>(t.v) + i, wide, left, v);
    }
  }
  __device__ __forceinline__ void step(const View<PT, GT>& t, int64_t blk, int lane, const Consts& c) {
    if constexpr (STATE8) update8(p, g, mu, vu, mb, vb, (uint32_t)(blk * 128 + lane * 4), t.key, c);
    else update32(p, g, m, v, c);
  }
  __device__ __forceinline__ void write(const View<PT, GT>& t, int64_t blk, int lane, bool wide, int left) const {
    const int64_t i = blk * 128 + lane * 4;
    store(t.p + i, wide, left, p);
    if constexpr (STATE8) {
      store_codes(static_cast<uint8_t*>(t.m) + i, wide, left, mu);
      store_codes(static_cast<uint8_t*>(t.v) + i, wide, left, vu);
      if (lane == 0) {
        t.ms[blk] = (uint8_t)mb;
        t.vs[blk] = (uint8_t)vb;
      }
    } else {
      store(static_cast<float*>(t.m) + i, wide, left, m);
      store(static_cast<float*>(t.v) + i, wide, left, v);
    }
  }
};

// One CTA per chunk of 32 blocks; a warp takes 4 neighbouring ones, with the loads of all in
// flight (177M elements in 820 tensors, before the table of groups: 548 us, with 2 a warp 591).
// Many short CTAs beat resident ones that loop over chunks: 64M elements took 172 us, 209 to 227
// in a loop (a warp's next loads there queue behind its byte-sized scale stores), and dealing
// contiguous runs of chunks to resident CTAs with a register prefetch was slower still.
template <typename PT, typename GT, bool STATE8, int CAP>
__global__ void __launch_bounds__(256, 3) step_kernel(const __grid_constant__ Args<CAP> args) {
  constexpr int U = kChunkBlocks / 8;
  grid_dependency_wait();
  allow_dependents();
  const Consts c = args.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunk = blockIdx.x;
  // first tensor with chunk < chunk_end: one of those that the chunk's group touches, mostly one or
  // two (a search over the whole list: 177M elements in 820 tensors took 536 us, not 492)
  int lo = args.group[chunk >> args.shift], hi = args.group[(chunk >> args.shift) + 1];
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (chunk < args.chunk_end[mid]) hi = mid;
    else lo = mid + 1;
  }
  View<PT, GT> t;
  t.p = static_cast<PT*>(args.p[lo]);
  t.g = static_cast<const GT*>(args.g[lo]);
  t.m = args.m[lo];
  t.v = args.v[lo];
  t.ms = args.ms[lo];
  t.vs = args.vs[lo];
  t.n = args.n[lo];
  t.key = args.key[lo];
  constexpr uintptr_t kState = STATE8 ? 3 : 15;
  t.wide = ((reinterpret_cast<uintptr_t>(t.p) & (4 * sizeof(PT) - 1)) |
            (reinterpret_cast<uintptr_t>(t.g) & (4 * sizeof(GT) - 1)) |
            ((reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) & kState)) == 0;
  const int64_t blk = (int64_t)(chunk - (lo ? args.chunk_end[lo - 1] : 0)) * kChunkBlocks + warp * U;
  Lane<PT, GT, STATE8> x[U];
  if (t.wide && (blk + U) * 128 <= t.n) {
#pragma unroll
    for (int u = 0; u < U; ++u) x[u].read(t, blk + u, lane, true, 4);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u].step(t, blk + u, lane, c);
      x[u].write(t, blk + u, lane, true, 4);
    }
  } else {                                           // a tensor's end, and odd addresses
#pragma unroll 1
    for (int u = 0; u < U; ++u) {
      if ((blk + u) * 128 >= t.n) break;             // whole warp
      const int left = (int)min((int64_t)4, t.n - (blk + u) * 128 - lane * 4);   // below 1: this lane has none
      x[0].read(t, blk + u, lane, t.wide, left);
      x[0].step(t, blk + u, lane, c);
      x[0].write(t, blk + u, lane, t.wide, left);
    }
  }
}

template <typename PT, typename GT, int CAP>
static void launch(const Args<CAP>& a, bool state8, cudaStream_t stream) {
  const int grid = a.chunk_end[a.tensors - 1];       // chunks, below 2^31
  launch_kernel(state8 ? step_kernel<PT, GT, true, CAP> : step_kernel<PT, GT, false, CAP>, grid, 256, 0, 1, stream, a);
}

// An in-place write that autograd's version counter sees, as one by a torch function does.
static void count_write(const at::Tensor* t) {
  if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

using Ptrs = std::vector<const at::Tensor*>;
struct Lists {
  const Ptrs &p, &g, &m, &v, &ms, &vs;
};

// Fills parameter blocks of CAP tensors and launches each.
template <int CAP>
static void run(const Lists& l, const Consts& consts, bool state8, uint32_t seed, cudaStream_t stream) {
  const bool pf = l.p[0]->scalar_type() == at::kFloat, gf = l.g[0]->scalar_type() == at::kFloat;
  Args<CAP> a;
  a.c = consts;
  a.tensors = 0;
  int64_t chunks = 0;
  auto flush = [&]() {
    if (a.tensors == 0) return;
    a.shift = 0;
    while ((chunks - 1) >> a.shift >= kGroups) ++a.shift;
    const int groups = (int)((chunks - 1) >> a.shift) + 1;
    for (int g = 0, t = 0; g <= groups; ++g) {
      while (t < a.tensors - 1 && (int64_t)g << a.shift >= a.chunk_end[t]) ++t;
      a.group[g] = (uint16_t)t;
    }
    if (pf && gf) launch<float, float, CAP>(a, state8, stream);
    else if (pf) launch<float, __nv_bfloat16, CAP>(a, state8, stream);
    else if (gf) launch<__nv_bfloat16, float, CAP>(a, state8, stream);
    else launch<__nv_bfloat16, __nv_bfloat16, CAP>(a, state8, stream);
    a.tensors = 0;
    chunks = 0;
  };
  for (size_t i = 0; i < l.p.size(); ++i) {
    const int64_t n = l.p[i]->numel();
    if (n == 0) continue;
    const int64_t mine = ((n + 127) / 128 + kChunkBlocks - 1) / kChunkBlocks;
    TORCH_CHECK(mine < (int64_t(1) << 30), "adamw_multi_: tensor ", std::to_string(i), " too large");
    if (a.tensors == CAP || chunks + mine >= (int64_t(1) << 31)) flush();
    const int t = a.tensors++;
    chunks += mine;
    a.p[t] = l.p[i]->data_ptr();
    a.g[t] = l.g[i]->data_ptr();
    a.m[t] = l.m[i]->data_ptr();
    a.v[t] = l.v[i]->data_ptr();
    a.ms[t] = state8 ? l.ms[i]->data_ptr<uint8_t>() : nullptr;
    a.vs[t] = state8 ? l.vs[i]->data_ptr<uint8_t>() : nullptr;
    a.n[t] = n;
    a.chunk_end[t] = (int)chunks;
    a.key[t] = mix((uint32_t)i * kMix3 + seed);
  }
  flush();
}

}  // namespace adamw8

// In place on every tensor of the lists; ms / vs empty: fp32 moments.
void adamw_multi(const std::vector<const at::Tensor*>& p, const std::vector<const at::Tensor*>& g,
                 const std::vector<const at::Tensor*>& m, const std::vector<const at::Tensor*>& v,
                 const std::vector<const at::Tensor*>& ms, const std::vector<const at::Tensor*>& vs, double lr,
                 double b1, double b2, double eps, double wd, int64_t step, double gscale, int64_t seed) {
  using namespace adamw8;
  const size_t count = p.size();
  const bool state8 = !ms.empty() || !vs.empty();
  TORCH_CHECK(g.size() == count && m.size() == count && v.size() == count &&
              (!state8 || (ms.size() == count && vs.size() == count)), "adamw_multi_: lists of one length");
  if (count == 0) return;
  TORCH_CHECK(step >= 1, "adamw_multi_: step counts from 1");
  const auto pt = p[0]->scalar_type(), gt = g[0]->scalar_type();
  TORCH_CHECK(pt == at::kFloat || pt == at::kBFloat16, "adamw_multi_: parameters fp32 or bf16");
  TORCH_CHECK(gt == at::kFloat || gt == at::kBFloat16, "adamw_multi_: gradients fp32 or bf16");
  TORCH_CHECK(p[0]->is_cuda(), "adamw_multi_: CUDA tensors");
  const c10::Device dev = p[0]->device();
  const auto mt = state8 ? at::kFloat8_e4m3fn : at::kFloat, vt = state8 ? at::kByte : at::kFloat;
  auto good = [&](const at::Tensor* t, at::ScalarType dt, int64_t n) {
    return t->device() == dev && t->scalar_type() == dt && t->numel() == n && t->is_contiguous();
  };
  for (size_t i = 0; i < count; ++i) {
    const int64_t n = p[i]->numel();
    TORCH_CHECK(good(p[i], pt, n) && good(g[i], gt, n) && good(m[i], mt, n) && good(v[i], vt, n),
                "adamw_multi_: tensor ", std::to_string(i), ": p, g and moments contiguous, of one size and device, p and g of one "
                "type throughout, moments ", state8 ? "e4m3 and uint8" : "fp32");
    if (state8)
      TORCH_CHECK(good(ms[i], at::kByte, (n + 127) / 128) && good(vs[i], at::kByte, (n + 127) / 128),
                  "adamw_multi_: tensor ", std::to_string(i), ": one uint8 scale per 128 elements and moment");
  }
  c10::cuda::CUDAGuard guard(dev);
  auto stream = c10::cuda::getCurrentCUDAStream();
  Consts c;
  c.b1 = (float)b1;
  c.b2 = (float)b2;
  c.c1 = (float)(1.0 - b1);
  c.c2 = (float)(1.0 - b2);
  c.eps = (float)eps;
  c.keep = (float)(1.0 - lr * wd);
  c.rate = (float)(lr / (1.0 - std::pow(b1, (double)step)));
  c.inv_bc2s = (float)(1.0 / std::sqrt(1.0 - std::pow(b2, (double)step)));
  c.gscale = (float)gscale;
  const Lists lists{p, g, m, v, ms, vs};
  // a short list has a small parameter block: 4 KB instead of 30 KB to copy with the launch
  if (count <= kSmallCap) run<kSmallCap>(lists, c, state8, (uint32_t)seed, stream);
  else run<kCap>(lists, c, state8, (uint32_t)seed, stream);
  for (const Ptrs* written : {&p, &m, &v, &ms, &vs})
    for (const at::Tensor* t : *written) count_write(t);
}

}  // namespace osp
