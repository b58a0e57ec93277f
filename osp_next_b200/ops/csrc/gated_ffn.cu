// Gated feed-forward block:  h = act(x Wg^T) o (x Wu^T),  y = h Wd^T, and its gradients.
//
//   act(g) = g sigmoid(c (g)),  c(g) = g (SiLU) or 2 sqrt(2/pi) (g + 0.044715 g^3) (GELU, tanh form)
//   forward   one kernel forms both projections: a tile of 256 accumulator columns holds 128 of g and
//             the same 128 of u (TMA loads 128 rows of either weight behind one another, so no weight
//             is packed), and the epilogue writes act(g) u, in training g and u too
//   backward  dh = dy Wd with the epilogue  dg = dh u act'(g),  du = dh act(g),  h = act(g) u, which
//             also brings h back for dWd (it is not kept); then dx = dg Wg + du Wu as one product over
//             two operand pairs, [dWg; dWu] = [dg | du]^T x, dWd = dy^T h
//
// All are tiles of 128 x BN of one persistent kernel (a CTA per SM, 320 threads): warp 0 loads, warp 1
// issues tcgen05.mma into one of two accumulators, warps 2..9 are two groups of epilogue warps that take
// half of the tile's columns each.  Operands lie K-major or MN-major as the tensors are; results leave
// through shared memory as whole 64-byte row segments.  Sums are fp32 in tensor memory; g, u, dg, du and
// h are rounded to bf16 once, as operands of the next product have to be (dg, du, h; g and u: keep16).
//
// What bounds it: large blocks the power cap (20160 x 5120 -> 13824, training step: 20.4 ms, 1260 TFLOP/s; the
// gate kernel 1220, dx and the weight gradients 1320); few rows reading the weights (1 x 4096 -> 10240 ->
// 4096: 44 us, 0.87 of the copy rate; 154 rows 67 us).
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "launch.h"
#include <algorithm>
#include <string>

#include "tma_host.h"

namespace osp {
namespace ffn {

constexpr int kBM = 128, kBK = 64, kGroupM = 16, kThreads = 320;
constexpr int kRing = 196608;
constexpr int kStageRow = 80;                 // bytes per staged row (64 + 16 pad)
constexpr int kStageBytes = 32 * kStageRow;

enum Mode : int { kPlain = 0, kGate = 1, kGateBwd = 2 };
enum Act : int { kSilu = 0, kGeluTanh = 1 };

struct Args {
  int M, N, K, K2;             // result [M, N]; K2: depth of the second operand pair (kPlain)
  int act;
  __nv_bfloat16* out;          // kPlain: [M, N]; kGate: h [M, N]; kGateBwd: h [M, N]
  float* out32;                // kPlain: the result in fp32 instead (gradients of fp32 weights), or null
  uint16_t* gu;                // [M, 2 N]: g | u (keep16) written (kGate, or null), read (kGateBwd)
  __nv_bfloat16* dgu;          // [M, 2 N]: dg | du written (kGateBwd)
  int* err;
};

__device__ __forceinline__ float sigmoid_f(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

// act(g), and its derivative where asked for.  g sigmoid(z): tanh(a) = 2 sigmoid(2 a) - 1.
template <bool kGrad>
__device__ __forceinline__ float act_f(int act, float g, float& d) {
  float z = g, dz = 1.0f;
  if (act == kGeluTanh) {
    const float k = 1.5957691216057308f;      // 2 sqrt(2 / pi)
    const float g2 = g * g;
    z = k * g * fmaf(0.044715f, g2, 1.0f);
    if (kGrad) dz = k * fmaf(3.0f * 0.044715f, fminf(g2, 1e30f), 1.0f);   // finite: 0 times it stays 0
  }
  const float s = sigmoid_f(z);
  // act' = s + g s (1 - s) z'; far from 0 (1 - s) or s is 0
  if (kGrad) d = s + (g * s) * ((1.0f - s) * dz);
  return g * s;
}

// Projections kept for the backward pass in 16 bits: a sign and the place of the value among those with 9 bits of
// mantissa from 2^-20 to 2^16 and 6 bits below and above, over the whole range of fp32 (all ones for NaN and
// infinity).  As bf16 their rounding, 2^-9 of the value in the mean of a step's ends, would be as large as that of
// dg and du themselves and show in every gradient (weight gradients 3.5e-3 from 64 bits against 2.4e-3).
constexpr uint32_t kFine0 = 107u << 23, kFine1 = 143u << 23;      // 2^-20 and 2^16 as bits
constexpr uint32_t kCode0 = kFine0 >> 17, kCode1 = kCode0 + ((kFine1 - kFine0) >> 14);   // their codes
constexpr uint32_t kLow = (kFine0 >> 14) - kCode0, kHigh = kCode1 - (kFine1 >> 17);      // codes are cut bits -+ these
__device__ __forceinline__ uint32_t keep16(float v) {
  const uint32_t b = __float_as_uint(v), m = b & 0x7fffffffu;
  const bool fine = m - kFine0 < kFine1 - kFine0;
  const uint32_t near = (m + 0x1fffu + ((m >> 14) & 1u)) >> 14, far = (m + 0xffffu + ((m >> 17) & 1u)) >> 17;
  uint32_t t = fine ? near - kLow : far + (m >= kFine1 ? kHigh : 0u);
  t = m >= 0x7f800000u ? 0x7fffu : min(t, (0x7f800000u >> 17) + kHigh - 1u);   // the largest stay finite
  return ((b >> 16) & 0x8000u) | t;
}
__device__ __forceinline__ float kept(uint32_t c) {       // 16 bits
  const uint32_t t = c & 0x7fffu;
  uint32_t m = t < kCode0 ? t << 17 : t < kCode1 ? (t + kLow) << 14 : (t - kHigh) << 17;
  m = t == 0x7fffu ? 0x7fc00000u : m;
  return __uint_as_float(m | ((c & 0x8000u) << 16));
}
struct AsBf16 {
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};
struct AsKept {
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return keep16(a) | keep16(b) << 16; }
  static __device__ __forceinline__ float low(uint32_t w) { return kept(w & 0xffffu); }
  static __device__ __forceinline__ float high(uint32_t w) { return kept(w >> 16); }
};

__device__ __forceinline__ void tile_coords(int t, int num_m, int num_n, int& mb, int& nb) {
  const int per_group = kGroupM * num_n;
  const int g = t / per_group;
  const int first_m = g * kGroupM;
  const int gsize = min(num_m - first_m, kGroupM);
  const int r = t - g * per_group;
  mb = first_m + r % gsize;
  nb = r / gsize;
}

template <typename As>
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(As::pack(v[0], v[1]), As::pack(v[2], v[3]), As::pack(v[4], v[5]), As::pack(v[6], v[7]));
}
template <typename As>
__device__ __forceinline__ void unpack8(const uint4& w, float* v) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = As::low(r[i]);
    v[2 * i + 1] = As::high(r[i]);
  }
}

// A warp's 32 rows x 32 columns (a row per lane) to dst [rows of `pitch`], in 64-byte row segments.
template <typename As = AsBf16, typename T>
__device__ __forceinline__ void store_tile(const float* v, uint8_t* stg, T* dst, long pitch, long row0,
                                           int rows, int col0, int cols, int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(stg + lane * kStageRow + j * 16) = pack8<As>(v + 8 * j);
  __syncwarp();
  const int q = lane >> 2, cc = lane & 3;
  if (col0 + cc * 8 < cols) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = i * 8 + q;
      if (row0 + rr < rows)
        *reinterpret_cast<uint4*>(dst + (row0 + rr) * pitch + col0 + cc * 8) =
            *reinterpret_cast<const uint4*>(stg + rr * kStageRow + cc * 16);
    }
  }
  __syncwarp();
}
// The same way in: 32 columns of this lane's row, zeros outside.
template <typename As, typename T>
__device__ __forceinline__ void load_tile(float* v, uint8_t* stg, const T* src, long pitch, long row0,
                                          int rows, int col0, int cols, int lane) {
  const int q = lane >> 2, cc = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = i * 8 + q;
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (row0 + rr < rows && col0 + cc * 8 < cols)
      w = *reinterpret_cast<const uint4*>(src + (row0 + rr) * pitch + col0 + cc * 8);
    *reinterpret_cast<uint4*>(stg + rr * kStageRow + cc * 16) = w;
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) unpack8<As>(*reinterpret_cast<const uint4*>(stg + lane * kStageRow + j * 16), v + 8 * j);
  __syncwarp();
}

// kGate: the tile's BN accumulator columns are BN / 2 of g and BN / 2 of u; A [M, K], B1 = Wg, B2 = Wu.
// kPlain with K2 > 0: D = A1 B1^T + A2 B2^T.
template <int BN, int MODE, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kThreads, 1)
gemm(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
     const __grid_constant__ CUtensorMap tmA2, const __grid_constant__ CUtensorMap tmB2, const Args args) {
  constexpr uint32_t A_BYTES = kBM * kBK * 2, B_BYTES = BN * kBK * 2;
  constexpr int STAGES = kRing / (A_BYTES + B_BYTES);
  constexpr uint32_t MN_BOX = 64 * kBK * 2;
  constexpr uint32_t IDESC = idesc_bf16(kBM, BN, B_MN, A_MN);
  constexpr int OUT_N = MODE == kGate ? BN / 2 : BN;        // result columns of a tile

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint8_t* epi = sB + STAGES * B_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi + 8 * kStageBytes);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* done = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int num_m = (args.M + kBM - 1) / kBM;
  const int num_n = (args.N + OUT_N - 1) / OUT_N;
  const int num_tiles = num_m * num_n;
  const int num_kb1 = (args.K + kBK - 1) / kBK;
  const int num_kb = num_kb1 + (args.K2 + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tfull[a], 1); mbar_init(&tempty[a], 8); }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    if (MODE == kGate || args.K2 > 0) prefetch_tmap(&tmB2);
    if (args.K2 > 0) prefetch_tmap(&tmA2);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int t = blockIdx.x; t < num_tiles && !*abort_flag; t += gridDim.x) {
        int mb, nb;
        tile_coords(t, num_m, num_n, mb, nb);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, args.err, kErrGemmProducer)) { *abort_flag = 1; break; }
          mbar_expect_tx(&full[stage], A_BYTES + B_BYTES);
          const bool second = kb >= num_kb1;
          const CUtensorMap* ta = second ? &tmA2 : &tmA;
          const CUtensorMap* tb = second ? &tmB2 : &tmB;
          const int kc = (second ? kb - num_kb1 : kb) * kBK;
          uint8_t* a = sA + stage * A_BYTES;
          uint8_t* b = sB + stage * B_BYTES;
          if constexpr (A_MN) {
#pragma unroll
            for (int c = 0; c < kBM / 64; ++c) tma_load_2d(ta, &full[stage], a + c * MN_BOX, mb * kBM + 64 * c, kc);
          } else {
            tma_load_2d(ta, &full[stage], a, kc, mb * kBM);
          }
          if constexpr (MODE == kGate) {
            tma_load_2d(&tmB, &full[stage], b, kc, nb * OUT_N);
            tma_load_2d(&tmB2, &full[stage], b + B_BYTES / 2, kc, nb * OUT_N);
          } else if constexpr (B_MN) {
#pragma unroll
            for (int c = 0; c < BN / 64; ++c) tma_load_2d(tb, &full[stage], b + c * MN_BOX, nb * BN + 64 * c, kc);
          } else {
            tma_load_2d(tb, &full[stage], b, kc, nb * BN);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, it = 0;
      uint32_t phase = 0;
      for (int t = blockIdx.x; t < num_tiles && !*abort_flag; t += gridDim.x, ++it) {
        const int acc = it & 1;
        if (!mbar_wait(&tempty[acc], ((it >> 1) & 1) ^ 1, args.err, kErrGemmMma)) { *abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t d = tmem_base + acc * BN;
        bool ok = true;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full[stage], phase, args.err, kErrGemmMma)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a = smem_u32(sA + stage * A_BYTES), b = smem_u32(sB + stage * B_BYTES);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            const uint64_t ad = A_MN ? sdesc_sw128(a + k * 2048, MN_BOX, 1024) : sdesc_sw128(a + k * 32, 16, 1024);
            const uint64_t bd = B_MN ? sdesc_sw128(b + k * 2048, MN_BOX, 1024) : sdesc_sw128(b + k * 32, 16, 1024);
            umma_bf16(d, ad, bd, IDESC, (kb > 0 || k > 0) ? 1u : 0u);
          }
          umma_commit(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        umma_commit(&tfull[acc]);
        if (!ok) { *abort_flag = 1; break; }
      }
      umma_commit(done);
      mbar_wait(done, 0, args.err, kErrGemmTeardown);
    }
  } else {
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    uint8_t* stg = epi + (warp - 2) * kStageBytes;
    int it = 0;
    for (int t = blockIdx.x; t < num_tiles; t += gridDim.x, ++it) {
      if (*abort_flag) break;
      int mb, nb;
      tile_coords(t, num_m, num_n, mb, nb);
      const int acc = it & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], (it >> 1) & 1, args.err, kErrGemmEpilogue))) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const long row0 = (long)mb * kBM + quarter * 32;
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * BN;
#pragma unroll 1
      for (int c = half * (OUT_N / 64); c < (half + 1) * (OUT_N / 64); ++c) {
        const int col0 = nb * OUT_N + c * 32;
        if (col0 >= args.N) continue;                       // uniform across the warp
        uint32_t r[32];
        tmem_ld32(t_row + c * 32, r);
        float v[32];
        if constexpr (MODE == kGate) {
          uint32_t ru[32];
          tmem_ld32(t_row + BN / 2 + c * 32, ru);
          tmem_ld_wait();
          float u[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) { v[j] = __uint_as_float(r[j]); u[j] = __uint_as_float(ru[j]); }
          if (args.gu) {
            store_tile<AsKept>(v, stg, args.gu, 2l * args.N, row0, args.M, col0, args.N, lane);
            store_tile<AsKept>(u, stg, args.gu + args.N, 2l * args.N, row0, args.M, col0, args.N, lane);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float d;
            v[j] = act_f<false>(args.act, v[j], d) * u[j];
          }
        } else if constexpr (MODE == kGateBwd) {
          float g[32], u[32];
          load_tile<AsKept>(g, stg, args.gu, 2l * args.N, row0, args.M, col0, args.N, lane);
          load_tile<AsKept>(u, stg, args.gu + args.N, 2l * args.N, row0, args.M, col0, args.N, lane);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float d;
            const float a = act_f<true>(args.act, g[j], d), dh = __uint_as_float(r[j]);
            v[j] = a * u[j];
            g[j] = dh * u[j] * d;
            u[j] = dh * a;
          }
          store_tile(g, stg, args.dgu, 2l * args.N, row0, args.M, col0, args.N, lane);
          store_tile(u, stg, args.dgu + args.N, 2l * args.N, row0, args.M, col0, args.N, lane);
        } else {
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
        }
        if (MODE == kPlain && args.out32) {
          // a lane's row piece is a whole 128-byte line
          if (row0 + lane < args.M) {
            float4* o = reinterpret_cast<float4*>(args.out32 + (row0 + lane) * args.N + col0);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (col0 + 4 * j < args.N) o[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
        } else {
          store_tile(v, stg, args.out, args.N, row0, args.M, col0, args.N, lane);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

// ---------------------------------------------------------------------------- few rows
// Up to kFewRows rows of x: what takes time is reading the weights once.  The product is formed as
// W x^T, so that 128 weight rows fill the tensor core's M and the rows of x (padded to 16) its N; a
// CTA holds 128 rows of Wg and the same of Wu (two accumulators, so a thread owns g and u of its
// weight row), or 128 rows of Wd.  Two CTAs share an SM where their accumulators take 256 columns of
// tensor memory.  Tiles that are too few to fill the SMs split K over a cluster of up to 8 CTAs,
// whose parts are added through distributed shared memory in rank order: no workspace, and results do
// not depend on timing.  The down projection starts while the gate kernel runs and loads its first
// weights before it waits for it.  192 threads: warp 0 loads, warp 1 MMAs, warps 2..5 results.
// The same form serves the backward pass: dh = dy Wd with its epilogue and dx = dg Wg + du Wu read the
// weights as they lie, MN-major (kWMn).
struct FewArgs {
  int M, N, KB;                // rows of x, result columns, blocks of 64 along K (of both operand pairs)
  int KB1;                     // of the first pair
  int bnx;                     // rows of x that a CTA takes (blockIdx.y: which), a multiple of 16
  int stages;                  // of the ring
  int splits;
  int chunk;                   // rows of x whose sums fit the ring, a multiple of 16
  int cols;                    // tensor-memory columns
  int act;
  int ahead;                   // load weights before the wait for the kernel in front
  __nv_bfloat16* out;          // [M, N] (kPlain, or null; kGate, kGateBwd: h)
  float* out32;                // kPlain: the result in fp32 instead, or null
  uint16_t* gu;                // as in Args
  __nv_bfloat16* dgu;
  int* err;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {   // every warp of every CTA arrives converged
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 load_from_cta(const float* p, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

constexpr int kFewRows = 256;
constexpr int kFewThreads = 192;
constexpr int kFewMaxStages = 12;
constexpr uint32_t kWTile = 128 * kBK * 2;

template <int MODE, bool kWMn>
__global__ void __launch_bounds__(kFewThreads)
few_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
           const __grid_constant__ CUtensorMap tmX2, const __grid_constant__ CUtensorMap tmW2, const FewArgs args) {
  constexpr int kAcc = MODE == kGate ? 2 : 1;
  constexpr uint32_t MN_BOX = 64 * kBK * 2;
  const uint32_t x_bytes = args.bnx * kBK * 2;
  const uint32_t stage_bytes = kAcc * kWTile + x_bytes;
  const int stages = args.stages;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty = full + kFewMaxStages;
  uint64_t* tfull = empty + kFewMaxStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull + 1);
  uint8_t* ring = smem + 1024;
  float* part = reinterpret_cast<float*>(ring);            // [kAcc][chunk][128] over the ring when it is done with

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int split = args.splits > 1 ? (int)cluster_rank() : 0;
  const int tile = blockIdx.x / args.splits;
  const int x0 = blockIdx.y * args.bnx, my_rows = min(args.bnx, args.M - x0);
  const int kb0 = (int)((long)args.KB * split / args.splits), kb1 = (int)((long)args.KB * (split + 1) / args.splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(tfull, 1);
    fence_mbar_init();
    prefetch_tmap(&tmX);
    prefetch_tmap(&tmW);
    if (MODE == kGate || args.KB > args.KB1) prefetch_tmap(&tmW2);
    if (args.KB > args.KB1) prefetch_tmap(&tmX2);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, args.cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (warp != 0 || !args.ahead) {
    grid_dependency_wait();
    allow_dependents();
  }

  if (warp == 0) {
    if (lane == 0) {
      auto load_w = [&](int kb, int stage) {
        uint8_t* dst = ring + stage * stage_bytes;
        mbar_expect_tx(&full[stage], stage_bytes);
        if constexpr (MODE == kGate) {
          tma_load_2d(&tmW, &full[stage], dst, kb * kBK, tile * 128);
          tma_load_2d(&tmW2, &full[stage], dst + kWTile, kb * kBK, tile * 128);
        } else {
          const bool second = kb >= args.KB1;
          const CUtensorMap* tm = second ? &tmW2 : &tmW;
          const int kc = (second ? kb - args.KB1 : kb) * kBK;
          if constexpr (kWMn) {
            tma_load_2d(tm, &full[stage], dst, tile * 128, kc);
            tma_load_2d(tm, &full[stage], dst + MN_BOX, tile * 128 + 64, kc);
          } else {
            tma_load_2d(tm, &full[stage], dst, kc, tile * 128);
          }
        }
      };
      auto load_x = [&](int kb, int stage) {
        const bool second = MODE != kGate && kb >= args.KB1;
        tma_load_2d(second ? &tmX2 : &tmX, &full[stage], ring + stage * stage_bytes + kAcc * kWTile,
                    (second ? kb - args.KB1 : kb) * kBK, x0);
      };
      const int n = min(stages, kb1 - kb0);
      for (int i = 0; i < n; ++i) load_w(kb0 + i, i);
      if (args.ahead) grid_dependency_wait();
      for (int i = 0; i < n; ++i) load_x(kb0 + i, i);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0 + n; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase, args.err, kErrGemmProducer)) break;
        load_w(kb, stage);
        load_x(kb, stage);
        if (++stage == stages) { stage = 0; phase ^= 1; }
      }
      // the last loads have landed before the ring is reused and the block ends
      for (int s = 0; s < n; ++s) mbar_wait(&full[s], s < stage ? phase ^ 1 : phase, args.err, kErrGemmTeardown);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_bf16(128, args.bnx, false, kWMn);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[stage], phase, args.err, kErrGemmMma)) break;
        tc_fence_after();
        const uint32_t w = smem_u32(ring + stage * stage_bytes), x = w + kAcc * kWTile;
#pragma unroll
        for (int a = 0; a < kAcc; ++a)
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            umma_bf16(tmem + a * args.bnx,
                      kWMn ? sdesc_sw128(w + k * 2048, MN_BOX, 1024) : sdesc_sw128(w + a * kWTile + k * 32, 16, 1024),
                      sdesc_sw128(x + k * 32, 16, 1024), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
        umma_commit(&empty[stage]);
        if (++stage == stages) { stage = 0; phase ^= 1; }
      }
      umma_commit(tfull);
    }
    __syncwarp();
  }

  // Sums leave tensor memory (a lane per weight row) for shared memory, [row of x][128], and from there
  // a warp per row of x adds the parts of all CTAs and writes 128 results in one piece; as many rows
  // of x at a time as the ring has room for.
  const int quarter = warp & 3;
  const int n0 = tile * 128 + lane * 4;
  bool ok = true;
  if (warp >= 2) {
    ok = __all_sync(0xffffffffu, mbar_wait(tfull, 0, args.err, kErrGemmEpilogue));
    tc_fence_after();
  }
  for (int c0 = 0; c0 < my_rows; c0 += args.chunk) {
    const int rows = min(args.chunk, my_rows - c0);
    if (warp >= 2 && ok) {
      const uint32_t t_row = tmem + ((uint32_t)(quarter * 32) << 16) + c0;
      float* mine = part + quarter * 32 + lane;
      for (int m0 = 0; m0 < rows; m0 += 16) {              // rows of x from M on are zeros of the tile
        uint32_t r[kAcc][16];
#pragma unroll
        for (int a = 0; a < kAcc; ++a) tmem_ld16(t_row + a * args.bnx + m0, r[a]);
        tmem_ld_wait();
#pragma unroll
        for (int a = 0; a < kAcc; ++a)
#pragma unroll
          for (int j = 0; j < 16; ++j) mine[(a * args.chunk + m0 + j) * 128] = __uint_as_float(r[a][j]);
      }
    }
    if (args.splits > 1) cluster_sync();
    else __syncthreads();
    if (warp >= 2 && ok && n0 < args.N) {
#pragma unroll 2
      for (int m = split + (warp - 2) * args.splits; m < rows; m += 4 * args.splits) {
        float4 v[kAcc];
#pragma unroll
        for (int a = 0; a < kAcc; ++a) {
          const float* src = part + (a * args.chunk + m) * 128 + lane * 4;
          if (args.splits == 1) {
            v[a] = *reinterpret_cast<const float4*>(src);
          } else {
            float4 p[8];
#pragma unroll
            for (int s = 0; s < 8; ++s)
              if (s < args.splits) p[s] = load_from_cta(src, s);
            v[a] = p[0];
#pragma unroll
            for (int s = 1; s < 8; ++s)
              if (s < args.splits) { v[a].x += p[s].x; v[a].y += p[s].y; v[a].z += p[s].z; v[a].w += p[s].w; }
          }
        }
        const long at = (long)(x0 + c0 + m) * args.N + n0, at2 = (long)(x0 + c0 + m) * 2 * args.N + n0;
        float f[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, d;
        if constexpr (MODE == kGate) {
          const float u[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
          if (args.gu) {
            *reinterpret_cast<uint2*>(args.gu + at2) = make_uint2(AsKept::pack(f[0], f[1]), AsKept::pack(f[2], f[3]));
            *reinterpret_cast<uint2*>(args.gu + at2 + args.N) =
                make_uint2(AsKept::pack(u[0], u[1]), AsKept::pack(u[2], u[3]));
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = act_f<false>(args.act, f[e], d) * u[e];
        } else if constexpr (MODE == kGateBwd) {
          const uint2 wg = *reinterpret_cast<const uint2*>(args.gu + at2);
          const uint2 wu = *reinterpret_cast<const uint2*>(args.gu + at2 + args.N);
          const float g[4] = {AsKept::low(wg.x), AsKept::high(wg.x), AsKept::low(wg.y), AsKept::high(wg.y)};
          const float u[4] = {AsKept::low(wu.x), AsKept::high(wu.x), AsKept::low(wu.y), AsKept::high(wu.y)};
          float dg[4], du[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = act_f<true>(args.act, g[e], d);
            dg[e] = f[e] * u[e] * d;
            du[e] = f[e] * a;
            f[e] = a * u[e];
          }
          *reinterpret_cast<uint2*>(args.dgu + at2) = make_uint2(pack_bf16x2(dg[0], dg[1]), pack_bf16x2(dg[2], dg[3]));
          *reinterpret_cast<uint2*>(args.dgu + at2 + args.N) =
              make_uint2(pack_bf16x2(du[0], du[1]), pack_bf16x2(du[2], du[3]));
        }
        if (MODE == kPlain && args.out32)
          *reinterpret_cast<float4*>(args.out32 + at) = make_float4(f[0], f[1], f[2], f[3]);
        else
          *reinterpret_cast<uint2*>(args.out + at) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
      }
    }
    if (args.splits > 1) cluster_sync();                   // no CTA goes on while its part may be read
    else __syncthreads();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, args.cols);
  }
}

template <int BN>
constexpr int smem_bytes() {
  constexpr int stage = kBM * kBK * 2 + BN * kBK * 2;
  return 1024 + kRing / stage * stage + 8 * kStageBytes + (2 * (kRing / stage) + 5) * 8 + 16;
}

// A row-major matrix; `mn`: its rows run along K, boxes are 64 columns x kBK rows.
static CUtensorMap map_of(const at::Tensor& t, bool mn, int rows_box) {
  return make_tmap_2d_bf16(t.data_ptr(), t.size(1), t.size(0), t.stride(0), 64, mn ? kBK : rows_box);
}

template <int BN, int MODE, bool A_MN, bool B_MN>
static void launch(const at::Tensor& a, const at::Tensor& b, const at::Tensor* a2, const at::Tensor* b2, Args args,
                   cudaStream_t stream) {
  constexpr int b_rows = MODE == kGate ? BN / 2 : BN;
  const CUtensorMap ma = map_of(a, A_MN, kBM), mb = map_of(b, B_MN, b_rows);
  const CUtensorMap ma2 = a2 ? map_of(*a2, A_MN, kBM) : ma, mb2 = b2 ? map_of(*b2, B_MN, b_rows) : mb;
  auto kern = gemm<BN, MODE, A_MN, B_MN>;
  constexpr int smem = smem_bytes<BN>();
  smem_opt_in(reinterpret_cast<const void*>(kern), smem);
  constexpr int out_n = MODE == kGate ? BN / 2 : BN;
  const long tiles = ((long)args.M + kBM - 1) / kBM * ((args.N + out_n - 1) / out_n);
  kern<<<(unsigned)std::min<long>(tiles, num_sms(a.get_device())), kThreads, smem, stream>>>(ma, mb, ma2, mb2, args);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Whether the form for few rows takes a product: up to kFewRows of them (154 x 4096 -> 10240 -> 4096: 65 us
// against 124), and more where the tiles of the other form leave SMs idle.  Neither bound is the best for every
// size: 1536 -> 8960 -> 1536 takes 54 us at 256 rows and 47 at 300, where its gate product leaves this form, and
// tiles just above one wave (149 to some 220) take two waves of the other.
static bool few_rows(int64_t M, int64_t N, int out_n, int sms) {
  return M <= kFewRows || (M + kBM - 1) / kBM * ((N + out_n - 1) / out_n) < sms;
}

// The product of `args` (its sizes and pointers) in the form for few rows; weights [N, K], or [K, N] with kWMn.
template <int MODE, bool kWMn>
static void launch_few(const at::Tensor& x, const at::Tensor& w, const at::Tensor* x2, const at::Tensor* w2,
                       const Args& args, bool ahead, cudaStream_t stream) {
  const int sms = num_sms(x.get_device());
  constexpr int acc = MODE == kGate ? 2 : 1;
  FewArgs a{};
  a.M = args.M;
  a.N = args.N;
  a.KB1 = (args.K + kBK - 1) / kBK;
  a.KB = a.KB1 + (args.K2 + kBK - 1) / kBK;
  const int blocks = (a.M + kFewRows - 1) / kFewRows;
  a.bnx = ((a.M + blocks - 1) / blocks + 15) / 16 * 16;
  a.cols = 32;
  while (a.cols < acc * a.bnx) a.cols *= 2;
  const int stage = acc * (int)kWTile + a.bnx * kBK * 2;
  const bool two = a.cols <= 256 && 111 * 1024 / stage >= 3;     // CTAs per SM
  a.stages = std::min(kFewMaxStages, (two ? 111 : 224) * 1024 / stage);
  const int tiles = (a.N + 127) / 128;
  // as many parts of K as there is room for, of at least 4 blocks
  a.splits = std::max(1, std::min({8, (two ? 2 : 1) * sms / (tiles * blocks), a.KB / 4}));
  a.chunk = std::min(a.bnx, a.stages * stage / (acc * 512) / 16 * 16);
  a.act = args.act;
  a.ahead = ahead ? 1 : 0;
  a.out = args.out;
  a.out32 = args.out32;
  a.gu = args.gu;
  a.dgu = args.dgu;
  a.err = args.err;
  const CUtensorMap mx = map_of(x, false, a.bnx), mw = map_of(w, kWMn, 128);
  const CUtensorMap mx2 = x2 ? map_of(*x2, false, a.bnx) : mx, mw2 = w2 ? map_of(*w2, kWMn, 128) : mw;
  auto kern = few_kernel<MODE, kWMn>;
  smem_opt_in(reinterpret_cast<const void*>(kern), 227 * 1024);
  launch_kernel(kern, dim3(tiles * a.splits, blocks), kFewThreads, 2048 + a.stages * stage, a.splits, stream, mx, mw,
                mx2, mw2, a);
}

static void check(const at::Tensor& t, const at::Tensor& x, int64_t rows, int64_t cols, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 &&
              t.size(0) == rows && t.size(1) == cols, "gated_ffn: ", what, " bf16 [", std::to_string(rows), ", ", std::to_string(cols), "]");
  TORCH_CHECK(cols % 8 == 0 && t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= cols &&
              reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "gated_ffn: ", what,
              " in rows at multiples of 16 bytes");
  TORCH_CHECK(rows < (1ll << 30) && cols < (1ll << 30), "gated_ffn: ", what, " too large");
}

static Args make_args(const at::Tensor& x, int64_t M, int64_t N, int64_t K, int64_t act) {
  Args a{};
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.act = (int)act;
  a.err = error_word(x.get_device());
  return a;
}

}  // namespace ffn

at::Tensor ffn_product(const at::Tensor& a, const at::Tensor& b, const c10::optional<at::Tensor>& a2,
                       const c10::optional<at::Tensor>& b2, bool a_mn, bool b_mn, bool f32, bool ahead);

// {h [M, F]} or, with `keep`, {h, gu [M, 2 F]}: h = act(x wg^T) (x wu^T).
std::vector<at::Tensor> gated_linear_fwd(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, int64_t act,
                                         bool keep) {
  using namespace ffn;
  TORCH_CHECK(x.dim() == 2 && wg.dim() == 2, "gated_ffn: x [M, K], weights [F, K]");
  const int64_t M = x.size(0), K = x.size(1), F = wg.size(0);
  check(x, x, M, K, "x");
  check(wg, x, F, K, "gate weight");
  check(wu, x, F, K, "up weight");
  TORCH_CHECK(F % 8 == 0 && K > 0, "gated_ffn: F a multiple of 8");
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor h = at::empty({M, F}, x.options()), gu;
  if (keep) gu = at::empty({M, 2 * F}, x.options().dtype(at::kShort));
  if (M > 0 && F > 0) {
    Args a = make_args(x, M, F, K, act);
    a.out = reinterpret_cast<__nv_bfloat16*>(h.data_ptr());
    a.gu = keep ? reinterpret_cast<uint16_t*>(gu.data_ptr()) : nullptr;
    auto stream = c10::cuda::getCurrentCUDAStream();
    if (few_rows(M, F, 128, num_sms(x.get_device()))) launch_few<kGate, false>(x, wg, nullptr, &wu, a, false, stream);
    else launch<256, kGate, false, false>(x, wg, nullptr, &wu, a, stream);
  }
  return {h, gu};
}

// {y [..., C], x as a matrix, gu} of the whole block, gu with `keep` alone; nothing where an operand is not as the
// kernels read it (bf16, sizes multiples of 8, rows at multiples of 16 bytes): the caller then makes copies.
std::vector<at::Tensor> gated_ffn_fwd(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu,
                                      const at::Tensor& wd, int64_t act, bool keep) {
  auto fits = [&](const at::Tensor& t) {
    return t.is_cuda() && t.device() == x.device() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 &&
           t.size(0) > 0 && t.size(1) > 0 && t.size(1) % 8 == 0 && t.stride(1) == 1 && t.stride(0) % 8 == 0 &&
           t.stride(0) >= t.size(1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  };
  if (x.dim() < 1 || x.size(-1) == 0) return {};
  const int64_t K = x.size(-1);
  const at::Tensor x2 = x.dim() == 2 ? x : x.reshape({x.numel() / K, K});
  if (!fits(x2) || !fits(wg) || !fits(wu) || !fits(wd) || wg.size(1) != K || wu.sizes() != wg.sizes() ||
      wd.size(1) != wg.size(0) || wd.size(0) % 8 != 0 || act < 0 || act > 1)
    return {};
  auto h = gated_linear_fwd(x2, wg, wu, act, keep);
  at::Tensor y = ffn_product(h[0], wd, c10::nullopt, c10::nullopt, false, false, false, true);
  if (x.dim() != 2) {
    auto sizes = x.sizes().vec();
    sizes.back() = wd.size(0);
    y = y.view(sizes);
  }
  return {y, x2, h[1]};
}

// {h [M, F], dgu [M, 2 F]} of dy [M, C], wd [C, F] and the kept gu [M, 2 F].
std::vector<at::Tensor> gated_linear_bwd(const at::Tensor& dy, const at::Tensor& wd, const at::Tensor& gu, int64_t act) {
  using namespace ffn;
  TORCH_CHECK(dy.dim() == 2 && wd.dim() == 2, "gated_ffn: dy [M, C], down weight [C, F]");
  const int64_t M = dy.size(0), C = dy.size(1), F = wd.size(1);
  check(dy, dy, M, C, "output gradient");
  check(wd, dy, C, F, "down weight");
  TORCH_CHECK(gu.device() == dy.device() && gu.scalar_type() == at::kShort && gu.dim() == 2 && gu.size(0) == M &&
              gu.size(1) == 2 * F && gu.is_contiguous() && F % 8 == 0 && C > 0, "gated_ffn: contiguous kept projections, F a multiple of 8");
  c10::cuda::CUDAGuard guard(dy.device());
  at::Tensor h = at::empty({M, F}, dy.options()), dgu = at::empty({M, 2 * F}, dy.options());
  if (M > 0 && F > 0) {
    Args a = make_args(dy, M, F, C, act);
    a.out = reinterpret_cast<__nv_bfloat16*>(h.data_ptr());
    a.gu = reinterpret_cast<uint16_t*>(gu.data_ptr());
    a.dgu = reinterpret_cast<__nv_bfloat16*>(dgu.data_ptr());
    auto stream = c10::cuda::getCurrentCUDAStream();
    if (few_rows(M, F, 256, num_sms(dy.get_device())))
      launch_few<kGateBwd, true>(dy, wd, nullptr, nullptr, a, false, stream);
    else
      launch<256, kGateBwd, false, true>(dy, wd, nullptr, nullptr, a, stream);
  }
  return {h, dgu};
}

// `ahead`: the kernel in front on this stream is the gate kernel that wrote `a`.
// A B^T (+ A2 B2^T) in bf16 or fp32.  a [M, K] or, with a_mn, [K, M]; b [N, K] or, with b_mn, [K, N].
at::Tensor ffn_product(const at::Tensor& a, const at::Tensor& b, const c10::optional<at::Tensor>& a2,
                       const c10::optional<at::Tensor>& b2, bool a_mn, bool b_mn, bool f32, bool ahead) {
  using namespace ffn;
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2, "gated_ffn: matrices");
  const int64_t M = a.size(a_mn ? 1 : 0), K = a.size(a_mn ? 0 : 1), N = b.size(b_mn ? 1 : 0);
  check(a, a, a.size(0), a.size(1), "operand");
  check(b, a, b_mn ? K : N, b_mn ? N : K, "operand");
  TORCH_CHECK(N % 8 == 0 && a2.has_value() == b2.has_value(), "gated_ffn: result columns a multiple of 8");
  c10::cuda::CUDAGuard guard(a.device());
  Args args = make_args(a, M, N, K, 0);
  if (a2.has_value()) {
    check(*a2, a, a.size(0), a.size(1), "second operand");
    check(*b2, a, b.size(0), b.size(1), "second operand");
    args.K2 = (int)K;
  }
  at::Tensor out = at::empty({M, N}, f32 ? a.options().dtype(at::kFloat) : a.options());
  if (M == 0 || N == 0) return out;
  if (K == 0) return out.zero_();
  if (f32) args.out32 = out.data_ptr<float>();
  else args.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  const at::Tensor* pa = a2.has_value() ? &*a2 : nullptr;
  const at::Tensor* pb = b2.has_value() ? &*b2 : nullptr;
  auto stream = c10::cuda::getCurrentCUDAStream();
  TORCH_CHECK(b_mn || !a_mn, "gated_ffn: operand order");
  const bool few = !a_mn && few_rows(M, N, 256, num_sms(a.get_device()));
  if (few && b_mn) launch_few<kPlain, true>(a, b, pa, pb, args, ahead, stream);
  else if (few) launch_few<kPlain, false>(a, b, pa, pb, args, ahead, stream);
  else if (a_mn) launch<256, kPlain, true, true>(a, b, pa, pb, args, stream);
  else if (b_mn) launch<256, kPlain, false, true>(a, b, pa, pb, args, stream);
  else launch<256, kPlain, false, false>(a, b, pa, pb, args, stream);
  return out;
}

// Gradients {dx, dwg, dwu, dwd} of the block for dy [M, C], those that are asked for; in fp32 where `*32`.
// x, weights and gu as gated_ffn_fwd left them.
std::vector<at::Tensor> gated_ffn_bwd(const at::Tensor& dy_, const at::Tensor& x, const at::Tensor& wg,
                                      const at::Tensor& wu, const at::Tensor& wd, const at::Tensor& gu, int64_t act,
                                      bool need_x, bool need_g, bool need_u, bool need_d, bool x32, bool w32, bool d32) {
  const int64_t M = x.size(0), F = wg.size(0), C = wd.size(0);
  at::Tensor dy = dy_.to(at::kBFloat16);
  if (dy.dim() != 2) dy = dy.reshape({M, dy.size(-1)});
  TORCH_CHECK(dy.dim() == 2 && dy.size(0) == M && dy.size(1) == C, "gated_ffn: gradient of the output");
  if (dy.stride(1) != 1 || dy.stride(0) % 8 != 0 || dy.stride(0) < C ||
      reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 != 0)
    dy = dy.clone(at::MemoryFormat::Contiguous);
  auto hd = gated_linear_bwd(dy, wd, gu, act);
  const at::Tensor dg = hd[1].narrow(1, 0, F), du = hd[1].narrow(1, F, F);
  at::Tensor dx, dwg, dwu, dwd;
  if (need_x) dx = ffn_product(dg, wg, du, wu, false, true, x32, false);
  if (need_g && need_u) {
    const at::Tensor both = ffn_product(hd[1], x, c10::nullopt, c10::nullopt, true, true, w32, false);
    dwg = both.narrow(0, 0, F);
    dwu = both.narrow(0, F, F);
  } else if (need_g) {
    dwg = ffn_product(dg, x, c10::nullopt, c10::nullopt, true, true, w32, false);
  } else if (need_u) {
    dwu = ffn_product(du, x, c10::nullopt, c10::nullopt, true, true, w32, false);
  }
  if (need_d) dwd = ffn_product(dy, hd[0], c10::nullopt, c10::nullopt, true, true, d32, false);
  return {dx, dwg, dwu, dwd};
}

}  // namespace osp
