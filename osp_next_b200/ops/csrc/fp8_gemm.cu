// Block-scaled fp8 product for sm_100a:  D[M,N] = act( sum_kb sa[m,kb] sb[n,kb] sum_{k in kb} a[m,k] b[n,k] + bias[n] )
// with e4m3 codes and power-of-two scales in the format of fp8.cuh, both operands K-major.
//
// The scales are applied by the tensor core: tcgen05.mma kind::mxf8f6f4.block_scale multiplies
// each group of 32 along K by a power of two per row of A and per row of B, read from TMEM.
// A block of 128 is four such groups with one scale, so the four MMAs of a block name the same
// byte of the scale words.  Sums stay in the fp32 accumulator in TMEM over the whole of K (over runs
// of 12 blocks where the result is fp32, see kRun), with no rescaling in registers between blocks.
//
// What bounds it: large products run at the power cap, 2500 to 2640 TFLOP/s at an SM clock of 1.33 to
// 1.5 GHz with 136 cycles per 128 x 256 x 32 MMA (128 at the full rate); the same tiles on CTA pairs
// (cta_group::2) were slower (2390).  An MMA of fewer columns costs nearly as much, so 256 columns are
// taken where they fill the GPU: 4096 x 5120 x 5120 takes 84 us, in tiles of 128 columns 119, of 64 194.
//
// Structure (one CTA per SM, 384 threads):
//   warp 0      TMA producer: 128 x 128 codes of A and BN x 128 of B per stage (128B swizzle);
//               with every fourth block, the 512-byte scale chunks of the next four
//   warp 1      one thread issues tcgen05.cp (scale chunk -> TMEM, once per four blocks) and
//               tcgen05.mma 128 x BN x 32, into one of two accumulators
//   warps 4..11 epilogue: two groups of four warps, half of the tile's columns each (where they
//               keep 128 sums a thread, with 208 registers, of which warps 0..3 give up a part)
// A product of few rows runs in another form (skinny_kernel).
// TMEM (512 columns): two accumulators of 256 columns and 16 columns of scales do not fit, so
// at BN = 256 the accumulators overlap by 16 columns: accumulator 0 is 0..255, accumulator 1
// 240..495, scales 496..511.  The epilogue reads the shared columns first and tells the MMA
// warp so; the next tile then starts while the rest is still being read.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/sum.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"
#include "launch.h"
#include "tma_host.h"

namespace osp {

std::vector<at::Tensor> fp8_quantize(const at::Tensor& x, bool tile_scale, bool rows, bool cols, bool sums);

namespace fp8 {

constexpr int kBM = 128;
constexpr int kBK = 128;                      // one scale block, one 128-byte swizzle span
constexpr int kGroupM = 16;
constexpr int kThreads = 384;
constexpr int kStageRow = 80;                 // bytes per staged output row (64 + 16 pad)
constexpr int kStageBytes = 32 * kStageRow;
constexpr uint32_t kScaleCol = 496;           // TMEM columns of the scales: A 496..499, B 500..507

template <int BN> struct Shape {
  static constexpr int kChunksB = BN > 128 ? 2 : 1;             // 128-row scale chunks of a B tile (at
                                                                // BN = 64 a product has one tile of columns)
  static constexpr uint32_t kA = kBM * kBK, kB = BN * kBK;
  static constexpr uint32_t kScales = kChunkBytes * (1 + kChunksB);
  static constexpr int kStages = 196608 / (kA + kB) > 8 ? 8 : 196608 / (kA + kB);
  static constexpr uint32_t kAccStride = BN == 256 ? 240 : BN;  // column offset of accumulator 1
  static constexpr bool kOverlap = BN == 256;
  static constexpr int smem_bytes() {
    return 1024 + kStages * (int)(kA + kB + kScales) + (2 * kStages + 7) * 8 + 16 + 128 + 8 * kStageBytes +
           16 * BN;      // bias: BN / 2 columns for each of 8 warps
  }
};

struct Args {
  int M, N, KB;              // KB: blocks of 128 along K
  const uint8_t* sa;         // packed scales of A, of B
  const uint8_t* sb;
  const float* bias;         // [N] or null
  int act;                   // 0 none, 1 gelu_tanh
  void* out;                 // [M, N] bf16 or f32
  __nv_bfloat16* aux;        // [M, N] pre-activation or null
  int vec;                   // rows of out (and aux) start on 16 bytes
  int* err;
};

__device__ __forceinline__ void bulk_load(uint64_t* bar, void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :: "r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// One 512-byte scale chunk -> 4 TMEM columns, repeated in each quarter of the lanes.
__device__ __forceinline__ void cp_scales(uint32_t tmem, uint32_t saddr) {
  // no swizzle; 8-row core matrices of 16-byte rows, 128 bytes apart
  const uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1u << 46);
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(d) : "memory");
}
__device__ __forceinline__ void umma_mxf8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t tmem_sa, uint32_t tmem_sb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(tmem_sa), "r"(tmem_sb), "r"(accumulate) : "memory");
}
// True in one lane of a converged warp, always the same one.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// e4m3 x e4m3 with power-of-two scales; the scale-byte numbers go into bits 4 (B) and 29 (A).
__host__ __device__ constexpr uint32_t idesc_mxf8(int M, int N) {
  return ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void tile_coords(int t, int num_m, int num_n, int& mb, int& nb) {
  const int per_group = kGroupM * num_n;
  const int g = t / per_group;
  const int first_m = g * kGroupM;
  const int gsize = min(num_m - first_m, kGroupM);
  const int r = t - g * per_group;
  mb = first_m + r % gsize;
  nb = r / gsize;
}

// 0.5 x (1 + tanh(u)) = x / (1 + e^(-2u)), u = sqrt(2/pi) (x + 0.044715 x^3): one exponential and
// one reciprocal by the hardware approximations (a few 2^-23), where tanhf takes some 25 steps;
// at the power limit, where this kernel runs, they cost clock (2290 against 2560 TFLOP/s).
__device__ __forceinline__ float gelu_tanh_f(float x) {
  const float k = -2.f * 0.7978845608028654f * 1.4426950408889634f;       // to a power of two
  return __fdividef(x, 1.f + exp2f(x * (k + k * 0.044715f * x * x)));
}

// Accumulation over a long K.  The tensor core cuts the sum to its fp32 accumulator at each of the
// K / 32 steps, always toward zero (by 3/8 of a last place in the mean: it forms the sum in quarters of
// one): over K = 14040 tokens a weight gradient came out 5e-6 small.  An fp32 result is therefore
// accumulated in runs of kRun blocks, which the epilogue adds up in its registers, rounded to nearest
// (adding the runs up in L2 took the time half again).  Weight gradients of 8960 x 1536 over 14040 tokens
// of very different sizes, 40 of them, against 64 bits: runs of 16 blocks 6.4e-7 in the mean and 1.4e-6 at
// most in 155.6 us, of 12 blocks 4.5e-7 and 7.4e-7 in 158.7, of 8 blocks 3.1e-7 and 6.9e-7 in 163.8; an
// fp32 product of the same operands 5.5e-7 and 7.9e-7.  A second run costs most where it is short
// (20000 x 8192 over 1664: 266 us in one, 281 in two; over 2048: 307 and 317).
// bf16 results have one run: the cut (7e-6 over K = 20160) moves one in some 800 of them by a last
// place, and runs would cost 3.5 % (13824 x 5120 over 20160 tokens: 1033 us, in runs 1068).
constexpr int kRun = 12;
static_assert(kRun % 4 == 0, "a run begins with a chunk of four blocks' scales");

__device__ __forceinline__ void store_scalar(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_scalar(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

// A warp's 32 rows x 32 columns of results (one row per lane) -> out, through shared memory so
// that 64 bytes of a row are written as one segment (16 bytes by 32 lanes to 32 rows took twice
// the time of the whole product at K = 1536 in fp32).
template <typename OutT>
__device__ __forceinline__ void store_chunk(OutT* out, const float* v, uint8_t* stg, int lane, long row0, int col0,
                                            int M, int N, bool vec) {
  const bool whole = vec && col0 + 32 <= N;           // 16-byte stores fit
  if constexpr (sizeof(OutT) == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 w;
      w.x = pack_bf16x2(v[8 * j + 0], v[8 * j + 1]);
      w.y = pack_bf16x2(v[8 * j + 2], v[8 * j + 3]);
      w.z = pack_bf16x2(v[8 * j + 4], v[8 * j + 5]);
      w.w = pack_bf16x2(v[8 * j + 6], v[8 * j + 7]);
      *reinterpret_cast<uint4*>(stg + lane * kStageRow + j * 16) = w;
    }
    __syncwarp();
    if (whole) {
      const int q = lane >> 2, cc = lane & 3;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rr = i * 8 + q;
        if (row0 + rr < M)
          *reinterpret_cast<uint4*>(out + (row0 + rr) * N + col0 + cc * 8) =
              *reinterpret_cast<const uint4*>(stg + rr * kStageRow + cc * 16);
      }
    } else if (col0 + lane < N) {                       // any row length: a row's 32 elements by 32 lanes
#pragma unroll 8
      for (int rr = 0; rr < 32; ++rr)
        if (row0 + rr < M) out[(row0 + rr) * N + col0 + lane] = reinterpret_cast<const OutT*>(stg + rr * kStageRow)[lane];
    }
    __syncwarp();
  } else {
    const int q = lane >> 2, cc = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {                     // 16 columns at a time: 64 bytes of a row
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(stg + lane * kStageRow + j * 16) =
            make_float4(v[16 * h + 4 * j], v[16 * h + 4 * j + 1], v[16 * h + 4 * j + 2], v[16 * h + 4 * j + 3]);
      __syncwarp();
      if (whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rr = i * 8 + q;
          if (row0 + rr < M)
            *reinterpret_cast<float4*>(out + (row0 + rr) * N + col0 + 16 * h + cc * 4) =
                *reinterpret_cast<const float4*>(stg + rr * kStageRow + cc * 16);
        }
      } else if (col0 + 16 * h + (lane & 15) < N) {
#pragma unroll 8
        for (int rr = lane >> 4; rr < 32; rr += 2)
          if (row0 + rr < M)
            out[(row0 + rr) * N + col0 + 16 * h + (lane & 15)] =
                reinterpret_cast<const OutT*>(stg + rr * kStageRow)[lane & 15];
      }
      __syncwarp();
    }
  }
}

// Bias (the chunk's 32, in shared memory), activation and store of a warp's 32 x 32 chunk.
template <typename OutT>
__device__ __forceinline__ void finish_chunk(const Args& args, float* v, const float* bias, uint8_t* stg, int lane,
                                             long row0, int col0) {
  if (args.bias) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 b = reinterpret_cast<const float4*>(bias)[j];
      v[4 * j] += b.x; v[4 * j + 1] += b.y; v[4 * j + 2] += b.z; v[4 * j + 3] += b.w;
    }
  }
  if (args.aux) store_chunk(args.aux, v, stg, lane, row0, col0, args.M, args.N, args.vec);
  if (args.act == 1) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = gelu_tanh_f(v[j]);
  }
  store_chunk(reinterpret_cast<OutT*>(args.out), v, stg, lane, row0, col0, args.M, args.N, args.vec);
}

// Launched with 12 warps x 168 registers; 4 x 64 + 8 x 208 of them are what is used.
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 64;"); }
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 208;"); }

template <int BN, typename OutT, bool RUNS>
__global__ void __launch_bounds__(kThreads, 1)
gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Args args) {
  using S = Shape<BN>;
  constexpr int STAGES = S::kStages;
  constexpr uint32_t IDESC = idesc_mxf8(kBM, BN);
  constexpr bool kSplitRegs = RUNS && BN == 256;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * S::kA;
  uint8_t* sS = sB + STAGES * S::kB;
  uint64_t* full = reinterpret_cast<uint64_t*>(sS + STAGES * S::kScales);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;      // [2] accumulator finished
  uint64_t* tempty = tfull + 2;          // [2] accumulator read
  uint64_t* tearly = tempty + 2;         // [2] its columns shared with the other one read
  uint64_t* done = tearly + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* epi_stage = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(abort_flag + 1) + 127) & ~uintptr_t(127));

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int num_m = (args.M + kBM - 1) / kBM;
  const int num_n = (args.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n;
  const int num_kb = args.KB;
  const int kgroups = (num_kb + 3) >> 2;
  const int runs = RUNS ? (num_kb + kRun - 1) / kRun : 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tfull[a], 1); mbar_init(&tempty[a], 8); mbar_init(&tearly[a], 4); }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_dependency_wait();
  allow_dependents();

  if (warp < 4) {
    if constexpr (kSplitRegs) fewer_registers();         // by all warps of the warpgroup
    if (warp == 0) {
      // ---------------------------------------------------------------- producer
      if (lane == 0) {
        const int last_chunk = (args.N + 127) / 128 - 1;
        int stage = 0;
        uint32_t phase = 0;
        for (int t = blockIdx.x; t < num_tiles && !*abort_flag; t += gridDim.x) {
          int mb, nb;
          tile_coords(t, num_m, num_n, mb, nb);
          for (int kb = 0; kb < num_kb; ++kb) {
            if (!mbar_wait(&empty[stage], phase ^ 1, args.err, kErrFp8Producer)) { *abort_flag = 1; break; }
            const bool with_scales = (kb & 3) == 0;
            mbar_expect_tx(&full[stage], S::kA + S::kB + (with_scales ? S::kScales : 0));
            tma_load_2d(&tmA, &full[stage], sA + stage * S::kA, kb * kBK, mb * kBM);
            tma_load_2d(&tmB, &full[stage], sB + stage * S::kB, kb * kBK, nb * BN);
            if (with_scales) {
              uint8_t* d = sS + stage * S::kScales;
              bulk_load(&full[stage], d, args.sa + ((long)mb * kgroups + (kb >> 2)) * kChunkBytes, kChunkBytes);
#pragma unroll
              for (int c = 0; c < S::kChunksB; ++c) {
                // a tile's second chunk may lie past the end of N: its rows are zeros, any scale will do
                const int chunk = min(nb * BN / 128 + c, last_chunk);
                bulk_load(&full[stage], d + (1 + c) * kChunkBytes,
                          args.sb + ((long)chunk * kgroups + (kb >> 2)) * kChunkBytes, kChunkBytes);
              }
            }
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
          }
        }
        // the last loads have landed before the block ends, whoever gave up waiting for them: stages
        // before `stage` were filled in this round, the others in the one before (or never)
        for (int s = 0; s < STAGES; ++s) mbar_wait(&full[s], s < stage ? phase : phase ^ 1, args.err, kErrFp8Teardown);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA issuer
      // The whole warp runs the loop and one elected lane issues: the operands of the MMAs then stay
      // in uniform registers, and the descriptors of a stage differ from the first's by an addend.
      const uint64_t a_desc = sdesc_sw128(smem_u32(sA), 16, 1024), b_desc = sdesc_sw128(smem_u32(sB), 16, 1024);
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      const uint32_t t_sa = tmem_base + kScaleCol, t_sb = t_sa + 4;
      // (tile, run) pairs in order; `it` counts them
      for (int t = blockIdx.x, run = 0; t < num_tiles && !*abort_flag; ++it) {
        const int kb0 = run * kRun, kb1 = runs == 1 ? num_kb : min(num_kb, kb0 + kRun);
        const int acc = it & 1;
        const uint32_t acc_phase = (it >> 1) & 1;
        bool ok = mbar_wait(&tempty[acc], acc_phase ^ 1, args.err, kErrFp8Mma);
        // the previous tile's accumulator (use (it - 1) / 2 of it) shares columns with this one
        if (ok && S::kOverlap && it > 0) ok = mbar_wait(&tearly[acc ^ 1], ((it - 1) >> 1) & 1, args.err, kErrFp8Mma);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) { *abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * S::kAccStride;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, args.err, kErrFp8Mma));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            if ((kb & 3) == 0) {
              // cp and mma of one thread execute in order: the scales are in place for the
              // MMAs below, and the MMAs before them have read the old ones
              const uint32_t s_addr = smem_u32(sS + stage * S::kScales);
              cp_scales(t_sa, s_addr);
#pragma unroll
              for (int c = 0; c < S::kChunksB; ++c) cp_scales(t_sa + 4 + 4 * c, s_addr + (1 + c) * kChunkBytes);
            }
            const uint64_t ad = a_desc + stage * (S::kA >> 4), bd = b_desc + stage * (S::kB >> 4);
            const uint32_t idesc = IDESC | ((uint32_t)(kb & 3) << 4) | ((uint32_t)(kb & 3) << 29);
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k)
              umma_mxf8(d_tmem, ad + 2 * k, bd + 2 * k, idesc, t_sa, t_sb, (kb > kb0 || k > 0) ? 1u : 0u);
            umma_commit(&empty[stage]);
            if (kb + 1 == kb1) umma_commit(&tfull[acc]);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) { *abort_flag = 1; break; }
        if (++run == runs) { run = 0; t += gridDim.x; }
      }
      if (elect_one()) umma_commit(done);
      mbar_wait(done, 0, args.err, kErrFp8Teardown);
    }
  } else {
    // ---------------------------------------------------------------- epilogue (warps 4..11)
    if constexpr (kSplitRegs) more_registers();
    constexpr int PER = BN / 64;                // 32-column chunks of each of the two groups
    const int quarter = warp & 3;               // TMEM lanes 32 * quarter ..
    const int eg = (warp - 4) >> 2;
    uint8_t* stg = epi_stage + (warp - 4) * kStageBytes;
    float* sbias = reinterpret_cast<float*>(epi_stage + 8 * kStageBytes) + (warp - 4) * PER * 32;
    float sum[RUNS ? PER : 1][32];                        // the runs so far
    int it = 0;
    for (int t = blockIdx.x, run = 0; t < num_tiles; ++it) {
      if (*abort_flag) break;
      int mb, nb;
      tile_coords(t, num_m, num_n, mb, nb);
      const int acc = it & 1;
      // the bias of the warp's columns, fetched while the MMAs run: beside the operands' traffic a
      // load takes thousands of cycles, which per chunk made the epilogue longer than the MMAs
      if (args.bias && run == 0) {
        __syncwarp();
#pragma unroll
        for (int c = 0; c < PER; ++c) {
          const int col = nb * BN + (eg * PER + c) * 32 + lane;
          sbias[c * 32 + lane] = col < args.N ? args.bias[col] : 0.f;
        }
        __syncwarp();
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], (it >> 1) & 1, args.err, kErrFp8Epilogue))) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const long row0 = (long)mb * kBM + quarter * 32;
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * S::kAccStride;
      // The columns that the accumulators share (the last of 0, the first of 1) are read first, and
      // the next tile's MMAs may start; the rest frees the accumulator.
      auto shared_read = [&](int i) {
        if (S::kOverlap && i == 0 && eg == (acc ^ 1)) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tearly[acc]);
        }
      };
      auto all_read = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[acc]);
      };
      if constexpr (RUNS) {
        auto add_up = [&](auto backwards) {
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            constexpr bool kBack = decltype(backwards)::value;
            const int c = kBack ? PER - 1 - i : i;
            uint32_t r[32];
            tmem_ld32(t_row + (eg * PER + c) * 32, r);
            tmem_ld_wait();
            shared_read(i);
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[c][j] = run == 0 ? __uint_as_float(r[j]) : sum[c][j] + __uint_as_float(r[j]);
          }
        };
        if (S::kOverlap && acc == 0) add_up(std::true_type());
        else add_up(std::false_type());
        all_read();
        if (run + 1 == runs) {
#pragma unroll
          for (int c = 0; c < PER; ++c) {
            const int col0 = nb * BN + (eg * PER + c) * 32;
            if (col0 < args.N) finish_chunk<OutT>(args, sum[c], sbias + c * 32, stg, lane, row0, col0);
          }
        }
      } else {
        auto chunk = [&](int i) { return (S::kOverlap && acc == 0) ? PER - 1 - i : i; };
        float r[2][32];
        tmem_ld32(t_row + (eg * PER + chunk(0)) * 32, reinterpret_cast<uint32_t*>(r[0]));
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          tmem_ld_wait();
          shared_read(i);
          if (i + 1 < PER)                                // on its way while this one is stored
            tmem_ld32(t_row + (eg * PER + chunk(i + 1)) * 32, reinterpret_cast<uint32_t*>(r[(i + 1) & 1]));
          else
            all_read();
          const int col0 = nb * BN + (eg * PER + chunk(i)) * 32;
          if (col0 < args.N) finish_chunk<OutT>(args, r[i & 1], sbias + chunk(i) * 32, stg, lane, row0, col0);
        }
      }
      if (++run == runs) { run = 0; t += gridDim.x; }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------- few rows
// Up to 64 rows of A: the time is that of reading B, the weight.  The roles are exchanged, D^T =
// B A^T, so that 128 rows of the weight fill the tensor core's M and the BNX (16 to 64) rows of A its
// N.  CTAs of 100 KB share an SM in pairs; where the tiles are too few to fill the GPU a cluster
// of up to 8 CTAs splits K and adds its parts through distributed shared memory, in rank order
// (the result does not depend on timing, and no workspace is needed).  The weight's first
// stages are loaded before the wait for the quantiser of A.  1 x 5120 -> 30720: 28.4 us with the
// quantiser, 0.85 of the copy rate on the weight's bytes; 128 rows take 27.5 us here (cold caches)
// and 21.5 in gemm_kernel's tiles, 64 rows about the same in both.
// 192 threads: warp 0 TMA producer, warp 1 MMA issuer, warps 2..5 epilogue.
template <int BNX> struct Skinny {
  static constexpr uint32_t kW = 128 * kBK, kX = BNX * kBK, kScales = 2 * kChunkBytes;
  static constexpr int kStages = 101 * 1024 / (kW + kX + kScales);
  static constexpr uint32_t kScaleCol = 2 * BNX;         // behind two accumulators
  static constexpr uint32_t kTmemCols = 2 * BNX + 8 <= 64 ? 64 : 2 * BNX + 8 <= 128 ? 128 : 256;
  static constexpr int smem_bytes() { return 1024 + kStages * (int)(kW + kX + kScales) + (2 * kStages + 4) * 8 + 16; }
  static constexpr int kPartRow = BNX + 4;               // floats of a weight row's part, padded
  static_assert(kStages * (int)(kW + kX) >= kPartRow * 128 * 4, "the parts of a split fit the ring");
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Every warp of the cluster's CTAs arrives converged (the barrier is of the aligned form, and the
// code before it may have left a warp's lanes apart).
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Four floats at `p` in this CTA's shared memory, read from CTA `rank` of the cluster.
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

template <int BNX, typename OutT>
__global__ void __launch_bounds__(192, 2)
skinny_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const Args args,
              int splits, bool weight_first) {
  using S = Skinny<BNX>;
  constexpr int STAGES = S::kStages;
  constexpr uint32_t IDESC = idesc_mxf8(128, BNX);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sW = smem;
  uint8_t* sX = sW + STAGES * S::kW;
  uint8_t* sS = sX + STAGES * S::kX;
  uint64_t* full = reinterpret_cast<uint64_t*>(sS + STAGES * S::kScales);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;                      // [2]
  uint64_t* tempty = tfull + 2;                          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  float* part = reinterpret_cast<float*>(smem);          // [128][kPartRow], over the ring when it is done with

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int split = splits > 1 ? (int)cluster_rank() : 0;
  const int tile = blockIdx.x / splits;
  const int kgroups = (args.KB + 3) >> 2;
  const int kb0 = 4 * (int)((long)kgroups * split / splits);
  const int kb1 = min(args.KB, 4 * (int)((long)kgroups * (split + 1) / splits));
  // an fp32 result is summed over runs of blocks in the epilogue's registers (see kRun)
  const int run_len = sizeof(OutT) == 4 ? kRun : kb1 - kb0;
  const int runs = (kb1 - kb0 + run_len - 1) / run_len;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tfull[a], 1); mbar_init(&tempty[a], 4); }
    fence_mbar_init();
    prefetch_tmap(&tmX);
    prefetch_tmap(&tmW);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // only the producer of the weight's first stages goes ahead, if nothing before can have written it
  if (warp != 0 || !weight_first) {
    grid_dependency_wait();
    allow_dependents();
  }

  if (warp == 0) {
    if (lane == 0) {
      auto load_w = [&](int kb, int stage) {
        const bool first = (kb & 3) == 0;
        mbar_expect_tx(&full[stage], S::kW + S::kX + (first ? S::kScales : 0));
        tma_load_2d(&tmW, &full[stage], sW + stage * S::kW, kb * kBK, tile * 128);
        if (first)
          bulk_load(&full[stage], sS + stage * S::kScales, args.sb + ((long)tile * kgroups + (kb >> 2)) * kChunkBytes,
                    kChunkBytes);
      };
      auto load_x = [&](int kb, int stage) {
        tma_load_2d(&tmX, &full[stage], sX + stage * S::kX, kb * kBK, 0);
        if ((kb & 3) == 0)
          bulk_load(&full[stage], sS + stage * S::kScales + kChunkBytes, args.sa + (long)(kb >> 2) * kChunkBytes,
                    kChunkBytes);
      };
      const int ahead = min(STAGES, kb1 - kb0);
      for (int i = 0; i < ahead; ++i) load_w(kb0 + i, i);
      grid_dependency_wait();
      for (int i = 0; i < ahead; ++i) load_x(kb0 + i, i);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0 + ahead; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase, args.err, kErrFp8Producer)) break;
        load_w(kb, stage);
        load_x(kb, stage);
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      // the last loads have landed before the ring is reused and the block ends
      for (int s = 0; s < ahead; ++s) mbar_wait(&full[s], s < stage ? phase ^ 1 : phase, args.err, kErrFp8Teardown);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t t_sa = tmem_base + S::kScaleCol, t_sb = t_sa + 4;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int run = 0; run < runs && ok; ++run) {
        const int first = kb0 + run * run_len, last = min(kb1, first + run_len);
        const int acc = run & 1;
        if (!(ok = mbar_wait(&tempty[acc], ((run >> 1) & 1) ^ 1, args.err, kErrFp8Mma))) break;
        tc_fence_after();
        for (int kb = first; kb < last; ++kb) {
          if (!(ok = mbar_wait(&full[stage], phase, args.err, kErrFp8Mma))) break;
          tc_fence_after();
          if ((kb & 3) == 0) {
            const uint32_t s_addr = smem_u32(sS + stage * S::kScales);
            cp_scales(t_sa, s_addr);
            cp_scales(t_sb, s_addr + kChunkBytes);
          }
          const uint32_t w_addr = smem_u32(sW + stage * S::kW), x_addr = smem_u32(sX + stage * S::kX);
          const uint32_t idesc = IDESC | ((uint32_t)(kb & 3) << 4) | ((uint32_t)(kb & 3) << 29);
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k)
            umma_mxf8(tmem_base + acc * BNX, sdesc_sw128(w_addr + k * 32, 16, 1024),
                      sdesc_sw128(x_addr + k * 32, 16, 1024), idesc, t_sa, t_sb, (kb > first || k > 0) ? 1u : 0u);
          umma_commit(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        umma_commit(&tfull[acc]);
      }
    }
    __syncwarp();
  }

  const int quarter = warp & 3;
  const int local = quarter * 32 + lane;                 // row of the weight tile
  const int n = tile * 128 + local;
  const float bias = (warp >= 2 && args.bias && n < args.N) ? args.bias[n] : 0.f;
  auto put = [&](int m, float v) {
    v += bias;
    const long o = (long)m * args.N + n;
    if (args.aux) args.aux[o] = __float2bfloat16(v);
    store_scalar(reinterpret_cast<OutT*>(args.out) + o, args.act ? gelu_tanh_f(v) : v);
  };
  if (warp >= 2) {
    const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16);
    float v[BNX];
#pragma unroll
    for (int j = 0; j < BNX; ++j) v[j] = 0.f;
    for (int run = 0; run < runs; ++run) {
      const int acc = run & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], (run >> 1) & 1, args.err, kErrFp8Epilogue))) break;
      tc_fence_after();
#pragma unroll
      for (int m0 = 0; m0 < BNX; m0 += 16) {
        if (m0 < args.M) {
          uint32_t r[16];
          tmem_ld16(t_row + acc * BNX + m0, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) v[m0 + j] += __uint_as_float(r[j]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
    }
#pragma unroll
    for (int m0 = 0; m0 < BNX; m0 += 4) {
      if (m0 < args.M) {
        if (splits > 1) {
          *reinterpret_cast<float4*>(part + local * S::kPartRow + m0) =
              make_float4(v[m0], v[m0 + 1], v[m0 + 2], v[m0 + 3]);
        } else if (n < args.N) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (m0 + j < args.M) put(m0 + j, v[m0 + j]);
        }
      }
    }
  }
  if (splits > 1) {
    cluster_sync();
    if (warp >= 2 && n < args.N) {
      // rows of A dealt to the CTAs four at a time; all parts of four rows in flight together
      for (int m = 4 * split; m < args.M; m += 4 * splits) {
        float4 t[8];
#pragma unroll
        for (int s = 0; s < 8; ++s)
          if (s < splits) t[s] = load_from_cta(part + local * S::kPartRow + m, s);
        float4 v = t[0];
#pragma unroll
        for (int s = 1; s < 8; ++s)
          if (s < splits) { v.x += t[s].x; v.y += t[s].y; v.z += t[s].z; v.w += t[s].w; }
        put(m, v.x);
        if (m + 1 < args.M) put(m + 1, v.y);
        if (m + 2 < args.M) put(m + 2, v.z);
        if (m + 3 < args.M) put(m + 3, v.w);
      }
    }
    cluster_sync();                                      // no CTA leaves while its part may be read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// 2-D map over e4m3 codes [rows, Kp]: boxes of 128 bytes x box_rows, 128B swizzle, zeros outside.
static CUtensorMap make_tmap(const at::Tensor& t, uint32_t box_rows) {
  CUtensorMap m;
  const cuuint64_t dims[2] = {(cuuint64_t)t.size(1), (cuuint64_t)t.size(0)};
  const cuuint64_t strides[1] = {(cuuint64_t)t.size(1)};
  const cuuint32_t box[2] = {(cuuint32_t)kBK, box_rows}, estr[2] = {1, 1};
  const CUresult r = encode_tiled_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, t.data_ptr(), dims, strides, box, estr,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed: ", std::to_string((int)r));
  return m;
}

template <int BN, typename OutT, bool RUNS>
static void launch(const at::Tensor& a, const at::Tensor& b, const Args& args, cudaStream_t stream) {
  constexpr int smem = Shape<BN>::smem_bytes();
  static_assert(smem <= 232448, "shared memory");
  const int tiles = ((args.M + kBM - 1) / kBM) * ((args.N + BN - 1) / BN);
  launch_kernel(gemm_kernel<BN, OutT, RUNS>, std::min(tiles, num_sms(a.get_device())), kThreads, smem, 1, stream,
                make_tmap(a, kBM), make_tmap(b, BN), args);
}

template <int BNX, typename OutT>
static void launch_skinny(const at::Tensor& a, const at::Tensor& b, const Args& args, bool weight_first,
                          cudaStream_t stream) {
  // as many parts of K as fill two CTAs per SM, at most 8 (a portable cluster), whole scale
  // chunks each; then no more parts than the longest of them needs
  const int tiles = (args.N + 127) / 128, kgroups = (args.KB + 3) / 4;
  const int most = std::max(1, std::min({8, kgroups, 2 * num_sms(a.get_device()) / tiles}));
  const int longest = (kgroups + most - 1) / most;
  const int splits = (kgroups + longest - 1) / longest;
  launch_kernel(skinny_kernel<BNX, OutT>, tiles * splits, 192, Skinny<BNX>::smem_bytes(), splits, stream,
                make_tmap(a, BNX), make_tmap(b, 128), args, splits, weight_first);
}

// `behind`: the stream's last kernel is the quantiser of `a`, whose own predecessors have completed
// when a kernel starts behind it: the weight, which it does not write, may be read at once.
template <typename OutT>
static void product(const at::Tensor& a, const at::Tensor& b, const Args& args, bool behind, cudaStream_t stream) {
  if (args.M <= 16) return launch_skinny<16, OutT>(a, b, args, behind, stream);
  if (args.M <= 32) return launch_skinny<32, OutT>(a, b, args, behind, stream);
  if (args.M <= 64) return launch_skinny<64, OutT>(a, b, args, behind, stream);
  // an MMA of 128 columns takes nearly the time of one of 256: narrow tiles only where one round of
  // them covers the result (128 x 4096 -> 5120: 17.6 us in tiles of 128 columns, 20.3 of 256; 512 rows,
  // two rounds against one: 28.2 and 22.5)
  const long tiles128 = (long)((args.M + 127) / 128) * ((args.N + 127) / 128);
  const bool narrow = args.N <= 128 || tiles128 <= num_sms(a.get_device());
  if constexpr (sizeof(OutT) == 4) {
    if (args.KB > kRun) {
      if (args.N <= 64) launch<64, OutT, true>(a, b, args, stream);
      else if (narrow) launch<128, OutT, true>(a, b, args, stream);
      else launch<256, OutT, true>(a, b, args, stream);
      return;
    }
  }
  if (args.N <= 64) launch<64, OutT, false>(a, b, args, stream);
  else if (narrow) launch<128, OutT, false>(a, b, args, stream);
  else launch<256, OutT, false>(a, b, args, stream);
}

}  // namespace fp8

static void check_operand(const char* name, const at::Tensor& t, const at::Tensor& s, int64_t kp, int dev) {
  TORCH_CHECK(t.is_cuda() && s.is_cuda() && t.get_device() == dev && s.get_device() == dev, "fp8_matmul: ", name,
              " on the device of a");
  TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn && t.dim() == 2 && t.is_contiguous() && t.size(1) == kp &&
              kp % 128 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              "fp8_matmul: ", name, " e4m3 codes [rows, ", std::to_string(kp), "], contiguous, 16-byte aligned, K a multiple of 128");
  TORCH_CHECK(s.scalar_type() == at::kByte && s.is_contiguous() &&
              s.numel() == (t.size(0) + 127) / 128 * ((kp + 511) / 512) * 512 &&
              reinterpret_cast<uintptr_t>(s.data_ptr()) % 16 == 0, "fp8_matmul: packed scales of ", name);
}

// {act(A B^T + bias) [M, N], its pre-activation in bf16 if asked for}; a [M, Kp], b [N, Kp] e4m3 with
// packed scales sa, sb
static std::vector<at::Tensor> multiply(const at::Tensor& a, const at::Tensor& sa, const at::Tensor& b,
                                        const at::Tensor& sb, const c10::optional<at::Tensor>& bias_, int64_t act,
                                        bool f32, bool aux, bool behind) {
  TORCH_CHECK(a.is_cuda() && a.dim() == 2, "fp8_matmul: a on the GPU");
  const int dev = a.get_device();
  const int64_t kp = a.size(1);
  check_operand("a", a, sa, kp, dev);
  check_operand("b", b, sb, kp, dev);
  TORCH_CHECK(a.size(0) < (int64_t(1) << 31) - 256 && b.size(0) < (int64_t(1) << 31) - 256, "fp8_matmul: sizes below 2^31");
  TORCH_CHECK(act == 0 || act == 1, "fp8_matmul: act");
  c10::cuda::CUDAGuard guard(a.device());
  fp8::Args args{};
  args.M = (int)a.size(0);
  args.N = (int)b.size(0);
  args.KB = (int)(kp / 128);
  args.sa = sa.data_ptr<uint8_t>();
  args.sb = sb.data_ptr<uint8_t>();
  at::Tensor bias;
  if (bias_.has_value()) {
    TORCH_CHECK(bias_->is_cuda() && bias_->get_device() == dev && bias_->dim() == 1 && bias_->numel() == args.N,
                "fp8_matmul: bias [N] on the device of a");
    bias = bias_->to(at::kFloat).contiguous();
    args.bias = bias.data_ptr<float>();
  }
  std::vector<at::Tensor> out;
  out.push_back(at::empty({args.M, args.N}, a.options().dtype(f32 ? at::kFloat : at::kBFloat16)));
  args.act = (int)act;
  args.out = out[0].data_ptr();
  args.vec = args.N % 8 == 0;
  if (aux) {
    out.push_back(at::empty({args.M, args.N}, a.options().dtype(at::kBFloat16)));
    args.aux = reinterpret_cast<__nv_bfloat16*>(out[1].data_ptr());
  }
  args.err = error_word(dev);
  if (args.M == 0 || args.N == 0) return out;
  TORCH_CHECK(args.KB > 0, "fp8_matmul: K of at least 1");
  auto stream = c10::cuda::getCurrentCUDAStream();
  if (f32) fp8::product<float>(a, b, args, behind, stream);
  else fp8::product<__nv_bfloat16>(a, b, args, behind, stream);
  return out;
}

std::vector<at::Tensor> fp8_gemm(const at::Tensor& a, const at::Tensor& sa, const at::Tensor& b, const at::Tensor& sb,
                                 const c10::optional<at::Tensor>& bias, int64_t act, bool f32, bool aux) {
  return multiply(a, sa, b, sb, bias, act, f32, aux, false);
}

// The same of x [..., K] in bf16, fp16 or fp32, quantised here.
std::vector<at::Tensor> fp8_linear(const at::Tensor& x, const at::Tensor& b, const at::Tensor& sb,
                                   const c10::optional<at::Tensor>& bias, int64_t act, bool f32, bool aux) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1 && x.size(-1) > 0, "fp8_matmul: a [..., K] on the GPU");
  const at::Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  const auto q = fp8_quantize(x2, false, true, false, false);
  return multiply(q[0], q[1], b, sb, bias, act, f32, aux, x2.numel() > 0);
}

// A training step of a linear in two calls (the same steps as the functions above, without a
// Python call for each): x [M, K], w [N, K], none of the sizes zero.
// -> {y, pre-activation if asked for, x^T as blocks of tokens (need_w), w^T (need_x)}, codes and scales
std::vector<at::Tensor> fp8_linear_forward(const at::Tensor& x, const at::Tensor& w,
                                           const c10::optional<at::Tensor>& bias, int64_t act, bool aux, bool need_x,
                                           bool need_w) {
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1) && x.numel() > 0 && w.numel() > 0,
              "fp8_linear: x [M, K], w [N, K], not empty");
  const auto wq = fp8_quantize(w, true, true, need_x, false);
  const auto xq = fp8_quantize(x, false, true, need_w, false);
  const auto y = multiply(xq[0], xq[1], wq[0], wq[1], bias, act, false, aux, true);
  return {y[0], aux ? y[1] : at::Tensor(), xq[2], xq[3], wq[2], wq[3]};
}

// -> {dx [M, K], dw [N, K], db [N]} of g [M, N], those that are needed
std::vector<at::Tensor> fp8_linear_backward(const at::Tensor& g, const c10::optional<at::Tensor>& xc,
                                            const c10::optional<at::Tensor>& xs, const c10::optional<at::Tensor>& wc,
                                            const c10::optional<at::Tensor>& ws, bool need_b, bool dx_f32, bool dw_f32) {
  const bool need_x = wc.has_value(), need_w = xc.has_value();
  TORCH_CHECK(need_x || need_w, "fp8_linear: gradients of x or w");
  const bool sums = need_b && need_x && need_w;
  const auto q = fp8_quantize(g, false, need_x, need_w, sums);
  std::vector<at::Tensor> out(3);
  if (need_x) out[0] = multiply(q[0], q[1], *wc, *ws, c10::nullopt, 0, dx_f32, false, true)[0];
  if (need_w) out[1] = multiply(q[2], q[3], *xc, *xs, c10::nullopt, 0, dw_f32, false, !need_x)[0];
  if (sums) out[2] = q[4].sum(0);
  return out;
}

}  // namespace osp
