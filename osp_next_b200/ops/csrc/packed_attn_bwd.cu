// Gradients of packed attention (packed_attn_fwd.cu): grouped heads, causal or not.
//
//   delta = rowsum(dO o O),  P = 2^(S scale log2e - lse log2e),  dS = P o (dO V^T - delta)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO   (dK, dV summed over the heads of a group)
//
// Two kernels, P recomputed in both (7 products instead of 5), no atomics, so results do not depend
// on the order in which CTAs run:
//   dkdv  a CTA per tile of 128 keys and key head, keys on the lanes of tensor memory; it passes over
//         the row tiles (packed_attn.cuh: positions x group heads) from the first query that sees
//         its first key on, and dV += P^T dO, dK += dS^T Q sum the group's heads by themselves
//   dq    a CTA per row tile and key head, over the key tiles up to its last query's limit
// Both run the order of products and waits of attention_bwd.cu: elementwise work of one step under
// the products of the next.  Columns of dkdv rise with the query's position, so the causal mask is a
// first column per key; in dq it is a limit per row.  Items of dkdv with far more than their share of
// the work (the first keys of a long causal sequence) are split along the queries; their fp32 parts
// are added in a fixed order by packed_join_kernel.
//
// What bounds it: products and elementwise work in turn; 16 heads of 128 over 8192 tokens, all pairs: dK, dV
// 860 us and dQ 673 (1.28 and 1.23 PFLOP/s of products); 12 causal samples of 5 to 4096 tokens, 16 heads to 4:
// 186 and 161 us, tensor pipe 50 % and 43 % active.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "packed_attn.cuh"
#include "packed_attn_host.h"

namespace osp {

namespace {
constexpr int kT = pa::kRows;
constexpr int kBwdThreads = 384;
}  // namespace

struct PackedBwdArgs {
  const int* items;
  int G, P, Hq, Hkv, Dr;
  int units, at_once;      // items x key heads, heads run together (pa::unit_of)
  int causal;
  const float* lse;        // [Nq, Hq] natural log
  const float* delta;      // [Nq, Hq]
  __nv_bfloat16* dq;       // [Nq, Hq, Dr]
  __nv_bfloat16* dk;       // [Nk, Hkv, Dr]
  __nv_bfloat16* dv;
  float* part;             // [slots, Hkv, 2 (dV, dK), 128, Dr]
  float scale;
  int* err;
};

// delta of each (token, head) row: 16 lanes x 8 elements, two rows per warp.
__global__ void packed_delta_kernel(const __nv_bfloat16* __restrict__ o, const uint8_t* __restrict__ low,
                                    const __nv_bfloat16* __restrict__ dout, float* __restrict__ delta, long rows,
                                    int Dr) {
  const long row = ((long)blockIdx.x * blockDim.x + threadIdx.x) / 16;
  const int c = (threadIdx.x % 16) * 8;
  float acc = 0.f;
  if (row < rows && c < Dr) {
    const uint4 a = *reinterpret_cast<const uint4*>(o + row * Dr + c);
    const uint4 g = *reinterpret_cast<const uint4*>(dout + row * Dr + c);
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, gw[4] = {g.x, g.y, g.z, g.w};
    const uint2 l = low ? *reinterpret_cast<const uint2*>(low + row * Dr + c) : make_uint2(0u, 0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&aw[i]));
      const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&gw[i]));
      const uint32_t lw = (i < 2 ? l.x : l.y) >> (16 * (i & 1));
      acc = fmaf(x.x + pa::low_value(lw & 0xffu), y.x, acc);
      acc = fmaf(x.y + pa::low_value(lw >> 8 & 0xffu), y.y, acc);
    }
  }
#pragma unroll
  for (int s = 8; s > 0; s >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, s);
  if (row < rows && c == 0) delta[row] = acc;
}

// Operands in tensor memory: two warps share a lane quarter, each owns 64 fp32 columns and packs its
// values as 32 columns of bf16 pairs at the start of its own range, so K step k (16 rows, 8 pair
// columns) starts at column 8 k, plus 32 for the second half.
__device__ __forceinline__ uint32_t pair_col(int k) { return 8u * k + (k >= 4 ? 32u : 0u); }

__device__ __forceinline__ void store_pairs(uint32_t taddr, const float* v) {
  tmem_st4(taddr, pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// What rounding those values to bf16 left, rounded in turn (kTwo).  Packs of sequences of up to 32 rows multiply dS
// as two bf16 numbers: their dQ and dK are then off by little more than the rounding of the result, 1.8e-3 to 1.9e-3
// from 64 bits.  With one number it is 2.5e-3, up to 2.9e-3 in a batch of few rows; longer sequences, where the
// second product would take its time, stay at 2.4e-3 (400 samples of 16 tokens, 16 heads of 64 to 4: dK, dV 77 and
// with two 84 us, dQ 55 and 59; with the choice made inside the kernels dK, dV over 4096 tokens took 159 for 154).
__device__ __forceinline__ void store_rest(uint32_t taddr, const float* v) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i] - bf16_round(v[i]);
  store_pairs(taddr, r);
}

// ---------------------------------------------------------------------------- dK, dV
template <int D>
struct KeySmem {
  static constexpr int BOX = kT * 128, DB = D / 64, TILE = DB * BOX;
  static constexpr int OFF_V = TILE;
  static constexpr int OFF_STAGE = 2 * TILE;              // 2 stages of (Q, dO)
  static constexpr int STAGE = 2 * TILE;
  static constexpr int OFF_VEC = OFF_STAGE + 2 * STAGE;   // 2 stages x (lse log2e, delta)[128]
  static constexpr int OFF_BAR = OFF_VEC + 2 * 2 * kT * 4;
  static constexpr int BYTES = OFF_BAR + 256 + 1024;
};

template <int D, bool kTwo>
__global__ void __launch_bounds__(kBwdThreads, 1)
packed_dkdv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                   PackedBwdArgs args) {
  using L = KeySmem<D>;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
    prefetch_tmap(&tmDO);
  }
  int item_no, kvh;
  pa::unit_of(args.units, args.Hkv, args.at_once, item_no, kvh);
  const pa::KeyItem it = pa::load_key_item(args.items, item_no);
  const int G = args.G, P = args.P;
  const int n_q = (it.n_q + P - 1) / P;                   // row tiles
  const int used = G * P;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sK = smem;
  uint8_t* sV = smem + L::OFF_V;
  uint8_t* sStage = smem + L::OFF_STAGE;
  float* sVec = reinterpret_cast<float*>(smem + L::OFF_VEC);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* kv_full = bars + 0;
  uint64_t* q_full = bars + 1;      // [2]  bytes of the loads + 32 producer lanes
  uint64_t* q_empty = bars + 3;     // [2]
  uint64_t* s_full = bars + 5;
  uint64_t* dp_full = bars + 6;
  uint64_t* p_full = bars + 7;      // 8 warps
  uint64_t* ds_full = bars + 8;     // 8 warps
  uint64_t* done = bars + 9;
  uint64_t* tail = bars + 10;       // loads of the row tile that reaches over the sequence's end
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 11);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 12);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 1 + 32); mbar_init(&q_empty[i], 1); }
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_full, 8);
    mbar_init(ds_full, 8);
    mbar_init(done, 1);
    mbar_init(tail, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp >= 4 && warp < 8 && used < kT) {   // rows that no load writes: zeros, for good
    pa::zero_rows(sStage + (warp - 4) * L::TILE, L::DB, used, lane);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tDP = tmem + 128u, tDV = tmem + 256u, tDK = tmem + 256u + (uint32_t)D;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0 && n_q > 0) {
      mbar_expect_tx(kv_full, 2 * L::TILE);
      for (int db = 0; db < L::DB; ++db) {
        tma_load_3d(&tmK, kv_full, sK + db * L::BOX, db * 64, kvh, it.k_row);
        tma_load_3d(&tmV, kv_full, sV + db * L::BOX, db * 64, kvh, it.k_row);
      }
    }
    // this lane's four columns of a row tile: log-sum-exp and delta, fetched a tile ahead
    int col[4];
    float vl[4], vd[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = lane + 32 * e;
      col[e] = c / G * args.Hq + c % G;
    }
    const float* lse0 = args.lse + (long)it.q_row * args.Hq + kvh * G;
    const float* del0 = args.delta + (long)it.q_row * args.Hq + kvh * G;
    auto fetch = [&](int i) {
      const int rows = min(P, it.n_q - i * P) * G;
      const long at = (long)i * P * args.Hq;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = lane + 32 * e < rows;
        vl[e] = in ? lse0[at + col[e]] : 0.f;
        vd[e] = in ? del0[at + col[e]] : 0.f;
      }
    };
    if (n_q > 0) fetch(0);
    for (int i = 0; i < n_q && !*abort_flag; ++i) {
      const int st = i & 1;
      const int rows = min(P, it.n_q - i * P) * G;             // rows of the sequence in this tile
      const bool cut = rows < used;
      uint8_t* dst = sStage + st * L::STAGE;
      bool ok = true;
      if (lane == 0) ok = mbar_wait(&q_empty[st], ((i >> 1) & 1) ^ 1, args.err, kErrAttnProducer);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) { *abort_flag = 1; break; }
      if (lane == 0) {
        uint64_t* bar = cut ? tail : &q_full[st];
        mbar_expect_tx(bar, 2 * L::DB * used * 128);
        for (int db = 0; db < L::DB; ++db) {
          tma_load_3d(&tmQ, bar, dst + db * L::BOX, db * 64, kvh * G, it.q_row + i * P);
          tma_load_3d(&tmDO, bar, dst + L::TILE + db * L::BOX, db * 64, kvh * G, it.q_row + i * P);
        }
        if (cut) mbar_arrive(&q_full[st]);
      }
      float* v = sVec + st * 2 * kT;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[lane + 32 * e] = vl[e] * pa::kLog2e;
        v[kT + lane + 32 * e] = vd[e];
      }
      if (i + 1 < n_q) fetch(i + 1);
      if (cut) {
        ok = __all_sync(0xffffffffu, mbar_wait(tail, 0, args.err, kErrAttnProducer));
        if (!ok) { *abort_flag = 1; break; }
        pa::zero_rows(dst, 2 * L::DB, rows, lane);             // Q and dO boxes lie one behind another
        fence_proxy_async_smem();
      }
      mbar_arrive(&q_full[st]);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0 && n_q > 0) {
      constexpr uint32_t ID_T = idesc_bf16(128, kT);
      constexpr uint32_t ID_G = idesc_bf16(128, D, /*b_mn_major=*/true);
      const uint32_t ka = smem_u32(sK), va = smem_u32(sV);
      auto mma_nt = [&](uint32_t d, uint32_t xa, uint32_t ya) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k / 4) * L::BOX + (k % 4) * 32;
          umma_bf16(d, sdesc_sw128(xa + off, 16, 1024), sdesc_sw128(ya + off, 16, 1024), ID_T, k > 0 ? 1u : 0u);
        }
      };
      auto mma_ts = [&](uint32_t d, uint32_t a_tmem, uint32_t ya, bool acc) {
#pragma unroll
        for (int k = 0; k < kT / 16; ++k)
          umma_bf16_ts(d, a_tmem + pair_col(k), sdesc_sw128(ya + k * 2048, L::BOX, 1024), ID_G,
                       (acc || k > 0) ? 1u : 0u);
      };
      auto mma_rest = [&](uint32_t d, uint32_t a_tmem, uint32_t ya, int steps) {
        for (int k = 0; k < steps; ++k)
          umma_bf16_ts(d, a_tmem + 32u + pair_col(k), sdesc_sw128(ya + k * 2048, L::BOX, 1024), ID_G, 1u);
      };
      auto qa = [&](int i) { return smem_u32(sStage + (i & 1) * L::STAGE); };
      auto da = [&](int i) { return smem_u32(sStage + (i & 1) * L::STAGE + L::TILE); };
      bool ok = mbar_wait(kv_full, 0, args.err, kErrAttnMma) && mbar_wait(&q_full[0], 0, args.err, kErrAttnMma);
      if (ok) {
        tc_fence_after();
        mma_nt(tS, ka, qa(0));
        umma_commit(s_full);
        mma_nt(tDP, va, da(0));
        umma_commit(dp_full);
      }
      for (int i = 0; i < n_q && ok; ++i) {
        if (!(ok = mbar_wait(p_full, i & 1, args.err, kErrAttnMma))) break;
        tc_fence_after();
        mma_ts(tDV, tS, da(i), i > 0);
        const bool more = i + 1 < n_q;
        if (more) {
          if (!(ok = mbar_wait(&q_full[(i + 1) & 1], ((i + 1) >> 1) & 1, args.err, kErrAttnMma))) break;
          tc_fence_after();
          mma_nt(tS, ka, qa(i + 1));
          umma_commit(s_full);
        }
        if (!(ok = mbar_wait(ds_full, i & 1, args.err, kErrAttnMma))) break;
        tc_fence_after();
        mma_ts(tDK, tDP, qa(i), i > 0);
        if (kTwo) mma_rest(tDK, tDP, qa(i), (min(P, it.n_q - i * P) * G + 15) / 16);
        umma_commit(&q_empty[i & 1]);
        if (more) {
          mma_nt(tDP, va, da(i + 1));
          umma_commit(dp_full);
        }
      }
      if (!ok) *abort_flag = 1;
      umma_commit(done);
      mbar_wait(done, 0, args.err, kErrAttnTeardown);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ elementwise (warps 4..11)
    const int quarter = warp & 3;
    const int half = (warp - 4) >> 2;                       // columns half * 64 .. + 63
    const int r = quarter * 32 + lane;                      // key of the tile
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const float c2 = args.scale * pa::kLog2e;
    bool ok = true;
    for (int i = 0; i < n_q; ++i) {
      const int st = i & 1;
      const float* v = sVec + st * 2 * kT + half * 64;
      const int hi = min(P, it.n_q - i * P) * G - half * 64;          // columns of the sequence
      const int ahead = it.lead + r - i * P;                          // first position that sees key r
      const int lo = (args.causal && ahead > 0 ? min(ahead, kT) * G : 0) - half * 64;
      const bool full = __all_sync(0xffffffffu, lo <= 0 && hi >= 64);
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(&q_full[st], (i >> 1) & 1, args.err, kErrAttnSoftmax)))) break;
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(s_full, i & 1, args.err, kErrAttnSoftmax)))) break;
      tc_fence_after();
      uint32_t sr[64];
      tmem_ld32(tS + lane_off + half * 64, sr);
      tmem_ld32(tS + lane_off + half * 64 + 32, sr + 32);
      tmem_ld_wait();
      float p[64];
#pragma unroll
      for (int c4 = 0; c4 < 16; ++c4) {
        const float4 l4 = *reinterpret_cast<const float4*>(v + 4 * c4);
        const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 4 * c4 + e;
          p[c] = ex2(fmaf(__uint_as_float(sr[c]), c2, -lv[e]));
        }
      }
      if (!full) {
#pragma unroll
        for (int c = 0; c < 64; ++c) p[c] = (c >= lo && c < hi) ? p[c] : 0.f;
      }
#pragma unroll
      for (int c8 = 0; c8 < 8; ++c8) store_pairs(tS + lane_off + half * 64 + c8 * 4, p + 8 * c8);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(dp_full, i & 1, args.err, kErrAttnSoftmax)))) break;
      tc_fence_after();
      tmem_ld32(tDP + lane_off + half * 64, sr);
      tmem_ld32(tDP + lane_off + half * 64 + 32, sr + 32);
      tmem_ld_wait();
      const int rest = (hi + 15) / 16 * 16;                           // columns with a second number
      // a masked place is cleared by its own select: its P is 0, but 0 * NaN is not
      auto ds = [&](auto masked) {
#pragma unroll
        for (int c8 = 0; c8 < 8; ++c8) {
          const float4 d0 = *reinterpret_cast<const float4*>(v + kT + 8 * c8);
          const float4 d1 = *reinterpret_cast<const float4*>(v + kT + 8 * c8 + 4);
          const float dl[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
          float g[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int c = 8 * c8 + e;
            g[e] = p[c] * (__uint_as_float(sr[c]) - dl[e]);
            if (decltype(masked)::value) g[e] = (c >= lo && c < hi) ? g[e] : 0.f;
          }
          store_pairs(tDP + lane_off + half * 64 + c8 * 4, g);
          if (kTwo && 8 * c8 < rest) store_rest(tDP + lane_off + half * 64 + 32 + c8 * 4, g);
        }
      };
      if (full) ds(std::false_type{});
      else ds(std::true_type{});
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (!ok) *abort_flag = 1;
    if (n_q > 0) {
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(done, 0, args.err, kErrAttnTeardown)))) *abort_flag = 1;
      tc_fence_after();
    }
    // K and V have been read for the last time: their place stages the results
    uint8_t* buf = smem + (warp - 4) * 4096;
    const int c0 = half * (D / 2), left = args.Dr - c0;
    const bool valid = ok && r < it.n_k, one = it.n_keys == 1;   // one key: dS is 0, not what dP - delta leaves
    if (it.slot < 0) {
      const long at = valid ? ((long)(it.k_row + r) * args.Hkv + kvh) * args.Dr + c0 : -1;
      pa::store_rows<D / 2>(buf, tDV + lane_off + c0, n_q > 0, 1.0f, args.dv, at, left, lane);
      pa::store_rows<D / 2>(buf, tDK + lane_off + c0, n_q > 0 && !one, args.scale, args.dk, at, left, lane);
    } else {
      const long at = valid ? (((long)it.slot * args.Hkv + kvh) * 2 * kT + r) * args.Dr + c0 : -1;
      pa::store_rows32<D / 2>(buf, tDV + lane_off + c0, 1.0f, args.part, at, left, lane);
      pa::store_rows32<D / 2>(buf, tDK + lane_off + c0, one ? 0.f : args.scale, args.part + (long)kT * args.Dr, at, left, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dV and dK of key tiles whose queries were split: parts added in their order.  A warp per row, 8 rows
// a block.
__global__ void __launch_bounds__(256)
packed_join_kernel(const int* joins, int Hkv, int Dr, const float* part, __nv_bfloat16* dk, __nv_bfloat16* dv) {
  const int4 j = reinterpret_cast<const int4*>(joins)[blockIdx.x];   // k_row, n_k, first slot, parts
  const int kvh = blockIdx.y, which = blockIdx.z & 1, c = (threadIdx.x % 32) * 4;
  const int r = (blockIdx.z >> 1) * 8 + threadIdx.x / 32;
  if (c >= Dr || r >= j.y) return;
  const long stride = (long)Hkv * 2 * kT * Dr;
  const float* src = part + (((long)j.z * Hkv + kvh) * 2 * kT + which * kT + r) * Dr + c;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < j.w; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(src + s * stride);
    acc[0] += v.x; acc[1] += v.y; acc[2] += v.z; acc[3] += v.w;
  }
  uint2 w;
  w.x = pack_bf16x2(acc[0], acc[1]);
  w.y = pack_bf16x2(acc[2], acc[3]);
  *reinterpret_cast<uint2*>((which ? dk : dv) + ((long)(j.x + r) * Hkv + kvh) * Dr + c) = w;
}

// ---------------------------------------------------------------------------- dQ
template <int D>
struct RowSmem {
  static constexpr int BOX = kT * 128, DB = D / 64, TILE = DB * BOX;
  static constexpr int OFF_DO = TILE;
  static constexpr int OFF_KV = 2 * TILE;            // 2 slots of (K, V)
  static constexpr int SLOT = 2 * TILE;
  static constexpr int OFF_BAR = OFF_KV + 2 * SLOT;
  static constexpr int BYTES = OFF_BAR + 256 + 1024;
};

template <int D, bool kTwo>
__global__ void __launch_bounds__(kBwdThreads, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                 PackedBwdArgs args) {
  using L = RowSmem<D>;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
    prefetch_tmap(&tmDO);
  }
  int item_no, kvh;
  pa::unit_of(args.units, args.Hkv, args.at_once, item_no, kvh);
  const pa::FwdItem it = pa::load_fwd_item(args.items, item_no);
  const int G = args.G, P = args.P;
  const int n_kv = it.kt1;
  const int last_rows = it.n_keys - (n_kv - 1) * kT;
  const bool has_tail = n_kv > 0 && last_rows < kT;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sQ = smem;
  uint8_t* sDO = smem + L::OFF_DO;
  uint8_t* sKV = smem + L::OFF_KV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_full = bars + 0;
  uint64_t* kv_full = bars + 1;     // [2]
  uint64_t* kv_empty = bars + 3;    // [2]
  uint64_t* s_full = bars + 5;
  uint64_t* s_cons = bars + 6;      // 8 warps: S(j) is in registers
  uint64_t* dp_full = bars + 7;
  uint64_t* ds_full = bars + 8;     // 8 warps
  uint64_t* done = bars + 9;
  uint64_t* tail = bars + 10;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 11);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 12);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
    mbar_init(s_full, 1);
    mbar_init(s_cons, 8);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 8);
    mbar_init(done, 1);
    mbar_init(tail, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tDP = tmem + 128u, tDQ = tmem + 256u;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    bool ok = true;
    if (lane == 0 && n_kv > 0) {
      mbar_expect_tx(q_full, 2 * L::DB * G * P * 128);
      for (int db = 0; db < L::DB; ++db) {
        tma_load_3d(&tmQ, q_full, sQ + db * L::BOX, db * 64, kvh * G, it.q_row);
        tma_load_3d(&tmDO, q_full, sDO + db * L::BOX, db * 64, kvh * G, it.q_row);
      }
      for (int j = 0; j < n_kv && !*abort_flag; ++j) {
        const int sl = j & 1;
        if (!(ok = mbar_wait(&kv_empty[sl], ((j >> 1) & 1) ^ 1, args.err, kErrAttnProducer))) break;
        uint64_t* bar = has_tail && j == n_kv - 1 ? tail : &kv_full[sl];
        mbar_expect_tx(bar, L::SLOT);
        uint8_t* dst = sKV + sl * L::SLOT;
        for (int db = 0; db < L::DB; ++db) {
          tma_load_3d(&tmK, bar, dst + db * L::BOX, db * 64, kvh, it.k_row + j * kT);
          tma_load_3d(&tmV, bar, dst + L::TILE + db * L::BOX, db * 64, kvh, it.k_row + j * kT);
        }
      }
    }
    __syncwarp();
    if (has_tail) {                       // dQ += dS K sums over the keys: no rows of a neighbour
      ok = __shfl_sync(0xffffffffu, ok && !*abort_flag, 0);
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(tail, 0, args.err, kErrAttnProducer));
      if (ok) {
        const int sl = (n_kv - 1) & 1;
        pa::zero_rows(sKV + sl * L::SLOT, L::DB, last_rows, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[sl]);
      }
    }
    if (!ok) *abort_flag = 1;
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0 && n_kv > 0) {
      constexpr uint32_t ID_T = idesc_bf16(128, kT);
      constexpr uint32_t ID_G = idesc_bf16(128, D, /*b_mn_major=*/true);
      const uint32_t qa = smem_u32(sQ), doa = smem_u32(sDO);
      auto mma_nt = [&](uint32_t d, uint32_t xa, uint32_t ya) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k / 4) * L::BOX + (k % 4) * 32;
          umma_bf16(d, sdesc_sw128(xa + off, 16, 1024), sdesc_sw128(ya + off, 16, 1024), ID_T, k > 0 ? 1u : 0u);
        }
      };
      auto ka = [&](int j) { return smem_u32(sKV + (j & 1) * L::SLOT); };
      auto va = [&](int j) { return smem_u32(sKV + (j & 1) * L::SLOT + L::TILE); };
      bool ok = mbar_wait(q_full, 0, args.err, kErrAttnMma) && mbar_wait(&kv_full[0], 0, args.err, kErrAttnMma);
      if (ok) {
        tc_fence_after();
        mma_nt(tS, qa, ka(0));
        umma_commit(s_full);
        mma_nt(tDP, doa, va(0));
        umma_commit(dp_full);
      }
      for (int j = 0; j < n_kv && ok; ++j) {
        const bool more = j + 1 < n_kv;
        if (more) {
          if (!(ok = mbar_wait(s_cons, j & 1, args.err, kErrAttnMma))) break;
          if (!(ok = mbar_wait(&kv_full[(j + 1) & 1], ((j + 1) >> 1) & 1, args.err, kErrAttnMma))) break;
          tc_fence_after();
          mma_nt(tS, qa, ka(j + 1));
          umma_commit(s_full);
        }
        if (!(ok = mbar_wait(ds_full, j & 1, args.err, kErrAttnMma))) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < kT / 16; ++k)
          umma_bf16_ts(tDQ, tDP + pair_col(k), sdesc_sw128(ka(j) + k * 2048, L::BOX, 1024), ID_G,
                       (j > 0 || k > 0) ? 1u : 0u);
        if (kTwo) {
          for (int k = 0; k < (it.n_keys + 15) / 16; ++k)
            umma_bf16_ts(tDQ, tDP + 32u + pair_col(k), sdesc_sw128(ka(j) + k * 2048, L::BOX, 1024), ID_G, 1u);
        }
        umma_commit(&kv_empty[j & 1]);
        if (more) {
          mma_nt(tDP, doa, va(j + 1));
          umma_commit(dp_full);
        }
      }
      if (!ok) *abort_flag = 1;
      umma_commit(done);
      mbar_wait(done, 0, args.err, kErrAttnTeardown);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ elementwise (warps 4..11)
    const int quarter = warp & 3;
    const int half = (warp - 4) >> 2;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const float c2 = args.scale * pa::kLog2e;
    const int pos = min(r / G, it.n_q - 1);
    const bool in = r < G * P && r / G < it.n_q;
    int limit = args.causal ? min(it.n_keys, it.limit + pos) : it.n_keys;
    if (limit == 1) limit = 0;                              // one key: dS is 0, not what dP - delta leaves
    const long row = (long)(it.q_row + r / G) * args.Hq + kvh * G + r % G;
    const float lse2 = in ? args.lse[row] * pa::kLog2e : 0.f;
    const float dlt = in ? args.delta[row] : 0.f;
    const int rest = (it.n_keys + 15) / 16 * 16 - half * 64;      // columns with a second number
    bool ok = true;
    for (int j = 0; j < n_kv; ++j) {
      const int nv = limit - j * kT - half * 64;
      const bool full = __all_sync(0xffffffffu, nv >= 64);
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(s_full, j & 1, args.err, kErrAttnSoftmax)))) break;
      tc_fence_after();
      uint32_t sr[64];
      tmem_ld32(tS + lane_off + half * 64, sr);
      tmem_ld32(tS + lane_off + half * 64 + 32, sr + 32);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_cons);
      float p[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) p[c] = ex2(fmaf(__uint_as_float(sr[c]), c2, -lse2));
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(dp_full, j & 1, args.err, kErrAttnSoftmax)))) break;
      tc_fence_after();
      tmem_ld32(tDP + lane_off + half * 64, sr);
      tmem_ld32(tDP + lane_off + half * 64 + 32, sr + 32);
      tmem_ld_wait();
      auto ds = [&](auto masked) {
#pragma unroll
        for (int c8 = 0; c8 < 8; ++c8) {
          float g[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int c = 8 * c8 + e;
            g[e] = p[c] * (__uint_as_float(sr[c]) - dlt);
            if (decltype(masked)::value) g[e] = c < nv ? g[e] : 0.f;
          }
          store_pairs(tDP + lane_off + half * 64 + c8 * 4, g);
          if (kTwo && 8 * c8 < rest) store_rest(tDP + lane_off + half * 64 + 32 + c8 * 4, g);
        }
      };
      if (full) ds(std::false_type{});
      else ds(std::true_type{});
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (!ok) *abort_flag = 1;
    if (n_kv > 0) {
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(done, 0, args.err, kErrAttnTeardown)))) *abort_flag = 1;
      tc_fence_after();
    }
    // Q and dO have been read for the last time: their place stages the results
    const int c0 = half * (D / 2);
    pa::store_rows<D / 2>(smem + (warp - 4) * 4096, tDQ + lane_off + c0, n_kv > 0, args.scale, args.dq,
                          ok && in ? row * args.Dr + c0 : -1, args.Dr - c0, lane);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------- host
template <int D, bool kTwo>
static void launch_packed_bwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                              const CUtensorMap& tdo, PackedBwdArgs a, const at::Tensor& rows, const at::Tensor& keys,
                              int64_t row_heads, int64_t key_heads, cudaStream_t stream) {
  if (keys.size(0) > 0) {
    auto kern = packed_dkdv_kernel<D, kTwo>;
    smem_opt_in(reinterpret_cast<const void*>(kern), KeySmem<D>::BYTES);
    a.items = keys.data_ptr<int>();
    a.units = (int)(keys.size(0) * a.Hkv);
    a.at_once = (int)std::clamp<int64_t>(key_heads, 1, a.Hkv);
    kern<<<(unsigned)a.units, kBwdThreads, KeySmem<D>::BYTES, stream>>>(tq, tk, tv, tdo, a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  if (rows.size(0) > 0) {
    auto kern = packed_dq_kernel<D, kTwo>;
    smem_opt_in(reinterpret_cast<const void*>(kern), RowSmem<D>::BYTES);
    a.items = rows.data_ptr<int>();
    a.units = (int)(rows.size(0) * a.Hkv);
    a.at_once = (int)std::clamp<int64_t>(row_heads, 1, a.Hkv);
    kern<<<(unsigned)a.units, kBwdThreads, RowSmem<D>::BYTES, stream>>>(tq, tk, tv, tdo, a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

// (dq, dk, dv) bf16.  `rows`, `keys`, `joins`: work lists of ops.SequencePack on the device; `two`: dS as two
// numbers, for sequences of up to 32 rows.
std::vector<at::Tensor> packed_attn_bwd(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_,
                                        const at::Tensor& o_, const at::Tensor& dout_, const at::Tensor& lse_,
                                        const c10::optional<at::Tensor>& low,
                                        const at::Tensor& rows, const at::Tensor& keys, const at::Tensor& joins,
                                        int64_t slots, int64_t row_heads, int64_t key_heads, bool causal, double scale,
                                        bool fill, bool two) {
  TORCH_CHECK(std::abs(scale) < 1e38, "packed_attention: a finite scale");
  const at::Tensor q = pa::tma_rows(q_), k = pa::tma_rows(k_), v = pa::tma_rows(v_);
  const at::Tensor o = pa::tma_rows(o_.contiguous()), lse = lse_.contiguous();
  const at::Tensor dout = pa::tma_rows(dout_.to(at::kBFloat16).contiguous());
  const pa::Shape s = pa::check_shapes(q, k, v, "packed_attention");
  pa::check_operand(dout, q, "packed_attention: gradient");
  TORCH_CHECK(dout.is_contiguous() && o.is_contiguous() && dout.sizes() == q.sizes() && o.sizes() == q.sizes() &&
              o.scalar_type() == at::kBFloat16 && o.device() == q.device(),
              "packed_attention: contiguous output and gradient shaped like q");
  TORCH_CHECK(lse.is_contiguous() && lse.scalar_type() == at::kFloat && lse.device() == q.device() &&
              lse.numel() == (int64_t)s.Nq * s.Hq, "packed_attention: fp32 log-sum-exp [tokens, heads]");
  if (low.has_value())
    TORCH_CHECK(low->device() == q.device() && low->scalar_type() == at::kByte && low->is_contiguous() &&
                low->numel() == q.numel(), "packed_attention: remainder of the output [tokens, heads, head_dim]");
  pa::check_list(rows, 8, q, "packed_attention: rows");
  pa::check_list(keys, 8, q, "packed_attention: keys");
  pa::check_list(joins, 4, q, "packed_attention: joins");
  TORCH_CHECK(std::max(rows.size(0), keys.size(0)) * s.Hkv < (1ll << 30), "packed_attention: too much work for one call");
  c10::cuda::CUDAGuard guard(q.device());
  auto opt = q.options();
  auto make = [&](at::IntArrayRef sizes) { return fill ? at::zeros(sizes, opt) : at::empty(sizes, opt); };
  at::Tensor dq = make({s.Nq, s.Hq, s.D}), dk = make({s.Nk, s.Hkv, s.D}), dv = make({s.Nk, s.Hkv, s.D});
  if ((rows.size(0) == 0 && keys.size(0) == 0) || s.Hq == 0 || s.D == 0) return {dq, dk, dv};
  if (s.Nq == 0) return {dq, dk.zero_(), dv.zero_()};
  auto stream = c10::cuda::getCurrentCUDAStream();
  at::Tensor delta = at::empty({s.Nq, s.Hq}, opt.dtype(at::kFloat));
  const long n = (long)s.Nq * s.Hq;
  if (n > 0) {
    packed_delta_kernel<<<(unsigned)((n * 16 + 255) / 256), 256, 0, stream>>>(
        reinterpret_cast<const __nv_bfloat16*>(o.data_ptr()), low.has_value() ? low->data_ptr<uint8_t>() : nullptr,
        reinterpret_cast<const __nv_bfloat16*>(dout.data_ptr()), delta.data_ptr<float>(), n, s.D);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  PackedBwdArgs a{};
  a.G = s.G;
  a.P = pa::kRows / s.G;
  a.Hq = s.Hq;
  a.Hkv = s.Hkv;
  a.Dr = s.D;
  a.causal = causal ? 1 : 0;
  a.lse = lse.data_ptr<float>();
  a.delta = delta.data_ptr<float>();
  a.dq = reinterpret_cast<__nv_bfloat16*>(dq.data_ptr());
  a.dk = reinterpret_cast<__nv_bfloat16*>(dk.data_ptr());
  a.dv = reinterpret_cast<__nv_bfloat16*>(dv.data_ptr());
  a.scale = (float)scale;
  a.err = error_word(q.get_device());
  at::Tensor part;
  if (slots > 0) {
    part = at::empty({slots, s.Hkv, 2, pa::kRows, s.D}, opt.dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  const CUtensorMap tq = pa::tile_map(q, q, s.D, s.G, a.P), tdo = pa::tile_map(dout, q, s.D, s.G, a.P);
  const CUtensorMap tk = pa::tile_map(k, q, s.D, 1, pa::kRows), tv = pa::tile_map(v, q, s.D, 1, pa::kRows);
  auto launch = two ? (s.D > 64 ? launch_packed_bwd<128, true> : launch_packed_bwd<64, true>)
                    : (s.D > 64 ? launch_packed_bwd<128, false> : launch_packed_bwd<64, false>);
  launch(tq, tk, tv, tdo, a, rows, keys, row_heads, key_heads, stream);
  if (joins.size(0) > 0) {
    TORCH_CHECK(slots > 0, "packed_attention: joins without slots");
    packed_join_kernel<<<dim3((unsigned)joins.size(0), (unsigned)s.Hkv, 2 * kT / 8), 256, 0, stream>>>(
        joins.data_ptr<int>(), s.Hkv, s.D, a.part, a.dk, a.dv);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {dq, dk, dv};
}

}  // namespace osp
