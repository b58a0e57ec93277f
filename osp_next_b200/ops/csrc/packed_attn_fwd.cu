// Attention forward over packed sequences: causal or not, grouped heads, head dims to 128, queries
// that are the last tokens of their keys, a bias by relative position (tcgen05 + TMEM + TMA).
//
//   S = scale q k^T + bias;  o = softmax(S) v over the keys that a query sees;  lse = log sum exp S
//
// A CTA computes one or two row tiles (packed_attn.cuh) that pass over the same key tiles, as the
// kernel in attention_fwd.cuh does: four warps a tile for the softmax (a thread per row, running
// maximum and sum in fp32, O rescaled only when the maximum grows by more than 2^8), one warp for the
// TMA loads and one for the MMAs; P goes to bf16 in tensor memory, over S.  Under a causal mask tile 0
// needs up to one key tile less than tile 1 and leaves the rest out.  A row's keys are those below
// a limit, so the mask costs one comparison per score, in tiles that hold such a limit only.
//
// Items with many keys and few rows are split along the keys: each part leaves its normalised fp32
// output, maximum and sum in a workspace and packed_combine_kernel joins them.
//
// What bounds it: long sequences the tensor pipe and the softmax in turn (20161 tokens, 28 heads of 128
// to 4, causal: 2.6 to 2.9 ms, 1000 to 1100 TFLOP/s); one query each over long keys memory (48 x 1024 to
// 8192 keys, 8 key heads: 127 to 138 us, 0.75 of the copy rate); short sequences the latency of a CTA's chain of
// load, product, softmax, product and store, some 9000 cycles beside 5000 a key tile (32 prompts of 20
// to 512 tokens, 64 heads of 64, bias: 136 us).  The bias is staged in shared memory, twice, one place
// apart, so that rows read aligned pairs (from global memory: 162 us there).
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>

#include "attention_fwd.cuh"
#include "packed_attn.cuh"
#include "packed_attn_host.h"

namespace osp {

struct PackedFwdArgs {
  const int* items;
  int units;                // items x heads that they are run for
  int heads;                // key heads, or query heads where a tile holds one head (bias)
  int at_once;              // heads run together (pa::unit_of)
  int kv_ratio;             // of those to one key head
  int G, P, Hq, Dr;         // heads and positions of a tile, query heads, head dim
  int causal;
  int q_box;                // bytes of a query box in shared memory (G * P rows, to 1024 bytes)
  int q_tile;               // of a row tile's queries, whose place its results take on their way out
  int slots;                // of the K / V ring
  __nv_bfloat16* out;       // [Nq, Hq, Dr]
  float* lse;               // [Nq, Hq] or null
  uint8_t* low;             // [Nq, Hq, Dr] what o's rounding left (pa::low_bits), or null
  float scale_log2;
  const float* bias;        // [Hq, 2 M - 1] or null
  int bias_m;               // M
  float* part_o;            // [slots, heads, kTiles * 128, Dr]
  float2* part_l;           // [slots, heads, kTiles * 128] (maximum, sum of 2^(S - maximum)), log2 domain
  int* err;
};

// kTiles row tiles in a CTA.  Two share the key tiles that they pass over and take turns on the tensor
// core; one leaves room for a second CTA on the SM (256 columns of tensor memory, at most 113 KB).
template <int D, int kTiles, bool kBias>
struct PackedFwdCfg {
  static constexpr int kProdWarp = 4 * kTiles, kMmaWarp = kProdWarp + 1, kThreads = 32 * (kProdWarp + 2);
  static constexpr int kCtas = kTiles == 2 ? 1 : 2;            // per SM
  static constexpr int BOX = pa::kRows * 128;
  static constexpr int DB = D / 64;
  static constexpr int TILE = DB * BOX;
  static constexpr int kMaxSlots = 5;
  static constexpr int kPiece = kTiles == 2 ? 128 : 64;        // bytes of a row of results that leave at once
  static constexpr int kOut = 32 * kPiece;                     // of a warp's 32 rows
  static constexpr int kBiasBytes = kBias ? 2 * 2 * 2 * pa::kRows * 4 : 0;   // of a row tile: 2 x 2 x 256 entries
  static constexpr int kRoom = kTiles == 2 ? 232448 : 115712;  // dynamic shared memory of a CTA
  // barriers and bias lie in front, at fixed places: pointers cost the softmax no registers
  static constexpr int OFF_BIAS = 1024;
  static constexpr int OFF_Q = OFF_BIAS + kTiles * kBiasBytes;
  static_assert(OFF_Q % 1024 == 0, "swizzled tiles");
  static constexpr int kExtra = OFF_Q + 1024;                  // + alignment of the base
  static constexpr uint32_t kCols = kTiles == 2 ? 512 : 256;
};

// Work of a CTA: an item of the list for one head.
template <int kTiles>
struct FwdUnit {
  pa::FwdItem it;
  int head, kvh;
  int n_t[kTiles];          // key tiles of each row tile: those below the limit of its last query
  int c_t[kTiles];          // columns of the last of them that any row sees
  int n_kv, last_rows;      // key tiles loaded, keys of the sequence in the last one
  bool has_tail;

  __device__ FwdUnit(const PackedFwdArgs& args, const pa::FwdItem& item, int h) : it(item), head(h) {
    constexpr int kT = pa::kRows;
    kvh = head / args.kv_ratio;
    n_kv = 0;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const int nq = min(args.P, it.n_q - t * args.P);
      const int lim = max(0, args.causal ? min(it.n_keys, it.limit + t * args.P + nq - 1) : it.n_keys);
      n_t[t] = nq > 0 ? max(0, min(it.kt1, (lim + kT - 1) / kT) - it.kt0) : 0;
      c_t[t] = min(kT, lim - (it.kt0 + n_t[t] - 1) * kT);
      n_kv = max(n_kv, n_t[t]);
    }
    last_rows = it.n_keys - (it.kt0 + n_kv - 1) * kT;
    has_tail = n_kv > 0 && last_rows < kT;
  }
};

// A bias times log2 e, to +-1e38: the type's lowest value hides a key, and a tile that it fills keeps a finite
// maximum (-inf - -inf is NaN), which the first key that is not hidden replaces.  A NaN stays one.
__device__ __forceinline__ float finite_bias(float b) {
  b *= pa::kLog2e;
  b = b < -1e38f ? -1e38f : b;
  return b > 1e38f ? 1e38f : b;
}

// Row maximum over the columns below `cols` (the warp's) and n_valid (the row's).
__device__ __forceinline__ float masked_max(const uint32_t* sr, int cols, int n_valid) {
  float mx = -INFINITY;
#pragma unroll
  for (int g = 0; g < pa::kRows / 16; ++g) {
    if (g * 16 >= cols) break;
    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int c = g * 16 + i;
      m4[i & 3] = fmaxf(m4[i & 3], c < n_valid ? __uint_as_float(sr[c]) : -INFINITY);
    }
    mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
  }
  return mx;
}

template <int D, bool kBias, int kTiles>
__global__ void __launch_bounds__(PackedFwdCfg<D, kTiles, kBias>::kThreads, PackedFwdCfg<D, kTiles, kBias>::kCtas)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, PackedFwdArgs args) {
  using L = PackedFwdCfg<D, kTiles, kBias>;
  using Unit = FwdUnit<kTiles>;
  constexpr int kT = pa::kRows, kMaxSlots = L::kMaxSlots;
  constexpr uint32_t kO = 128u * kTiles;                       // tensor memory: S tiles, then O tiles
  const int G = args.G, P = args.P, slots = args.slots;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  uint8_t* sQ = smem + L::OFF_Q;
  uint8_t* sKV = sQ + kTiles * args.q_tile;
  uint64_t* q_full = bars + 0;
  uint64_t* tail = bars + 1;                       // the V tile that reaches over the sequence's end
  uint64_t* kv_full = bars + 2;                    // [slots]
  uint64_t* kv_empty = kv_full + kMaxSlots;        // [slots]
  uint64_t* s_full = kv_empty + kMaxSlots;         // [kTiles]
  uint64_t* p_half = s_full + kTiles;              // [kTiles]
  uint64_t* p_full = p_half + kTiles;              // [kTiles]
  uint64_t* o_done = p_full + kTiles;              // [kTiles]
  uint64_t* bias_full = o_done + kTiles;           // [kTiles] a key tile's stretch of the bias, by the tile's four warps
  uint64_t* done = bias_full + kTiles;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(done + 2);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;

  // the item's fetch and the tensor maps' run under the set-up; the copy is for the way out
  int item_no, unit_head;
  pa::unit_of(args.units, args.heads, args.at_once, item_no, unit_head);
  const pa::FwdItem item = pa::load_fwd_item(args.items, item_no);
  pa::FwdItem* item_copy = reinterpret_cast<pa::FwdItem*>(smem + 512);
  if (warp == L::kProdWarp && lane == 0) {
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
    *item_copy = item;
  }
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(tail, 1);
    for (int i = 0; i < slots; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_half[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
      mbar_init(&bias_full[t], 4);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == L::kMmaWarp) {
    tmem_alloc(tmem_slot, L::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == L::kProdWarp) {
    // ------------------------------------------------------------------ producer
    bool ok = true;
    int slot = 0;
    uint32_t phase = 1;
    {
      const Unit un(args, item, unit_head);
      const int krow0 = un.it.k_row + un.it.kt0 * kT;
      const int units = 2 * un.n_kv;
      if (lane == 0 && un.n_kv > 0) {
        {
          int tiles = 0;
#pragma unroll
          for (int t = 0; t < kTiles; ++t) tiles += un.n_t[t] > 0;
          mbar_expect_tx(q_full, tiles * L::DB * G * P * 128);
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            for (int db = 0; db < L::DB && un.n_t[t] > 0; ++db)
              tma_load_3d(&tmQ, q_full, sQ + t * args.q_tile + db * args.q_box, db * 64, un.head * G, un.it.q_row + t * P);
        }
        for (int i = 0; i < units && ok; ++i) {
          if (*abort_flag || !mbar_wait(&kv_empty[slot], phase, args.err, kErrAttnProducer)) { ok = false; break; }
          uint64_t* bar = un.has_tail && i == units - 1 ? tail : &kv_full[slot];
          mbar_expect_tx(bar, L::TILE);
          const CUtensorMap* tm = (i & 1) ? &tmV : &tmK;
          for (int db = 0; db < L::DB; ++db)
            tma_load_3d(tm, bar, sKV + slot * L::TILE + db * L::BOX, db * 64, un.kvh, krow0 + (i >> 1) * kT);
          if (++slot == slots) { slot = 0; phase ^= 1; }
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (ok && un.has_tail) {
        ok = __all_sync(0xffffffffu, mbar_wait(tail, 0, args.err, kErrAttnProducer));
        if (ok) {
          const int at = __shfl_sync(0xffffffffu, slot == 0 ? slots - 1 : slot - 1, 0);
          pa::zero_rows(sKV + at * L::TILE, L::DB, un.last_rows, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&kv_full[at]);
        }
      }
    }
    if (!ok) *abort_flag = 1;
  } else if (warp == L::kMmaWarp) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t ID_S = idesc_bf16(128, kT);
      constexpr uint32_t ID_PV = idesc_bf16(128, D, /*b_mn_major=*/true);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, args.err, kErrAttnMma); };
      auto issue_s = [&](int t, int slot) {
        const uint32_t qa = smem_u32(sQ + t * args.q_tile);
        const uint32_t ka = smem_u32(sKV + slot * L::TILE);
        const uint32_t d = tmem + 128u * t;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_bf16(d, sdesc_sw128(qa + (k / 4) * args.q_box + (k % 4) * 32, 16, 1024),
                    sdesc_sw128(ka + (k / 4) * L::BOX + (k % 4) * 32, 16, 1024), ID_S, k > 0 ? 1u : 0u);
        umma_commit(&s_full[t]);
      };
      // P V over the keys of this tile: its last one may have fewer
      auto pv = [&](int t, const Unit& un, int j, int slot) -> bool {
        const uint32_t va = smem_u32(sKV + slot * L::TILE);
        const uint32_t d = tmem + kO + (uint32_t)D * t;
        const uint32_t pr = tmem + 128u * t;
        auto mma = [&](int k, bool acc) {
          umma_bf16_ts(d, pr + 8u * k, sdesc_sw128(va + k * 2048, L::BOX, 1024), ID_PV, acc ? 1u : 0u);
        };
        const int steps = j + 1 == un.n_t[t] ? (un.c_t[t] + 15) / 16 : kT / 16;
        if (!wait(&p_half[t], j & 1)) return false;
        tc_fence_after();
        if (steps == kT / 16) {                    // a rolled loop issues too slowly for whole tiles
#pragma unroll
          for (int k = 0; k < kT / 32; ++k) mma(k, j > 0 || k > 0);
        } else {
          for (int k = 0; k < min(steps, kT / 32); ++k) mma(k, j > 0 || k > 0);
        }
        if (!wait(&p_full[t], j & 1)) return false;
        tc_fence_after();
        if (steps == kT / 16) {
#pragma unroll
          for (int k = kT / 32; k < kT / 16; ++k) mma(k, true);
        } else {
          for (int k = kT / 32; k < steps; ++k) mma(k, true);
        }
        if (j + 1 == un.n_t[t]) umma_commit(&o_done[t]);
        return true;
      };
      bool ok = true;
      int slot = 0;
      uint32_t phase = 0;
      auto next = [&] { if (++slot == slots) { slot = 0; phase ^= 1; } };
      const Unit un(args, item, unit_head);
      const int n_kv = un.n_kv, n0 = un.n_t[0], n1 = un.n_t[kTiles - 1];
      if (n_kv > 0) ok = wait(q_full, 0) && wait(&kv_full[slot], phase);
      if (n_kv > 0 && ok) {
        tc_fence_after();
        if (n0 > 0) issue_s(0, slot);
        if (kTiles == 2 && n1 > 0) issue_s(1, slot);
        umma_commit(&kv_empty[slot]);
        next();
        for (int j = 0; j < n_kv; ++j) {
          const int sV = slot;
          if (!(ok = wait(&kv_full[sV], phase))) break;
          next();
          tc_fence_after();
          if (j < n0 && !(ok = pv(0, un, j, sV))) break;
          if (kTiles == 1) umma_commit(&kv_empty[sV]);
          const int sK = slot;
          if (j + 1 < n_kv) {
            if (!(ok = wait(&kv_full[sK], phase))) break;
            next();
            tc_fence_after();
            if (j + 1 < n0) issue_s(0, sK);
          }
          if (kTiles == 2) {
            if (j < n1 && !(ok = pv(1, un, j, sV))) break;
            umma_commit(&kv_empty[sV]);
            if (j + 1 < n1) issue_s(1, sK);
          }
          if (j + 1 < n_kv) umma_commit(&kv_empty[sK]);
        }
      }
      if (!ok) *abort_flag = 1;
      umma_commit(done);
      mbar_wait(done, 0, args.err, kErrAttnTeardown);
    }
  } else {
    // ------------------------------------------------------------------ softmax
    const int t = warp / 4;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;                // row of the tile
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + 128u * t + lane_off;
    const uint32_t tO = tS + kO + (uint32_t)(D - 128) * t;
    const float sl2 = args.scale_log2;
    float* bias_buf = reinterpret_cast<float*>(smem + L::OFF_BIAS + t * L::kBiasBytes);
    bool ok = true;
    do {
      // what the passes over the keys need; the rest of the unit is read again behind them, as the
      // scores of a row take 128 of a thread's 168 registers
      int n, last_cols, limit, bias_at, bias_row, bias_off;
      bool idle;
      {
        const Unit un(args, item, unit_head);
        const int nq = min(P, un.it.n_q - t * P);       // queries of the tile (<= 0: it has none)
        if (nq <= 0) break;                             // uniform for the tile's warps
        const int pos = min(r / G, nq - 1);             // rows behind the last query repeat its mask
        idle = !__any_sync(0xffffffffu, r / G < nq && r < G * P);   // a warp without rows keeps step, no more
        const int first = un.it.limit + t * P;          // 1 + position of the tile's first query
        limit = args.causal ? min(un.it.n_keys, first + pos) : un.it.n_keys;
        n = t == 0 ? un.n_t[0] : un.n_t[kTiles - 1];
        last_cols = t == 0 ? un.c_t[0] : un.c_t[kTiles - 1];
        const int key0 = un.it.kt0 * kT;
        // entry e of a key tile's stretch of the bias: key - position = key0 + e - (P - 1) - (first - 1)
        bias_at = key0 + r - P - first + 1 + args.bias_m;
        bias_row = un.head;
        limit -= key0;
        bias_off = P - 1 - pos;                         // even, or odd and one further on in the second copy
        bias_off += bias_off & 1 ? 2 * kT + 1 : 0;
      }
      float m_ref = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j) {
        if (kBias) {
          const float* row = args.bias + (long)bias_row * (2 * args.bias_m - 1);
          // twice, the second time one place further on, so that every row reads aligned pairs
          float* dst = bias_buf + (j & 1) * 4 * kT;
#pragma unroll
          for (int e = 0; e < 2 * kT; e += kT) {
            const int at = bias_at + j * kT + e;
            const float b = at >= 0 && at < 2 * args.bias_m - 1 ? finite_bias(row[at]) : 0.f;
            dst[r + e] = b;
            dst[2 * kT + ((r + e + 1) & (2 * kT - 1))] = b;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bias_full[t]);
          if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bias_full[t], j & 1, args.err, kErrAttnSoftmax)))) break;
        }
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], j & 1, args.err, kErrAttnSoftmax)))) break;
        tc_fence_after();
        const int n_valid = limit - j * kT;
        const int cols = j + 1 == n ? last_cols : kT;   // columns that any row of the tile sees
        const bool full = __all_sync(0xffffffffu, n_valid >= kT);
        if (!idle) {
          uint32_t sr[kT];
#pragma unroll
          for (int c = 0; c < kT / 32; ++c) tmem_ld32(tS + c * 32, sr + c * 32);
          tmem_ld_wait();
          if (kBias) {
            const float* brow = bias_buf + (j & 1) * 4 * kT + bias_off;
            const uint64_t sl2x2 = pk2(sl2, sl2);
#pragma unroll
            for (int g = 0; g < kT / 32; ++g) {
              if (g * 32 >= cols) break;
#pragma unroll
              for (int c = g * 32; c < g * 32 + 32; c += 2) {
                const float2 b = *reinterpret_cast<const float2*>(brow + c);
                float x, y;
                upk2(ffma2(pk2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), sl2x2, pk2(b.x, b.y)), x, y);
                sr[c] = __float_as_uint(x);
                sr[c + 1] = __float_as_uint(y);
              }
            }
          }
          const float mul = kBias ? 1.0f : sl2;
          float mx = full ? attn_row_max<kT, true>(sr, kT) : masked_max(sr, cols, n_valid);
          mx *= mul;
          const bool need = mx > m_ref + 8.0f;
          const float m_new = need ? mx : m_ref;
          // O is stable here: the PV of step j - 1 was issued before S(j), whose completion we waited for
          if (j > 0 && __any_sync(0xffffffffu, need)) {
            const float alpha = need ? ex2(m_ref - m_new) : 1.0f;
            l *= alpha;
            attn_rescale_o(tO, D, alpha);
          }
          m_ref = m_new;
          if (full) {
            l += attn_exp_store<64, true, 0u, 0>(sr, mul, m_ref, 64, tS);
          } else {
#pragma unroll
            for (int g = 0; g < 4; ++g)
              if (g * 16 < cols)
                l += attn_exp_store<16, false, 0u, 0>(sr + g * 16, mul, m_ref, n_valid - g * 16, tS + g * 8);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_half[t]);
          if (full) {
            l += attn_exp_store<64, true, 0u, 4>(sr + 64, mul, m_ref, 64, tS + 32);
          } else {
#pragma unroll
            for (int g = 4; g < 8; ++g)
              if (g * 16 < cols)
                l += attn_exp_store<16, false, 0u, 0>(sr + g * 16, mul, m_ref, n_valid - g * 16, tS + g * 8);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[t]);
        } else if (lane == 0) {
          mbar_arrive(&p_half[t]);
          mbar_arrive(&p_full[t]);
        }
      }
      if (ok && n > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], 0, args.err, kErrAttnSoftmax));
      }
      if (!ok) break;
      if (idle) break;
      tc_fence_after();
      const float inv_l = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);   // no key seen: 0; NaN stays
      const float lse2 = m_ref + __log2f(l);
      const pa::FwdItem it = *item_copy;
      const int rp = r / G, rh = r - rp * G;            // position and head of the row
      const bool in = rp < min(P, it.n_q - t * P) && r < G * P;
      const long row = (long)(it.q_row + t * P + rp) * args.Hq + unit_head * G + rh;
      const long prow = ((long)it.slot * args.heads + unit_head) * (kTiles * kT) + t * kT + r;
      if (in) {
        if (it.slot >= 0) args.part_l[prow] = make_float2(m_ref, l);
        else if (args.lse) args.lse[row] = lse2 * 0.69314718055994531f;
      }
      // kPiece bytes of each row at a time through shared memory, so that kPiece / 16 lanes write a
      // row's piece; the row's place comes from the lane that owns it
      constexpr int kLanes = L::kPiece / 16;
      uint8_t* buf = sQ + t * args.q_tile + quarter * L::kOut;   // the last S has been formed
      const int size = it.slot < 0 ? 2 : 4;             // bytes per value
      const int per = L::kPiece / size;                 // values of a row per pass: 64, 32 or 16
      const long at = in ? (it.slot < 0 ? row : prow) * args.Dr * size : -1;
      uint8_t* base = it.slot < 0 ? reinterpret_cast<uint8_t*>(args.out) : reinterpret_cast<uint8_t*>(args.part_o);
      const int piece = lane % kLanes;
      uint32_t o[32];
#pragma unroll 1
      for (int c0 = 0; c0 < args.Dr; c0 += 16) {        // 16 columns at a time
        if (c0 % 32 == 0) {
          if (n > 0) {
            tmem_ld32(tO + c0, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = o[i + 16];
        }
        const int first = c0 % per * size / 16;         // the first piece that these columns fill
        if (args.low && size == 2 && in) {              // for the gradient: 16 bytes of this lane's own row
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (c0 + 8 * h < args.Dr)
              *reinterpret_cast<uint2*>(args.low + row * args.Dr + c0 + 8 * h) = pa::low_bits8(o + 8 * h, inv_l);
        }
        if (size == 2) {
#pragma unroll
          for (int i = 0; i < 2; ++i) *pa::out_piece<L::kPiece>(buf, lane, first + i) = pa::pack8(o + 8 * i, inv_l);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(pa::out_piece<L::kPiece>(buf, lane, first + i)) =
                make_float4(__uint_as_float(o[4 * i]) * inv_l, __uint_as_float(o[4 * i + 1]) * inv_l,
                            __uint_as_float(o[4 * i + 2]) * inv_l, __uint_as_float(o[4 * i + 3]) * inv_l);
        }
        if ((c0 + 16) % per != 0 && c0 + 16 < args.Dr) continue;
        __syncwarp();
        const int b0 = c0 / per * L::kPiece + piece * 16;   // byte of the row
#pragma unroll
        for (int i = 0; i < 32 / (32 / kLanes); ++i) {
          const int rr = i * (32 / kLanes) + lane / kLanes;
          const long to = __shfl_sync(0xffffffffu, at, rr);
          if (to >= 0 && b0 < args.Dr * size)
            *reinterpret_cast<uint4*>(base + to + b0) = *pa::out_piece<L::kPiece>(buf, rr, piece);
        }
        __syncwarp();
      }
    } while (false);
    if (!ok) *abort_flag = 1;
  }

  tc_fence_before();
  __syncthreads();
  if (warp == L::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kCols);
  }
}

// o = sum_i w_i o_i / sum_i w_i over the parts of one item, w_i = l_i 2^(m_i - m) from their maxima and sums
// (apart: next to a maximum of 1e38 the logarithm of a sum would be lost).  A warp per row; block (join, key
// head, 8 rows).  The parts' weights are read by the lanes at once, 32 parts at a time.
__global__ void __launch_bounds__(256)
packed_combine_kernel(const int* joins, int G, int P, int tiles, int Hq, int Dr, const float* part_o,
                      const float2* part_l, __nv_bfloat16* out, float* lse, uint8_t* low) {
  const int4 j = reinterpret_cast<const int4*>(joins)[blockIdx.x];   // q_row, n_q, first slot, parts
  const int kvh = blockIdx.y, lane = threadIdx.x % 32;
  const int i = blockIdx.z * 8 + threadIdx.x / 32;
  if (i >= j.y * G) return;
  const int p = i / G, g = i % G, t = p / P;
  const long stride = (long)gridDim.y * tiles * pa::kRows;
  const long first = (long)j.z * stride + (long)kvh * tiles * pa::kRows + t * pa::kRows + (p - t * P) * G + g;
  float top = -INFINITY;
  for (int s = lane; s < j.w; s += 32) top = fmaxf(top, part_l[first + s * stride].x);   // NaN is in the sums
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < j.w; s0 += 32) {
    float mine = 0.f;
    if (s0 + lane < j.w) {
      const float2 ml = part_l[first + (s0 + lane) * stride];
      mine = exp2f(ml.x - base) * ml.y;
    }
    const int n = min(32, j.w - s0);
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float w = __shfl_sync(0xffffffffu, mine, s);
      sum += w;
      if (lane * 4 < Dr) {                     // a part without keys has zeros and weight 0
        const float4 v = *reinterpret_cast<const float4*>(part_o + (first + (s0 + s) * stride) * Dr + lane * 4);
        acc[0] += w * v.x; acc[1] += w * v.y; acc[2] += w * v.z; acc[3] += w * v.w;
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const long row = (long)(j.x + p) * Hq + kvh * G + g;
  if (lane * 4 < Dr) {
    uint2 w;
    w.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    w.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<uint2*>(out + row * Dr + lane * 4) = w;
    if (low) *reinterpret_cast<uint32_t*>(low + row * Dr + lane * 4) = pa::low_bits4(acc, inv);
  }
  if (lane == 0 && lse) lse[row] = (base + log2f(sum)) * 0.69314718055994531f;
}

template <int D, bool kBias, int kTiles>
static void launch_packed_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, PackedFwdArgs a,
                              cudaStream_t stream) {
  using L = PackedFwdCfg<D, kTiles, kBias>;
  a.q_box = (a.G * a.P * 128 + 1023) / 1024 * 1024;
  a.q_tile = std::max(L::DB * a.q_box, 4 * L::kOut);
  const int q_bytes = kTiles * a.q_tile;
  a.slots = std::min(L::kMaxSlots, (L::kRoom - L::kExtra - q_bytes) / L::TILE);
  auto kern = packed_fwd_kernel<D, kBias, kTiles>;
  smem_opt_in(reinterpret_cast<const void*>(kern), L::kRoom);
  kern<<<a.units, L::kThreads, q_bytes + a.slots * L::TILE + L::kExtra, stream>>>(tq, tk, tv, a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <int D, bool kBias>
static void launch_packed_fwd(int64_t tiles, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                              const PackedFwdArgs& a, cudaStream_t stream) {
  if (tiles == 1) launch_packed_fwd<D, kBias, 1>(tq, tk, tv, a, stream);
  else launch_packed_fwd<D, kBias, 2>(tq, tk, tv, a, stream);
}

// (o [Nq, Hq, D] bf16, lse [Nq, Hq] fp32 or empty, what o's rounding left or empty).  `items` / `joins` are int32 lists on the device,
// laid out by ops.SequencePack for this group size; the pack needs `rows` and `key_rows`, its longest
// sequence has `longest` rows.  Rows of no sequence are zeros.
std::vector<at::Tensor> packed_attn_fwd(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_,
                                        const at::Tensor& items, const at::Tensor& joins, int64_t slots,
                                        int64_t positions, int64_t tiles, int64_t at_once, bool causal, double scale,
                                        bool own_scale,
                                        const c10::optional<at::Tensor>& rel_bias_, bool want_lse, bool want_low,
                                        int64_t rows,
                                        int64_t key_rows, int64_t longest, bool dense) {
  TORCH_CHECK(own_scale || std::abs(scale) < 1e38, "packed_attention: a finite scale");
  // a row's maximum is taken before the scale, which has to be positive: (-q) k (-scale) otherwise
  const bool flip = !own_scale && scale < 0;
  if (flip) scale = -scale;
  const at::Tensor q = pa::tma_rows(flip ? q_.neg() : q_), k = pa::tma_rows(k_), v = pa::tma_rows(v_);
  const pa::Shape s = pa::check_shapes(q, k, v, "packed_attention");
  TORCH_CHECK(s.Nq >= rows && s.Nk >= key_rows, "packed_attention: fewer rows than the pack's");
  pa::check_list(items, 8, q, "packed_attention: items");
  pa::check_list(joins, 4, q, "packed_attention: joins");
  if (own_scale) scale = 1.0 / std::sqrt((double)std::max(1, s.D));
  const bool fill = !(dense && s.Nq == rows);
  c10::optional<at::Tensor> rel_bias;
  if (rel_bias_.has_value()) rel_bias = rel_bias_->to(at::kFloat).contiguous();
  c10::cuda::CUDAGuard guard(q.device());
  auto opt = q.options();
  at::Tensor out = fill ? at::zeros({s.Nq, s.Hq, s.D}, opt) : at::empty({s.Nq, s.Hq, s.D}, opt);
  at::Tensor lse;
  if (want_lse) {
    lse = at::empty({s.Nq, s.Hq}, opt.dtype(at::kFloat));
    if (fill) lse.fill_(-INFINITY);
  }
  at::Tensor low;
  if (want_low) low = at::empty({s.Nq, s.Hq, s.D}, opt.dtype(at::kByte));
  if (want_low && fill) low.zero_();
  const int64_t n = items.size(0);
  if (n == 0 || s.Hq == 0 || s.D == 0) return {out, lse, low};
  PackedFwdArgs a{};
  a.items = items.data_ptr<int>();
  // with a bias a tile holds one query head: its rows then read one stretch of the bias
  const int group = rel_bias.has_value() ? 1 : s.G;
  a.G = group;
  a.heads = s.Hq / group;
  a.kv_ratio = a.heads / s.Hkv;
  TORCH_CHECK(n * a.heads < (1ll << 30), "packed_attention: too much work for one call");
  a.units = (int)(n * a.heads);
  a.at_once = (int)std::clamp<int64_t>(at_once, 1, a.heads);
  a.P = (int)positions;
  TORCH_CHECK(a.P >= 1 && a.P * group <= pa::kRows && (tiles == 1 || tiles == 2), "packed_attention: row tiles");
  a.Hq = s.Hq;
  a.Dr = s.D;
  a.causal = causal ? 1 : 0;
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  a.low = want_low ? low.data_ptr<uint8_t>() : nullptr;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  if (rel_bias.has_value()) {
    TORCH_CHECK(rel_bias->is_cuda() && rel_bias->device() == q.device() && rel_bias->scalar_type() == at::kFloat &&
                rel_bias->is_contiguous() && rel_bias->dim() == 2 && rel_bias->size(0) == s.Hq &&
                rel_bias->size(1) % 2 == 1 && rel_bias->size(1) >= 2 * longest - 1,
                "packed_attention: rel_bias fp32 [heads, 2 M - 1], M at least the longest sequence");
    a.bias = rel_bias->data_ptr<float>();
    a.bias_m = (int)((rel_bias->size(1) + 1) / 2);
  }
  a.err = error_word(q.get_device());
  at::Tensor part_o, part_l;
  if (slots > 0) {
    part_o = at::empty({slots, a.heads, tiles * pa::kRows, s.D}, opt.dtype(at::kFloat));
    part_l = at::empty({slots, a.heads, tiles * pa::kRows, 2}, opt.dtype(at::kFloat));
    a.part_o = part_o.data_ptr<float>();
    a.part_l = reinterpret_cast<float2*>(part_l.data_ptr<float>());
  }
  const CUtensorMap tq = pa::tile_map(q, q, s.D, group, a.P);
  const CUtensorMap tk = pa::tile_map(k, q, s.D, 1, pa::kRows), tv = pa::tile_map(v, q, s.D, 1, pa::kRows);
  auto stream = c10::cuda::getCurrentCUDAStream();
  if (s.D > 64) {
    if (a.bias) launch_packed_fwd<128, true>(tiles, tq, tk, tv, a, stream);
    else launch_packed_fwd<128, false>(tiles, tq, tk, tv, a, stream);
  } else {
    if (a.bias) launch_packed_fwd<64, true>(tiles, tq, tk, tv, a, stream);
    else launch_packed_fwd<64, false>(tiles, tq, tk, tv, a, stream);
  }
  if (joins.size(0) > 0) {
    TORCH_CHECK(slots > 0, "packed_attention: joins without slots");
    const unsigned rows = (unsigned)(a.P * tiles * group);
    packed_combine_kernel<<<dim3((unsigned)joins.size(0), (unsigned)a.heads, (rows + 7) / 8), 256, 0, stream>>>(
        joins.data_ptr<int>(), group, a.P, (int)tiles, s.Hq, s.D, a.part_o, a.part_l, a.out, a.lse, a.low);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {out, lse, low};
}

}  // namespace osp
