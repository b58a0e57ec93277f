// Attention forward over packed sequences: causal or not, grouped heads, head dims to 128, queries
// that are the last tokens of their keys, a bias by relative position (tcgen05 + TMEM + TMA).
//
//   S = scale q k^T + bias;  o = softmax(S) v over the keys that a query sees;  lse = log sum exp S
//
// A CTA computes two row tiles (packed_attn.cuh) that pass over the same key tiles, as the kernel in
// attention_fwd.cuh does: warps 0-3 and 4-7 the softmax of tile 0 and 1 (a thread per row, running
// maximum and sum in fp32, O rescaled only when the maximum grows by more than 2^8), warp 8 the
// TMA loads, warp 9 the MMAs; P goes to bf16 in tensor memory, over S.  Under a causal mask tile 0
// needs up to one key tile less than tile 1 and leaves the rest out.  A row's keys are those below
// a limit, so the mask costs one comparison per score, in tiles that hold such a limit only.
//
// Items with many keys and few rows are split along the keys: each part leaves its normalised fp32
// output and log-sum-exp in a workspace and packed_combine_kernel joins them.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include "attention_fwd.cuh"
#include "packed_attn.cuh"
#include "packed_attn_host.h"

namespace osp {

struct PackedFwdArgs {
  const int* items;
  int G, P, Hq, Hkv, Dr;    // heads per key head, positions per tile, query and key heads, head dim
  int causal;
  __nv_bfloat16* out;       // [Nq, Hq, Dr]
  float* lse;               // [Nq, Hq] or null
  float scale_log2;
  const float* bias;        // [Hq, 2 M - 1] or null
  int bias_m;               // M
  float* part_o;            // [slots, Hkv, 2 * 128, Dr]
  float* part_l;            // [slots, Hkv, 2 * 128], log2 domain
  int* err;
};

template <int D>
struct PackedFwdCfg {
  static constexpr int kProdWarp = 8, kMmaWarp = 9, kThreads = 320;
  static constexpr int BOX = pa::kRows * 128;
  static constexpr int DB = D / 64;
  static constexpr int TILE = DB * BOX;
  static constexpr int kSlots = 5;
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_BAR = OFF_KV + kSlots * TILE;
  static constexpr int USED = OFF_BAR + 256;
  static constexpr int kMaxSmem = 232448;
  static constexpr int SLACK = (kMaxSmem - USED) < 1008 ? (kMaxSmem - USED) : 1008;
  static constexpr int BYTES = USED + SLACK;
};

// S values of a row (raw) -> scaled scores in the log2 domain with the bias added.
template <bool kFull>
__device__ __forceinline__ void add_bias(uint32_t* sr, float sl2, const float* brow, int n_valid) {
#pragma unroll
  for (int c = 0; c < pa::kRows; ++c) {
    const float b = (kFull || c < n_valid) ? __ldg(brow + c) : 0.f;
    sr[c] = __float_as_uint(fmaf(__uint_as_float(sr[c]), sl2, b * pa::kLog2e));
  }
}

template <int D, bool kBias>
__global__ void __launch_bounds__(PackedFwdCfg<D>::kThreads, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, PackedFwdArgs args) {
  using L = PackedFwdCfg<D>;
  constexpr int kT = pa::kRows, kSlots = L::kSlots;
  const pa::FwdItem it = pa::load_fwd_item(args.items, blockIdx.x / args.Hkv);
  const int kvh = blockIdx.x % args.Hkv;
  const int G = args.G, P = args.P;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  if (pad > (uint32_t)L::SLACK) {                              // CTA-uniform: report, do nothing
    if (threadIdx.x == 0) record_error(args.err, kErrAttnLayout);
    return;
  }
  uint8_t* smem = smem_raw + pad;
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + L::OFF_KV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_full = bars + 0;
  uint64_t* tail = bars + 1;                       // the V tile that reaches over the sequence's end
  uint64_t* kv_full = bars + 2;                    // [kSlots]
  uint64_t* kv_empty = kv_full + kSlots;           // [kSlots]
  uint64_t* s_full = kv_empty + kSlots;            // [2]
  uint64_t* p_half = s_full + 2;                   // [2]
  uint64_t* p_full = p_half + 2;                   // [2]
  uint64_t* o_done = p_full + 2;                   // [2]
  uint64_t* done = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(done + 2);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;

  // key tiles of each row tile: those below the limit of its last query
  int n_t[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int nq = min(P, it.n_q - t * P);
    const int lim = args.causal ? min(it.n_keys, it.limit + t * P + nq - 1) : it.n_keys;
    n_t[t] = nq > 0 ? max(0, min(it.kt1, (max(lim, 0) + kT - 1) / kT) - it.kt0) : 0;
  }
  const int n0 = n_t[0], n1 = n_t[1], n_kv = max(n0, n1);
  const int last_rows = it.n_keys - (it.kt0 + n_kv - 1) * kT;  // keys of the last tile
  const bool has_tail = n_kv > 0 && last_rows < kT;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(tail, 1);
    for (int i = 0; i < kSlots; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_half[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == L::kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == L::kProdWarp) {
    // ------------------------------------------------------------------ producer
    const int krow0 = it.k_row + it.kt0 * kT;
    auto load_kv = [&](int u, uint64_t* bar) {
      const int slot = u % kSlots;
      mbar_expect_tx(bar, L::TILE);
      const CUtensorMap* tm = (u & 1) ? &tmV : &tmK;
      for (int db = 0; db < L::DB; ++db)
        tma_load_3d(tm, bar, sKV + slot * L::TILE + db * L::BOX, db * 64, kvh, krow0 + (u >> 1) * kT);
    };
    const int units = 2 * n_kv;
    const int plain = has_tail ? units - 1 : units;
    bool ok = true;
    if (lane == 0 && n_kv > 0) {
      const int tiles = (n0 > 0) + (n1 > 0);
      mbar_expect_tx(q_full, tiles * L::DB * G * P * 128);
      for (int t = 0; t < 2; ++t)
        for (int db = 0; db < L::DB && n_t[t] > 0; ++db)
          tma_load_3d(&tmQ, q_full, sQ + t * L::TILE + db * L::BOX, db * 64, kvh * G, it.q_row + t * P);
      for (int u = 0; u < units && !*abort_flag; ++u) {
        if (!(ok = mbar_wait(&kv_empty[u % kSlots], ((u / kSlots) & 1) ^ 1, args.err, kErrAttnProducer))) break;
        load_kv(u, u < plain ? &kv_full[u % kSlots] : tail);
      }
    }
    __syncwarp();
    if (has_tail) {
      ok = __shfl_sync(0xffffffffu, ok && !*abort_flag, 0);
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(tail, 0, args.err, kErrAttnProducer));
      if (ok) {
        const int slot = (units - 1) % kSlots;
        pa::zero_rows(sKV + slot * L::TILE, L::DB, last_rows, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[slot]);
      }
    }
    if (!ok) *abort_flag = 1;
  } else if (warp == L::kMmaWarp) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0 && n_kv > 0) {
      constexpr uint32_t ID_S = idesc_bf16(128, kT);
      constexpr uint32_t ID_PV = idesc_bf16(128, D, /*b_mn_major=*/true);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, args.err, kErrAttnMma); };
      auto issue_s = [&](int t, int slot) {
        const uint32_t qa = smem_u32(sQ + t * L::TILE);
        const uint32_t ka = smem_u32(sKV + slot * L::TILE);
        const uint32_t d = tmem + 128u * t;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k / 4) * L::BOX + (k % 4) * 32;
          umma_bf16(d, sdesc_sw128(qa + off, 16, 1024), sdesc_sw128(ka + off, 16, 1024), ID_S, k > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[t]);
      };
      auto issue_pv = [&](int t, int slot, int k0, int k1, bool acc) {
        const uint32_t va = smem_u32(sKV + slot * L::TILE);
        const uint32_t d = tmem + 256u + (uint32_t)D * t;
        const uint32_t pr = tmem + 128u * t;
#pragma unroll
        for (int k = k0; k < k1; ++k)
          umma_bf16_ts(d, pr + 8u * k, sdesc_sw128(va + k * 2048, L::BOX, 1024), ID_PV, (acc || k > 0) ? 1u : 0u);
      };
      auto pv = [&](int t, int j, int slot) -> bool {
        if (!wait(&p_half[t], j & 1)) return false;
        tc_fence_after();
        issue_pv(t, slot, 0, kT / 32, j > 0);
        if (!wait(&p_full[t], j & 1)) return false;
        tc_fence_after();
        issue_pv(t, slot, kT / 32, kT / 16, j > 0);
        return true;
      };
      bool ok = wait(q_full, 0) && wait(&kv_full[0], 0);
      if (ok) {
        tc_fence_after();
        if (n0 > 0) issue_s(0, 0);
        if (n1 > 0) issue_s(1, 0);
        umma_commit(&kv_empty[0]);
      }
      for (int j = 0; j < n_kv && ok; ++j) {
        const int uV = 2 * j + 1, uK = 2 * j + 2;
        const int sV = uV % kSlots, sK = uK % kSlots;
        if (!(ok = wait(&kv_full[sV], (uV / kSlots) & 1))) break;
        tc_fence_after();
        if (j < n0) {
          if (!(ok = pv(0, j, sV))) break;
          if (j + 1 == n0) umma_commit(&o_done[0]);
        }
        if (j + 1 < n_kv && !(ok = wait(&kv_full[sK], (uK / kSlots) & 1))) break;
        tc_fence_after();
        if (j + 1 < n0) issue_s(0, sK);
        if (j < n1) {
          if (!(ok = pv(1, j, sV))) break;
          if (j + 1 == n1) umma_commit(&o_done[1]);
        }
        umma_commit(&kv_empty[sV]);
        if (j + 1 < n1) issue_s(1, sK);
        if (j + 1 < n_kv) umma_commit(&kv_empty[sK]);
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
    const uint32_t tO = tmem + 256u + (uint32_t)D * t + lane_off;
    const int nq = min(P, it.n_q - t * P);            // queries of the tile (<= 0: it has none)
    const int pos = min(r / G, max(nq, 1) - 1);       // rows behind the last query repeat its mask
    const int head = kvh * G + r % G;
    const bool in = r < G * P && r / G < nq;
    const int limit = args.causal ? min(it.n_keys, it.limit + t * P + pos) : it.n_keys;
    const float sl2 = args.scale_log2;
    const float* brow = nullptr;
    if (kBias)                                        // entry of key 0 for this query
      brow = args.bias + (long)(in ? head : kvh * G) * (2 * args.bias_m - 1) + args.bias_m -
             (it.limit + t * P + pos);
    float m_ref = -INFINITY, l = 0.f;
    bool ok = true;
    const int n = t == 0 ? n0 : n1;
    for (int j = 0; j < n; ++j) {
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], j & 1, args.err, kErrAttnSoftmax)))) break;
      tc_fence_after();
      const int key0 = (it.kt0 + j) * kT;
      const int n_valid = limit - key0;
      const bool full = __all_sync(0xffffffffu, n_valid >= kT);
      uint32_t sr[kT];
#pragma unroll
      for (int c = 0; c < kT / 32; ++c) tmem_ld32(tS + c * 32, sr + c * 32);
      tmem_ld_wait();
      if (kBias) {
        if (full) add_bias<true>(sr, sl2, brow + key0, kT);
        else add_bias<false>(sr, sl2, brow + key0, n_valid);
      }
      const float mul = kBias ? 1.0f : sl2;
      float mx = full ? attn_row_max<kT, true>(sr, kT) : attn_row_max<kT, false>(sr, n_valid);
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
      if (full) l += attn_exp_store<64, true, 0u, 0>(sr, mul, m_ref, 64, tS);
      else l += attn_exp_store<64, false, 0u, 0>(sr, mul, m_ref, n_valid, tS);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_half[t]);
      if (full) l += attn_exp_store<64, true, 0u, 4>(sr + 64, mul, m_ref, 64, tS + 32);
      else l += attn_exp_store<64, false, 0u, 4>(sr + 64, mul, m_ref, n_valid - 64, tS + 32);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], 0, args.err, kErrAttnSoftmax));
    if (!ok) *abort_flag = 1;
    tc_fence_after();
    const bool write = ok && in;
    const float inv_l = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);   // no key seen: 0; NaN stays
    const float lse2 = m_ref + __log2f(l);
    const long row = (long)(it.q_row + t * P + r / G) * args.Hq + head;
    const long prow = it.slot < 0 ? 0 : ((long)it.slot * args.Hkv + kvh) * (2 * kT) + t * kT + r;
    if (nq > 0) {
#pragma unroll 1
      for (int c = 0; c < args.Dr; c += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(tO + c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (!write) continue;
        if (it.slot < 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + 8 * i < args.Dr)
              *reinterpret_cast<uint4*>(args.out + row * args.Dr + c + 8 * i) = pa::pack8(o + 8 * i, inv_l);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + 4 * i < args.Dr)
              *reinterpret_cast<float4*>(args.part_o + prow * args.Dr + c + 4 * i) =
                  make_float4(__uint_as_float(o[4 * i]) * inv_l, __uint_as_float(o[4 * i + 1]) * inv_l,
                              __uint_as_float(o[4 * i + 2]) * inv_l, __uint_as_float(o[4 * i + 3]) * inv_l);
        }
      }
      if (write) {
        if (it.slot >= 0) args.part_l[prow] = lse2;
        else if (args.lse) args.lse[row] = lse2 * 0.69314718055994531f;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == L::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// o = sum_i 2^(l_i - l) o_i over the parts of one item, 2^l = sum_i 2^(l_i).  A warp per row.
__global__ void packed_combine_kernel(const int* joins, int G, int P, int Hq, int Dr, const float* part_o,
                                      const float* part_l, __nv_bfloat16* out, float* lse) {
  const int4 j = reinterpret_cast<const int4*>(joins)[blockIdx.x];   // q_row, n_q, first slot, parts
  const int kvh = blockIdx.y, lane = threadIdx.x % 32;
  for (int i = threadIdx.x / 32; i < j.y * G; i += blockDim.x / 32) {
    const int p = i / G, g = i % G;
    const int t = p / P;
    const long r = t * pa::kRows + (p - t * P) * G + g;
    const long stride = (long)gridDim.y * 2 * pa::kRows;
    const long first = (long)j.z * stride + (long)kvh * 2 * pa::kRows + r;
    float top = -INFINITY;
    for (int s = 0; s < j.w; ++s) {
      const float v = part_l[first + s * stride];
      top = v != v ? v : fmaxf(top, v);
    }
    float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    const float base = top == -INFINITY ? 0.f : top;
    for (int s = 0; s < j.w; ++s) {
      const float w = exp2f(part_l[first + s * stride] - base);
      sum += w;
      if (lane * 4 < Dr && w != 0.f) {
        const float4 v = *reinterpret_cast<const float4*>(part_o + (first + s * stride) * Dr + lane * 4);
        acc[0] += w * v.x; acc[1] += w * v.y; acc[2] += w * v.z; acc[3] += w * v.w;
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    const long row = (long)(j.x + p) * Hq + kvh * G + g;
    if (lane * 4 < Dr) {
      uint2 w;
      w.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
      w.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<uint2*>(out + row * Dr + lane * 4) = w;
    }
    if (lane == 0 && lse) lse[row] = (base + log2f(sum)) * 0.69314718055994531f;
  }
}

template <int D, bool kBias>
static void launch_packed_fwd(dim3 grid, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                              const PackedFwdArgs& a, cudaStream_t stream) {
  auto kern = packed_fwd_kernel<D, kBias>;
  smem_opt_in(reinterpret_cast<const void*>(kern), PackedFwdCfg<D>::BYTES);
  kern<<<grid, PackedFwdCfg<D>::kThreads, PackedFwdCfg<D>::BYTES, stream>>>(tq, tk, tv, a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// (o [Nq, Hq, D] bf16, lse [Nq, Hq] fp32 or empty).  `items` / `joins` are int32 lists on the device,
// laid out by ops.SequencePack for this group size; rows of no sequence are zeros (`fill`).
std::vector<at::Tensor> packed_attn_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                        const at::Tensor& items, const at::Tensor& joins, int64_t slots, bool causal,
                                        double scale, const c10::optional<at::Tensor>& rel_bias, bool want_lse,
                                        bool fill) {
  const pa::Shape s = pa::check_shapes(q, k, v, "packed_attention");
  pa::check_list(items, 8, q, "packed_attention: items");
  pa::check_list(joins, 4, q, "packed_attention: joins");
  c10::cuda::CUDAGuard guard(q.device());
  auto opt = q.options();
  at::Tensor out = fill ? at::zeros({s.Nq, s.Hq, s.D}, opt) : at::empty({s.Nq, s.Hq, s.D}, opt);
  at::Tensor lse;
  if (want_lse) {
    lse = at::empty({s.Nq, s.Hq}, opt.dtype(at::kFloat));
    if (fill) lse.fill_(-INFINITY);
  }
  const int64_t n = items.size(0);
  if (n == 0 || s.Hq == 0 || s.D == 0) return {out, lse};
  PackedFwdArgs a{};
  a.items = items.data_ptr<int>();
  a.G = s.G;
  a.P = pa::kRows / s.G;
  a.Hq = s.Hq;
  a.Hkv = s.Hkv;
  a.Dr = s.D;
  a.causal = causal ? 1 : 0;
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  if (rel_bias.has_value()) {
    TORCH_CHECK(rel_bias->is_cuda() && rel_bias->device() == q.device() && rel_bias->scalar_type() == at::kFloat &&
                rel_bias->is_contiguous() && rel_bias->dim() == 2 && rel_bias->size(0) == s.Hq &&
                rel_bias->size(1) % 2 == 1, "packed_attention: rel_bias fp32 [heads, 2 M - 1]");
    a.bias = rel_bias->data_ptr<float>();
    a.bias_m = (int)((rel_bias->size(1) + 1) / 2);
  }
  a.err = error_word(q.get_device());
  at::Tensor part_o, part_l;
  if (slots > 0) {
    part_o = at::empty({slots, s.Hkv, 2 * pa::kRows, s.D}, opt.dtype(at::kFloat));
    part_l = at::empty({slots, s.Hkv, 2 * pa::kRows}, opt.dtype(at::kFloat));
    a.part_o = part_o.data_ptr<float>();
    a.part_l = part_l.data_ptr<float>();
  }
  const CUtensorMap tq = pa::tile_map(q, q, s.D, s.G, a.P);
  const CUtensorMap tk = pa::tile_map(k, q, s.D, 1, pa::kRows), tv = pa::tile_map(v, q, s.D, 1, pa::kRows);
  dim3 grid((unsigned)(n * s.Hkv));
  auto stream = c10::cuda::getCurrentCUDAStream();
  if (s.D > 64) {
    if (a.bias) launch_packed_fwd<128, true>(grid, tq, tk, tv, a, stream);
    else launch_packed_fwd<128, false>(grid, tq, tk, tv, a, stream);
  } else {
    if (a.bias) launch_packed_fwd<64, true>(grid, tq, tk, tv, a, stream);
    else launch_packed_fwd<64, false>(grid, tq, tk, tv, a, stream);
  }
  if (joins.size(0) > 0) {
    TORCH_CHECK(slots > 0, "packed_attention: joins without slots");
    packed_combine_kernel<<<dim3((unsigned)joins.size(0), (unsigned)s.Hkv), 256, 0, stream>>>(
        joins.data_ptr<int>(), s.G, a.P, s.Hq, s.D, a.part_o, a.part_l, a.out, a.lse);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {out, lse};
}

}  // namespace osp
