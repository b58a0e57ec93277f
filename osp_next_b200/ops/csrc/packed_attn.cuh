// What the packed attention kernels share: work items, tile geometry and tail rows.
//
// Sequences of different lengths lie one behind another (or at any distance) in q [Nq, Hq, D] and
// k, v [Nk, Hkv, D]; G = Hq / Hkv query heads share a key head.  A tile of the tensor core's 128
// rows holds the G heads of P = 128 / G positions, row = position * G + head, which one TMA box
// {64 elements, G heads, P positions} lays out that way.  So a key tile is read once for its whole
// group, a sequence of few queries fills a tile with G times as many rows, and the gradients of a
// shared key head are sums over the rows of one accumulator: no atomics.  128 - G * P rows (2 for
// G = 3, 6, 7, 9; 3 for G = 5) stay unused.
//
// The host lays the work out once per pack: a list of items for each kernel, longest first, so that
// a grid of one CTA per item and key head ends with the short ones.
//
// Tiles that reach over a sequence's end hold rows of the next one.  Scores there are masked, but
// 0 * NaN is NaN in a product that sums over those rows, so the producer warp overwrites the rows
// behind the end with zeros in shared memory before it hands the tile on.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"
#include "attn_math.cuh"

namespace osp {
namespace pa {

constexpr int kRows = 128;           // rows of a tile: group heads x positions, or keys
constexpr float kLog2e = 1.4426950408889634f;

// One work item = 8 ints.
struct FwdItem {       // forward (two tiles of P positions) and dQ (one tile)
  int q_row;           // row of the first query
  int n_q;             // queries of the item
  int limit;           // keys that its first query sees if causal (may be negative)
  int k_row;           // row of the sequence's first key
  int n_keys;          // keys of the sequence
  int kt0, kt1;        // key tiles of the item
  int slot;            // place of its partial result, or -1
};
struct KeyItem {       // dK, dV of one tile of 128 keys
  int k_row;           // row of its first key
  int n_k;             // its keys
  int first;           // first query (of the sequence) that sees its first key
  int q_row;           // row of the query `first`
  int n_q;             // queries from there on
  int lead;            // key 0 is seen by query max(0, lead) of those, key i by query lead + i
  int slot;            // place of its partial result, or -1
  int n_keys;          // keys of the sequence
};

__device__ __forceinline__ const int4* item_ptr(const int* list, int i) {
  return reinterpret_cast<const int4*>(list) + 2 * i;
}
__device__ __forceinline__ FwdItem load_fwd_item(const int* list, int i) {
  const int4 a = item_ptr(list, i)[0], b = item_ptr(list, i)[1];
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}
__device__ __forceinline__ KeyItem load_key_item(const int* list, int i) {
  const int4 a = item_ptr(list, i)[0], b = item_ptr(list, i)[1];
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

// What rounding o to bf16 left, times 2^8, in e5m2: kept for the gradient alone.  delta = rowsum(dO o O)
// takes it in; from the rounded o, dS of short rows is off by as much as by its own rounding (dQ
// 2.6e-3 from 64 bits, 2.4e-3 with it).
constexpr float kLowScale = 256.0f;
__device__ __forceinline__ uint32_t low_pair(float a, float b) {
  const float2 r = make_float2((a - bf16_round(a)) * kLowScale, (b - bf16_round(b)) * kLowScale);
  return __nv_cvt_float2_to_fp8x2(r, __NV_SATFINITE, __NV_E5M2);
}
__device__ __forceinline__ uint32_t low_bits4(const float* v, float mul) {
  return low_pair(v[0] * mul, v[1] * mul) | low_pair(v[2] * mul, v[3] * mul) << 16;
}
__device__ __forceinline__ uint2 low_bits8(const uint32_t* v, float mul) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v[i]);
  return make_uint2(low_bits4(f, mul), low_bits4(f + 4, mul));
}
__device__ __forceinline__ float low_value(uint32_t byte) {       // e5m2 is the top byte of a half
  return __half2float(__ushort_as_half((unsigned short)(byte << 8))) * (1.0f / kLowScale);
}

// Item and head of this CTA.  Items are sorted longest first; `at_once` heads are run together, the next
// ones behind them, so that the CTAs that run at a time share keys in L2.
__device__ __forceinline__ void unit_of(int units, int heads, int at_once, int& item, int& head) {
  const int u = blockIdx.x, n = units / heads;
  const int group = u / (n * at_once), in = u - group * n * at_once;
  const int wide = min(at_once, heads - group * at_once);
  item = in / wide;
  head = group * at_once + in - item * wide;
}

// Zeros into rows [row0, 128) of `boxes` boxes of 128 rows x 128 bytes, by one warp.  Whole rows, so
// the swizzle inside a row does not matter.  The caller fences towards the async proxy.
__device__ __forceinline__ void zero_rows(uint8_t* tile, int boxes, int row0, int lane) {
  const int n = (kRows - row0) * 8;                // 16-byte pieces per box
  for (int b = 0; b < boxes; ++b) {
    uint4* p = reinterpret_cast<uint4*>(tile + b * kRows * 128 + row0 * 128);
    for (int i = lane; i < n; i += 32) p[i] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// 8 fp32 values of a row, scaled, as 16 bytes of bf16.
__device__ __forceinline__ uint4 pack8(const uint32_t* v, float mul) {
  uint4 w;
  w.x = pack_bf16x2(__uint_as_float(v[0]) * mul, __uint_as_float(v[1]) * mul);
  w.y = pack_bf16x2(__uint_as_float(v[2]) * mul, __uint_as_float(v[3]) * mul);
  w.z = pack_bf16x2(__uint_as_float(v[4]) * mul, __uint_as_float(v[5]) * mul);
  w.w = pack_bf16x2(__uint_as_float(v[6]) * mul, __uint_as_float(v[7]) * mul);
  return w;
}

// 16 bytes of a warp's 32 rows x kPiece bytes in shared memory, swizzled by the row: eight rows' pieces
// lie in different banks, and so do the pieces of a row.
template <int kPiece>
__device__ __forceinline__ uint4* out_piece(uint8_t* buf, int row, int piece) {
  const int x = kPiece == 128 ? row & 7 : (row >> 1) & 3;
  return reinterpret_cast<uint4*>(buf + row * kPiece + ((piece ^ x) << 4));
}

// kCols (32 or 64) columns of a warp's 32 rows of tensor memory, scaled, to bf16 rows in global memory:
// through `buf` (4 KB of the warp's own), so that 4 or 8 lanes write a row's piece.  `at`: place of this
// lane's row and first column in `base`, or -1; `have`: the accumulator was written (else zeros).
template <int kCols>
__device__ __forceinline__ void store_rows(uint8_t* buf, uint32_t taddr, bool have, float mul, __nv_bfloat16* base,
                                           long at, int valid, int lane) {
  constexpr int kLanes = kCols / 8;
#pragma unroll
  for (int h = 0; h < kCols / 32; ++h) {
    uint32_t o[32];
    if (have) {
      tmem_ld32(taddr + h * 32, o);
      tmem_ld_wait();
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) *out_piece<kCols * 2>(buf, lane, h * 4 + i) = pack8(o + 8 * i, mul);
  }
  __syncwarp();
  const int piece = lane % kLanes;
#pragma unroll
  for (int i = 0; i < kLanes; ++i) {
    const int rr = i * (32 / kLanes) + lane / kLanes;
    const long to = __shfl_sync(0xffffffffu, at, rr);
    if (to >= 0 && piece * 8 < valid)
      *reinterpret_cast<uint4*>(base + to + piece * 8) = *out_piece<kCols * 2>(buf, rr, piece);
  }
  __syncwarp();
}
// The same in fp32 (parts of a sum), 32 columns at a time.
template <int kCols>
__device__ __forceinline__ void store_rows32(uint8_t* buf, uint32_t taddr, float mul, float* base, long at, int valid,
                                             int lane) {
#pragma unroll
  for (int h = 0; h < kCols / 32; ++h) {
    uint32_t o[32];
    tmem_ld32(taddr + h * 32, o);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<float4*>(out_piece<128>(buf, lane, i)) =
          make_float4(__uint_as_float(o[4 * i]) * mul, __uint_as_float(o[4 * i + 1]) * mul,
                      __uint_as_float(o[4 * i + 2]) * mul, __uint_as_float(o[4 * i + 3]) * mul);
    __syncwarp();
    const int piece = lane % 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int rr = i * 4 + lane / 8;
      const long to = __shfl_sync(0xffffffffu, at, rr);
      if (to >= 0 && h * 32 + piece * 4 < valid)
        *reinterpret_cast<uint4*>(base + to + h * 32 + piece * 4) = *out_piece<128>(buf, rr, piece);
    }
    __syncwarp();
  }
}

}  // namespace pa
}  // namespace osp
