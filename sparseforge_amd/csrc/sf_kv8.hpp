// The 8-bit cache of keys and values: layout and the shapes its kernels share.
//
// A block is 64 consecutive positions of one sequence and one head; blocks are whole or, for the last one of a
// sequence, incomplete.  A whole block is int8 codes with one f32 scale each for keys and values, value = code *
// scale; the incomplete one is bf16, as the rows came.  Dp is the head dimension rounded up to 64, zeros past it.
//   codes  [B, H, blocks][64 Dp]      scales  [B, H, blocks]      tail  [B, H][64 Dp] bf16
// In a block, keys lie as [Dp / 64][key][64 dims] and values as [dim][4][16]: entry (g, e) of a dim is key
// 16 (e / 4) + 4 g + e % 4.  With v_mfma_f32_16x16x32_bf16 and the score tile transposed (keys as rows), a lane of
// group g = lane / 16 then holds the scores of keys 16 t + 4 g + 0..3 of its query, which are the entries of its
// 16 bytes of values: a wave's 16-byte loads, 1 KB in a row each, are the operands of both products once converted,
// and no score moves between lanes.
#pragma once

#include "sf_mfma.hpp"

namespace sf {
namespace {

constexpr int kKvBlock = 64;   // positions that share a scale
constexpr int kKvMaxD = 256;   // head dimension bound

__host__ __device__ __forceinline__ int64_t kv_pad(int64_t D) { return (D + 63) / 64 * 64; }

// Element of a block where dim d of key j lies.
__device__ __forceinline__ int kv_key_at(int j, int d) { return ((d >> 6) * kKvBlock + j) * 64 + (d & 63); }
__device__ __forceinline__ int kv_value_at(int j, int d) {
  return d * 64 + ((j >> 2) & 3) * 16 + (j >> 4) * 4 + (j & 3);
}

}  // namespace

struct KvCache {
  int8_t* k;  // codes
  int8_t* v;
  float* ks;  // scales
  float* vs;
  uint16_t* kt;  // tails
  uint16_t* vt;
  int32_t* starts;  // [B]: tokens held before the newest
  int32_t* ends;    // [B]: and with them
  int64_t blocks;   // capacity of a sequence in blocks
  int B, H, D, Dp;
};

namespace {

// The newest tokens of a sequence, [start, end), kept inside the capacity whatever the counters hold.
__device__ __forceinline__ void kv_range(const KvCache& c, int b, int n, int& start, int& end) {
  const int cap = static_cast<int>(c.blocks * kKvBlock);
  start = c.starts[b];
  end = c.ends[b];
  start = start < 0 ? 0 : start > cap ? cap : start;
  end = end < start ? start : end > cap ? cap : end;
  if (end - start > n) end = start + n;
}

}  // namespace

// The kernels' form of a cache after its checks (sf_kv8.hip).
int kv8_cache(const sf_kv8_cache* d, const char* what, KvCache& c);

}  // namespace sf
