// Pieces shared by the kernels that look for the top of a row (sf_top_logits.hip, sf_sample.hip).  One workgroup works on
// one row.  Its elements are taken in tiles of 8 * BLK, thread t holding elements [8 t, 8 t + 8) of a tile, so that
// tiles, waves and lanes follow each other in the order of the ids.
#pragma once

#include "sf_common.hpp"

namespace sf {
namespace {

typedef unsigned long long u64;

// A row's order as integers: larger logits have larger keys, -0 equals 0, NaN is largest.  bf16 needs 16 bits.
template <int DT>
__device__ __forceinline__ uint32_t top_key(float x) {
  return DT == SF_DTYPE_BF16 ? ordered_key(x) >> 16 : ordered_key(x);
}

template <int DT>
__device__ __forceinline__ void top_load8(const void* p, int64_t i, int n, float (&v)[8]) {
  if (n == 8) {
    if constexpr (DT == SF_DTYPE_BF16) {
      uint32_t w[4];
      __builtin_memcpy(w, static_cast<const uint16_t*>(p) + i, 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[2 * k] = __uint_as_float(w[k] << 16);
        v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    } else {
      __builtin_memcpy(v, static_cast<const float*>(p) + i, 32);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < n ? load_as_f32(p, i + k, DT) : 0.0f;
  }
}

// f(tile, first id, number of elements, elements) over a row.
template <int DT, int BLK, typename F>
__device__ __forceinline__ void top_scan(const void* row, int64_t base, int vocab, F&& f) {
  int tile = 0;
  for (int i = threadIdx.x * 8; i < vocab; i += BLK * 8, ++tile) {
    const int n = vocab - i < 8 ? vocab - i : 8;
    float v[8];
    top_load8<DT>(row, base + i, n, v);
    f(tile, i, n, v);
  }
}

template <int BLK>
__device__ __forceinline__ float block_max_f(float x, float (&part)[BLK / 64]) {
  for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  x = part[0];
  for (int w = 1; w < BLK / 64; ++w) x = fmaxf(x, part[w]);
  return x;
}

// The lowest element that is taken: everything with a larger key, and the first `keep` by id of those with this key.
struct Border {
  uint32_t key;
  u64 keep;   // elements (or, by weight, what is missing of the target above the key)
  u64 above;  // weight of the larger keys
};

// Finds in a row the key at which the count, or the weight, of the elements from the largest down reaches target
// (1 .. total): passes of 8 bits from the top, each over the elements whose higher bits are the border's.
template <int DT, int BLK, typename W>
__device__ Border radix_border(const void* row, int64_t base, int vocab, bool by_weight, u64 target, W&& weight,
                               u64 (&mass)[256], uint32_t (&count)[256], u64 (&shared)[3]) {
  constexpr int kBits = DT == SF_DTYPE_BF16 ? 16 : 32;
  uint32_t prefix = 0;
  u64 above = 0;
  for (int shift = kBits - 8; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += BLK) mass[i] = 0, count[i] = 0;
    __syncthreads();
    top_scan<DT, BLK>(row, base, vocab, [&](int, int, int n, const float (&v)[8]) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t key = top_key<DT>(v[k]);
        if (k < n && (static_cast<u64>(key) >> (shift + 8)) == prefix) {
          atomicAdd(&count[key >> shift & 255], 1u);
          atomicAdd(&mass[key >> shift & 255], weight(v[k]));
        }
      }
    });
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 left = target, over = above;
      int b = 255;
      for (; b > 0; --b) {
        const u64 here = by_weight ? mass[b] : count[b];
        if (here >= left) break;
        left -= here;
        over += mass[b];
      }
      shared[0] = b;
      shared[1] = left;
      shared[2] = over;
    }
    __syncthreads();
    prefix = prefix << 8 | static_cast<uint32_t>(shared[0]);
    target = shared[1];
    above = shared[2];
    __syncthreads();
  }
  return {prefix, target, above};
}

struct Place {
  int id;     // -1: none
  u64 total;  // weight of the row
};

// The first id at which the weight of the ids up to it exceeds at(total weight).
template <int DT, int BLK, int TILES, typename W, typename A>
__device__ Place locate(const void* row, int64_t base, int vocab, W&& weight, A&& at, u64 (&sums)[TILES * (BLK / 64)],
                        u64 (&shared)[3]) {
  constexpr int kWaves = BLK / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tiles = (vocab + BLK * 8 - 1) / (BLK * 8);
  for (int tile = 0; tile < tiles; ++tile) {
    const int i = tile * BLK * 8 + threadIdx.x * 8, n = vocab - i < 8 ? vocab - i : 8;
    u64 s = 0;
    if (n > 0) {
      float v[8];
      top_load8<DT>(row, base + i, n, v);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < n) s += weight(v[k], i + k);
    }
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if (lane == 0) sums[tile * kWaves + wave] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    u64 total = 0;
    for (int j = 0; j < tiles * kWaves; ++j) total += sums[j];
    u64 left = at(total);
    int j = 0;
    for (; j < tiles * kWaves && sums[j] <= left; ++j) left -= sums[j];
    shared[0] = j;
    shared[1] = left;
    shared[2] = total;
  }
  __syncthreads();
  const int j = static_cast<int>(shared[0]);
  const u64 left = shared[1], total = shared[2];
  __syncthreads();
  if (j >= tiles * kWaves) return {-1, total};
  if (wave == 0) {
    const int i = (j / kWaves) * BLK * 8 + (j % kWaves) * 512 + lane * 8, n = vocab - i < 8 ? vocab - i : 8;
    float v[8];
    u64 w[8], s = 0;
    if (n > 0) top_load8<DT>(row, base + i, n, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      w[k] = k < n ? weight(v[k], i + k) : 0;
      s += w[k];
    }
    u64 upto = s;
    for (int off = 1; off < 64; off <<= 1) {
      const u64 x = __shfl_up(upto, off, 64);
      if (lane >= off) upto += x;
    }
    u64 before = upto - s;
    if (before <= left && left < upto)
      for (int k = 0; k < 8; ++k) {
        if (before <= left && left < before + w[k]) shared[0] = i + k;
        before += w[k];
      }
  }
  __syncthreads();
  const int id = static_cast<int>(shared[0]);
  __syncthreads();
  return {id, total};
}

}  // namespace
}  // namespace sf
