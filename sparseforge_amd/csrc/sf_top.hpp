// Pieces shared by the kernels that look for the top of a row (sf_top_logits.hip, sf_sample.hip, sf_top_kl.hip).
#pragma once

#include "sf_common.hpp"

namespace sf {
namespace {

typedef unsigned long long u64;

// For the bodies of passes over a row: one that is called from many places may not be left as a function of its own, which
// would take the elements through memory.
#define SF_INLINE __attribute__((always_inline))

// 8 elements from any element's address, as they are stored.
template <int DT>
struct Raw8 {
  uint32_t w[DT == SF_DTYPE_BF16 ? 4 : 8];
  __device__ __forceinline__ void load(const void* row, int i) {
    __builtin_memcpy(w, static_cast<const char*>(row) + static_cast<int64_t>(i) * (DT == SF_DTYPE_BF16 ? 2 : 4),
                     sizeof(w));
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (DT == SF_DTYPE_BF16)
        v[k] = __uint_as_float(k & 1 ? w[k / 2] & 0xffff0000u : w[k / 2] << 16);
      else
        v[k] = __uint_as_float(w[k]);
    }
  }
  __device__ __forceinline__ void empty() {
#pragma unroll
    for (uint32_t& x : w) x = DT == SF_DTYPE_BF16 ? 0xff80ff80u : 0xff800000u;
  }
  // n of 8 elements, -inf behind them
  __device__ __forceinline__ void load_some(const void* row, int i, int n) {
    empty();
    for (int k = 0; k < n; ++k) {
      const uint32_t x = DT == SF_DTYPE_BF16 ? static_cast<const uint16_t*>(row)[i + k]
                                             : static_cast<const uint32_t*>(row)[i + k];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j == k) {
          if constexpr (DT == SF_DTYPE_BF16)
            w[j / 2] = j & 1 ? (w[j / 2] & 0xffffu) | x << 16 : (w[j / 2] & 0xffff0000u) | x;
          else
            w[j] = x;
        }
    }
  }
};

// A row in front of a workgroup of BLK threads.  Each wave has a range of the ids of its own, `pieces` times 512 long; of
// piece p of a wave (at most 32), lane l holds 8 ids.  The first H pieces stay in registers, the others are read again by every pass
// over the row.  What lies behind the row is -inf.
template <int DT, int BLK, int H>
struct Row {
  const void* row;
  int vocab, pieces;
  Raw8<DT> raw[H];

  __device__ __forceinline__ int wave_at(int wave) const { return wave * pieces * 512; }
  __device__ __forceinline__ int at(int p) const {
    return wave_at(threadIdx.x >> 6) + p * 512 + (threadIdx.x & 63) * 8;
  }
  __device__ __forceinline__ void fetch(Raw8<DT>& to, int i) const {
    const int n = vocab - i;
    if (n >= 8)
      to.load(row, i);
    else
      to.load_some(row, i, n);
  }
  __device__ __forceinline__ Row(const void* row_, int vocab_) : row(row_), vocab(vocab_) {
    pieces = (vocab + BLK * 8 - 1) / (BLK * 8);
#pragma unroll
    for (int p = 0; p < H; ++p)
      if (p < pieces) {
        if (at(p) + 8 <= vocab)
          raw[p].load(row, at(p));
        else
          raw[p].empty();
      }
    if (vocab % 8 != 0) {  // one thread has a piece that the row ends in
      const int in_wave = vocab / 8 * 8 - wave_at(threadIdx.x >> 6), last = in_wave / 512;
      if (in_wave >= 0 && in_wave < pieces * 512 && (in_wave % 512) / 8 == static_cast<int>(threadIdx.x & 63)) {
        Raw8<DT> some;
        some.load_some(row, vocab / 8 * 8, vocab % 8);
#pragma unroll
        for (int p = 0; p < H; ++p)
          if (p == last) raw[p] = some;
      }
    }
  }
  // f(piece, first id, elements)
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    float v[8];
#pragma unroll
    for (int p = 0; p < H; ++p)
      if (p < pieces) {
        raw[p].get(v);
        f(p, at(p), v);
      }
    for (int p = H; p < pieces; ++p) {
      Raw8<DT> more;
      fetch(more, at(p));
      more.get(v);
      f(p, at(p), v);
    }
  }
};

// The larger of two, NaN if either is (v_maximum3_f32 takes two of these).
__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float max8(const float (&v)[8]) {
  return nan_max(nan_max(nan_max(v[0], v[1]), nan_max(v[2], v[3])), nan_max(nan_max(v[4], v[5]), nan_max(v[6], v[7])));
}

// Inclusive sum over a wave's lanes.
template <typename T>
__device__ __forceinline__ T wave_scan(T x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T y = __shfl_up(x, off, 64);
    if (static_cast<int>(threadIdx.x & 63) >= off) x += y;
  }
  return x;
}
// Inclusive sum over a workgroup's threads.  part: of BLK / 64, not in use before or after without a barrier.
template <int BLK, typename T>
__device__ __forceinline__ T block_scan(T x, T* part) {
  x = wave_scan(x);
  if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = x;
  __syncthreads();
  T before = 0;
  for (int w = 0; w < BLK / 64; ++w)
    if (w < static_cast<int>(threadIdx.x >> 6)) before += part[w];
  return x + before;
}

// A candidate for the top of a row: larger ones come first, of equal logits the lower id.  -0 equals 0.
__device__ __forceinline__ u64 candidate(float x, int id) {
  return static_cast<u64>(ordered_key(x)) << 32 | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ int candidate_id(u64 c) { return static_cast<int>(~static_cast<uint32_t>(c)); }
__device__ __forceinline__ float candidate_logit(u64 c) {
  const uint32_t key = static_cast<uint32_t>(c >> 32);
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

constexpr int kTopBins = 1024;
constexpr int kTopCandidates = 2048;

struct TopShared {
  uint32_t bins[kTopBins];
  u64 found[kTopCandidates];
  uint32_t part[16];
  float edge[2][16];
  uint32_t limit;
  int n;
};

// A bound above which at least k elements of a row lie, and few others: those with (m - x) * scale < limit.  Its place
// comes from the maxima of the threads' groups of the row: the k-th largest of these is one, and a histogram over [the
// lowest, the highest] finds it.  With at least 2 k groups about 1.4 k elements lie above it.
struct Bound {
  float m, scale, limit;
  __device__ __forceinline__ bool holds(float x) const { return (m - x) * scale < limit; }
};

// best: the thread's groups' maxima (no NaN, not inf), m: the row's.  Where fewer than k groups have anything above -inf
// the bound takes everything above it.  sh.n is 0 afterwards.
template <int BLK, int GROUPS>
__device__ __forceinline__ Bound top_bound(const float (&best)[GROUPS], float m, int k, TopShared& sh) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  constexpr int kEach = kTopBins / BLK;
  float low = INFINITY;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) low = fminf(low, best[g] == -INFINITY ? INFINITY : best[g]);
  for (int off = 32; off > 0; off >>= 1) low = fminf(low, __shfl_xor(low, off, 64));
  if (lane == 0) sh.edge[0][wave] = low;
  for (int i = t; i < kTopBins; i += BLK) sh.bins[i] = 0;
  if (t == 0) sh.limit = ~0u, sh.n = 0;
  __syncthreads();
  for (int w = 0; w < BLK / 64; ++w) low = fminf(low, sh.edge[0][w]);
  // logits at both ends of the type: a difference of inf has no place
  const float scale = m - low < INFINITY ? fminf((kTopBins - 1) / (m - low), 1e30f) : 0.0f;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g)
    if (best[g] != -INFINITY) {
      const int bin = static_cast<int>((m - best[g]) * scale);
      atomicAdd(&sh.bins[bin >= 0 && bin < kTopBins ? bin : kTopBins - 1], 1u);
    }
  __syncthreads();
  uint32_t own[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += own[i] = sh.bins[t * kEach + i];
  uint32_t upto = block_scan<BLK>(sum, sh.part) - sum;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (upto < static_cast<uint32_t>(k) && upto + own[i] >= static_cast<uint32_t>(k)) sh.limit = t * kEach + i;
    upto += own[i];
  }
  __syncthreads();
  if (scale == 0.0f) return {INFINITY, 1.0f, 0.0f};  // nothing: the caller has to look at the row in another way
  return {m, scale, sh.limit == ~0u ? INFINITY : static_cast<float>(sh.limit + 1)};
}

// Gathers into sh.found the elements that wanted(x) holds for, of the thread's pieces whose bit is set in hits, and returns
// how many there are in all (sh.n has to be 0 before); more than kTopCandidates: too many (equal ones, most likely), and not all are there.  The pieces
// come from the caches: eight tests for each piece in registers are more code than the instruction cache holds.
template <int DT, int BLK, int H, typename F>
__device__ __forceinline__ int gather(const Row<DT, BLK, H>& row, F&& wanted, uint32_t hits, TopShared& sh) {
  while (hits) {
    const int i = row.at(__ffs(hits) - 1);
    hits &= hits - 1;
    Raw8<DT> raw;
    float v[8];
    row.fetch(raw, i);
    raw.get(v);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (wanted(v[j])) {
        const int at = atomicAdd(&sh.n, 1);
        if (at < kTopCandidates) sh.found[at] = candidate(v[j], i + j);
      }
  }
  __syncthreads();
  const int n = sh.n;
  if (threadIdx.x == 0 && n < kTopCandidates && n % 2) sh.found[n] = 0;  // rank_of reads two at a time
  __syncthreads();
  return n;
}

// Maxima of the thread's groups of pieces; the row's, NaN if it has one, in every thread.
template <int DT, int BLK, int H, int GROUPS>
__device__ __forceinline__ float row_max(const Row<DT, BLK, H>& row, float (&best)[GROUPS], float* part) {
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) best[g] = -INFINITY;
  row.each([&](int p, int, const float (&v)[8]) SF_INLINE {
    const float x = max8(v);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      if (GROUPS == 1 || p % GROUPS == g) best[g] = nan_max(best[g], x);
  });
  float m = best[0];
#pragma unroll
  for (int g = 1; g < GROUPS; ++g) m = nan_max(m, best[g]);
  for (int off = 32; off > 0; off >>= 1) m = nan_max(m, __shfl_xor(m, off, 64));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  m = part[0];
  for (int w = 1; w < BLK / 64; ++w) m = nan_max(m, part[w]);
  return m;
}

// How many of the n candidates come before c; where n is odd found[n] is 0.
__device__ __forceinline__ int rank_of(u64 c, const u64* found, int n) {
  int rank = 0;
  for (int j = 0; j < n; j += 2) {
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(found + j);
    rank += (x.x > c ? 1 : 0) + (x.y > c ? 1 : 0);
  }
  return rank;
}

// ---------------------------------------------------------------------------
// Passes that are right for every row, whatever its order and its equal values: a row's elements in tiles of 8 * BLK,
// thread t holding elements [8 t, 8 t + 8) of a tile, so that tiles, waves and lanes follow each other in the order of
// the ids.  Used where gather_top finds too many.
// ---------------------------------------------------------------------------
// A row's order as integers: larger logits have larger keys, -0 equals 0, NaN is largest.  bf16 needs 16 bits.
template <int DT>
__device__ __forceinline__ uint32_t top_key(float x) {
  return DT == SF_DTYPE_BF16 ? ordered_key(x) >> 16 : ordered_key(x);
}

template <int DT>
__device__ __forceinline__ void top_load8(const void* row, int i, int n, float (&v)[8]) {
  Raw8<DT> raw;
  if (n == 8)
    raw.load(row, i);
  else
    raw.load_some(row, i, n);
  raw.get(v);
}

// f(tile, first id, number of elements, elements) over a row.
template <int DT, int BLK, typename F>
__device__ __forceinline__ void top_scan(const void* row, int vocab, F&& f) {
  int tile = 0;
  for (int i = threadIdx.x * 8; i < vocab; i += BLK * 8, ++tile) {
    const int n = vocab - i < 8 ? vocab - i : 8;
    float v[8];
    top_load8<DT>(row, i, n, v);
    f(tile, i, n, v);
  }
}

constexpr int kAnySums = SF_TOP_MAX_VOCAB / 512;  // a sum for each wave and tile
struct AnyShared {
  u64 mass[256];
  uint32_t count[256];
  u64 sums[kAnySums];
  u64 shared[3];
};

// The lowest element that is taken: everything with a larger key, and the first `keep` by id of those with this key.
struct Border {
  uint32_t key;
  u64 keep;   // elements (or, by weight, what is missing of the target above the key)
  u64 above;  // weight of the larger keys
};

// Finds in a row the key at which the count, or the weight, of the elements from the largest down reaches target
// (1 .. total): passes of 8 bits from the top, each over the elements whose higher bits are the border's.
template <int DT, int BLK, typename W>
__device__ __forceinline__ Border radix_border(const void* row, int vocab, bool by_weight, u64 target, W&& weight, AnyShared& sh) {
  u64(&mass)[256] = sh.mass, (&shared)[3] = sh.shared;
  uint32_t(&count)[256] = sh.count;
  constexpr int kBits = DT == SF_DTYPE_BF16 ? 16 : 32;
  uint32_t prefix = 0;
  u64 above = 0;
  for (int shift = kBits - 8; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += BLK) mass[i] = 0, count[i] = 0;
    __syncthreads();
    top_scan<DT, BLK>(row, vocab, [&](int, int, int n, const float (&v)[8]) {
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
template <int DT, int BLK, typename W, typename A>
__device__ __forceinline__ Place locate(const void* row, int vocab, W&& weight, A&& at, AnyShared& sh) {
  u64(&sums)[kAnySums] = sh.sums, (&shared)[3] = sh.shared;
  constexpr int kWaves = BLK / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tiles = (vocab + BLK * 8 - 1) / (BLK * 8);
  for (int tile = 0; tile < tiles; ++tile) {
    const int i = tile * BLK * 8 + threadIdx.x * 8, n = vocab - i < 8 ? vocab - i : 8;
    u64 s = 0;
    if (n > 0) {
      float v[8];
      top_load8<DT>(row, i, n, v);
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
    if (n > 0) top_load8<DT>(row, i, n, v);
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
