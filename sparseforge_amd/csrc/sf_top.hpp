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
// piece p of a wave, lane l has 8 ids.  What lies behind the row is -inf.
template <int DT, int BLK>
struct RowAt {
  const void* row;
  int vocab, pieces;

  __device__ __forceinline__ RowAt(const void* row_, int vocab_)
      : row(row_), vocab(vocab_), pieces((vocab_ + BLK * 8 - 1) / (BLK * 8)) {}
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
};

// One that stays: the first H pieces in registers, the others are read again by every pass over the row.
template <int DT, int BLK, int H>
struct Row : RowAt<DT, BLK> {
  using Base = RowAt<DT, BLK>;
  using Base::at;
  using Base::fetch;
  using Base::pieces;
  using Base::row;
  using Base::vocab;
  using Base::wave_at;
  Raw8<DT> raw[H];

  __device__ __forceinline__ Row(const void* row_, int vocab_) : Base(row_, vocab_) {
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
    constexpr int kAhead = 4;  // pieces on their way
    Raw8<DT> more[kAhead];
    for (int q = H; q < pieces; q += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (q + u < pieces) fetch(more[u], at(q + u));
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (q + u < pieces) {
          more[u].get(v);
          f(q + u, at(q + u), v);
        }
    }
  }
  // The same as a loop, for an f of a hundred instructions and more, of which H copies would not stay in the instruction
  // cache: the first piece is taken and the others move up before it, which restores their order in the end.
  template <typename F>
  __device__ __forceinline__ void each_looped(F&& f) {
    float v[8];
#pragma unroll 1
    for (int p = 0; p < H; ++p) {
      const Raw8<DT> first = raw[0];
#pragma unroll
      for (int q = 0; q + 1 < H; ++q) raw[q] = raw[q + 1];
      raw[H - 1] = first;
      if (p < pieces) {
        first.get(v);
        f(p, at(p), v);
      }
    }
    if (pieces <= H) return;
    Raw8<DT> next[2];
    fetch(next[0], at(H));
    fetch(next[1], at(H + 1));
#pragma unroll 1
    for (int p = H; p < pieces; ++p) {
      next[0].get(v);
      next[0] = next[1];
      fetch(next[1], at(p + 2));  // behind the last piece another wave's, or nothing: not used
      f(p, at(p), v);
    }
  }
};

constexpr float kTopLow = -3.402823466e38f;  // start of a running maximum: finite, so that -inf minus it is not NaN

// The larger of two, NaN if either is (v_maximum3_f32 takes two of these).
__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float max8(const float (&v)[8]) {
  return nan_max(nan_max(nan_max(v[0], v[1]), nan_max(v[2], v[3])), nan_max(nan_max(v[4], v[5]), nan_max(v[6], v[7])));
}

// x of the lane that a DPP control names, `none` in lanes that it gives nothing.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t x, uint32_t none) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(static_cast<int>(none), static_cast<int>(x), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ u64 dpp(u64 x, u64 none) {
  return static_cast<u64>(dpp<CTRL, ROWS>(static_cast<uint32_t>(x >> 32), static_cast<uint32_t>(none >> 32))) << 32 |
         dpp<CTRL, ROWS>(static_cast<uint32_t>(x), static_cast<uint32_t>(none));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float x, float none) {
  return __uint_as_float(dpp<CTRL, ROWS>(__float_as_uint(x), __float_as_uint(none)));
}
// op over a wave's lanes up to each one, by shifts within rows of 16 lanes and the rows' last lanes; every lane of the
// wave has to be there.
template <typename T, typename F>
__device__ __forceinline__ T wave_scan(T x, T none, F&& op) {
  x = op(x, dpp<0x111>(x, none));
  x = op(x, dpp<0x112>(x, none));
  x = op(x, dpp<0x114>(x, none));
  x = op(x, dpp<0x118>(x, none));
  x = op(x, dpp<0x142, 0xa>(x, none));
  return op(x, dpp<0x143, 0xc>(x, none));
}
template <typename T>
__device__ __forceinline__ T wave_scan(T x) {
  return wave_scan(x, T(0), [](T a, T b) { return a + b; });
}
// The last lane's, in every one.
__device__ __forceinline__ uint32_t last_lane(uint32_t x) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), 63));
}
__device__ __forceinline__ float last_lane(float x) { return __uint_as_float(last_lane(__float_as_uint(x))); }
__device__ __forceinline__ u64 last_lane(u64 x) {
  return static_cast<u64>(last_lane(static_cast<uint32_t>(x >> 32))) << 32 | last_lane(static_cast<uint32_t>(x));
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
// The float of an ordered_key.
__device__ __forceinline__ float key_float(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ float candidate_logit(u64 c) { return key_float(static_cast<uint32_t>(c >> 32)); }

constexpr int kTopBins = 1024;

// CAP: candidates that there is room for.
template <int CAP>
struct TopShared {
  uint32_t bins[kTopBins];
  u64 found[CAP], mixed[CAP];
  uint32_t start[kTopBins + 1];
  uint32_t part[16];
  float edge[2][16];
  uint32_t limit;
  int n;
};

// A bound above which at least k elements of a row lie, and few others: those with half(x) * scale < limit, half(x) being
// half of m - x: the whole is more than a float where logits lie at both ends of the type.  Its place
// comes from the maxima of the threads' groups of the row: the k-th largest of these is one, and a histogram over [the
// lowest, the highest] finds its bin.  With at least 2 k groups about 1.4 k elements lie above it, with hardly more than k
// nearly all, and a row of less than 8 k logits has fewer: then the bound takes everything above -inf.  Where many groups share
// that bin (some logits lie far from all others: a mask of -1e4 or of the type's lowest value, say) the histogram is made
// again over what the bin holds: 512 rows of 131072 bf16, of which such a mask leaves one in 15, k 20: 39 us, 502 by the
// bits of every logit, 37 without the mask.
struct Bound {
  float m, scale, limit;
  float low;  // the lowest group of those above the bound, about
  __device__ __forceinline__ bool holds(float x) const { return half_below(0.5f * m, x) * scale < limit; }
  static __device__ __forceinline__ float half_below(float half_m, float x) { return fmaf(-0.5f, x, half_m); }
};

// best: the thread's groups' maxima (no NaN, not inf), m: the row's.  Where fewer than k groups have anything above -inf
// the bound takes everything above it.  sh.n is 0 afterwards.
template <int BLK, int GROUPS, int CAP>
__device__ __forceinline__ Bound top_bound(const float (&best)[GROUPS], float m, int k, TopShared<CAP>& sh) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  constexpr int kEach = kTopBins / BLK;
  const auto least = [](float a, float b) { return fminf(a, b); };
  const auto most = [](float a, float b) { return fmaxf(a, b); };
  float low = INFINITY, top = m;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) low = fminf(low, best[g] == -INFINITY ? INFINITY : best[g]);
  low = last_lane(wave_scan(low, INFINITY, least));
  if (lane == 0) sh.edge[0][wave] = low;
  uint32_t above = 0;
#pragma unroll 1
  for (int again = 3;; --again) {  // differences below 1e-30 are not told apart, however often
    for (int i = t; i < kTopBins; i += BLK) sh.bins[i] = 0;
    if (t == 0) sh.limit = ~0u, sh.n = 0;
    __syncthreads();
    for (int w = 0; w < BLK / 64; ++w) low = fminf(low, sh.edge[0][w]);
    const float half_top = 0.5f * top, scale = fminf((kTopBins - 1) / Bound::half_below(half_top, low), 2e30f);
    const auto bin_of = [&](float x) SF_INLINE {
      return static_cast<int>(fminf(Bound::half_below(half_top, x) * scale, static_cast<float>(kTopBins - 1)));
    };
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      if (best[g] >= low && best[g] <= top) atomicAdd(&sh.bins[bin_of(best[g])], 1u);
    __syncthreads();
    uint32_t own[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += own[i] = sh.bins[t * kEach + i];
    uint32_t upto = above + block_scan<BLK>(sum, sh.part) - sum;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (upto < static_cast<uint32_t>(k) && upto + own[i] >= static_cast<uint32_t>(k))
        sh.limit = t * kEach + i, sh.start[0] = own[i], sh.start[1] = upto;
      upto += own[i];
    }
    __syncthreads();
    const uint32_t limit = sh.limit;
    if (limit == ~0u) return {m, 1.0f, INFINITY, low};
    if (again == 0 || static_cast<int>(sh.start[0]) <= 16 + k / 4)
      return {top, scale, static_cast<float>(limit + 1), fmaxf(low, top - 2.0f * (static_cast<float>(limit + 1) / scale))};
    above = sh.start[1];
    float first = -INFINITY, last = INFINITY;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      if (best[g] >= low && best[g] <= top && bin_of(best[g]) == static_cast<int>(limit)) {
        first = fmaxf(first, best[g]);
        last = fminf(last, best[g]);
      }
    first = last_lane(wave_scan(first, -INFINITY, most));
    last = last_lane(wave_scan(last, INFINITY, least));
    if (lane == 0) sh.edge[0][wave] = last, sh.edge[1][wave] = first;
    __syncthreads();
    low = INFINITY, top = -INFINITY;
    for (int w = 0; w < BLK / 64; ++w) low = fminf(low, sh.edge[0][w]), top = fmaxf(top, sh.edge[1][w]);
    if (low == top) return {top, 2e30f, 1.0f, low};  // equal ones, and what is larger
  }
}

// Gathers into sh.found the elements within the bound of the thread's pieces p for which bit p % G of hits is set, and
// returns how many there are in all (sh.n has to be 0 before); more than CAP: too many (equal ones, most likely), and not
// all are there.  A thread has few such pieces and takes them from the caches.
template <int G, int DT, int BLK, int CAP>
__device__ __forceinline__ int gather(const RowAt<DT, BLK>& row, const Bound& bound, uint32_t hits, TopShared<CAP>& sh) {
  while (hits) {
#pragma unroll 1
    for (int p = __ffs(hits) - 1; p < row.pieces; p += G) {
      const int i = row.at(p);
      Raw8<DT> raw;
      float v[8];
      row.fetch(raw, i);
      raw.get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (bound.holds(v[j])) {
          const int at = atomicAdd(&sh.n, 1);
          if (at < CAP) sh.found[at] = candidate(v[j], i + j);
        }
    }
    hits &= hits - 1;
  }
  __syncthreads();
  return sh.n;
}

// Orders a[0 .. n) in LDS, falling; behind it up to the next power of two there has to be room.
template <int BLK>
__device__ __forceinline__ void sort_all(u64* a, int n) {
  const int t = threadIdx.x;
  int size = 2;
  while (size < n) size *= 2;
  for (int i = n + t; i < size; i += BLK) a[i] = 0;
  __syncthreads();
#pragma unroll 1
  for (int run = 2; run <= size; run *= 2)
#pragma unroll 1
    for (int step = run / 2; step > 0; step /= 2) {
      for (int i = t; i < size / 2; i += BLK) {
        const int at = 2 * i - (i & (step - 1));
        const u64 x = a[at], y = a[at + step];
        if ((x < y) == ((at & run) == 0)) a[at] = y, a[at + step] = x;
      }
      __syncthreads();
    }
}

// Orders sh.found[0 .. n), elements within the bound (m: the row's largest): counted into bins between the two, then placed
// among those of their bin; where more than 256 share one, by comparisons alone (1024 x 32000 bf16 with k 500: 39 us, 49
// with comparisons wherever 32 share one; logits rounded to halves 92, 437 without).
template <int BLK, int CAP>
__device__ __forceinline__ void sort_found(const Bound& bound, float m, int n, TopShared<CAP>& sh) {
  constexpr int kEach = kTopBins / BLK, kCrowd = 256;
  const int t = threadIdx.x;
  const float scale = fminf((kTopBins - 1) / (m - bound.low), 1e30f);
  const auto bin_of = [&](u64 c) SF_INLINE {
    return static_cast<int>(fminf((m - candidate_logit(c)) * scale, static_cast<float>(kTopBins - 1)));
  };
  for (int i = t; i < kTopBins; i += BLK) sh.bins[i] = 0;
  if (t == 0) sh.limit = 0;
  __syncthreads();
  for (int i = t; i < n; i += BLK) atomicAdd(&sh.bins[bin_of(sh.found[i])], 1u);
  __syncthreads();
  uint32_t own[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    sum += own[i] = sh.bins[t * kEach + i];
    if (own[i] > kCrowd) sh.limit = 1;
  }
  uint32_t at = block_scan<BLK>(sum, sh.part) - sum;
  if (sh.limit) {
    sort_all<BLK>(sh.found, n);
    return;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    sh.bins[t * kEach + i] = sh.start[t * kEach + i] = at;
    at += own[i];
  }
  if (t == 0) sh.start[kTopBins] = n;
  __syncthreads();
  for (int i = t; i < n; i += BLK) {
    const u64 c = sh.found[i];
    sh.mixed[atomicAdd(&sh.bins[bin_of(c)], 1u)] = c;
  }
  __syncthreads();
  for (int i = t; i < n; i += BLK) {
    const u64 c = sh.mixed[i];
    const int bin = bin_of(c), from = sh.start[bin], to = sh.start[bin + 1];
    int rank = from;
#pragma unroll 4
    for (int j = from; j < to; ++j) rank += sh.mixed[j] > c ? 1 : 0;
    sh.found[rank] = c;
  }
  __syncthreads();
}

// The largest of the threads' m, NaN if one is, in every thread.
template <int BLK>
__device__ __forceinline__ float row_max(float m, float* part) {
  m = last_lane(wave_scan(m, -INFINITY, [](float a, float b) { return nan_max(a, b); }));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  m = part[0];
  for (int w = 1; w < BLK / 64; ++w) m = nan_max(m, part[w]);
  return m;
}

// Reads a row once: the maxima of the thread's G groups of pieces (piece p is in group p % G), and also(elements) for every
// piece, four pieces on their way at a time.
template <int G, int DT, int BLK, typename F>
__device__ __forceinline__ void read_row(const RowAt<DT, BLK>& row, float (&best)[G], F&& also) {
#pragma unroll
  for (int g = 0; g < G; ++g) best[g] = -INFINITY;
#pragma unroll 1
  for (int q = 0; q < row.pieces; q += G)
#pragma unroll
    for (int g = 0; g < G; g += 4)
      if (q + g < row.pieces) {
        Raw8<DT> raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (row.at(q + g + u) + 8 <= row.vocab && q + g + u < row.pieces)
            raw[u].load(row.row, row.at(q + g + u));
          else
            raw[u].empty();
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float v[8];
          raw[u].get(v);
          best[g + u] = nan_max(best[g + u], max8(v));
          also(v);
        }
      }
  if (row.vocab % 8 != 0) {  // one thread has a piece that the row ends in
    const int i = row.vocab / 8 * 8 - row.wave_at(threadIdx.x >> 6);
    if (i >= 0 && i < row.pieces * 512 && i % 512 / 8 == static_cast<int>(threadIdx.x & 63)) {
      Raw8<DT> raw;
      float v[8];
      raw.load_some(row.row, row.vocab / 8 * 8, row.vocab % 8);
      raw.get(v);
      const float x = max8(v);
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (i / 512 % G == g) best[g] = nan_max(best[g], x);
      also(v);
    }
  }
}
// The bound for k elements from the groups' maxima of read_row, taken together to two a thread.
template <int BLK, int G, int CAP>
__device__ __forceinline__ Bound bound_of(const float (&best)[G], float m, int k, TopShared<CAP>& sh) {
  float two[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int g = 0; g < G; ++g) two[g & 1] = fmaxf(two[g & 1], best[g]);
  return top_bound<BLK>(two, m, k, sh);
}
template <int G>
__device__ __forceinline__ uint32_t hits_of(const float (&best)[G], const Bound& bound) {
  uint32_t hits = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) hits |= bound.holds(best[g]) ? 1u << g : 0u;
  return hits;
}

// ---------------------------------------------------------------------------
// Passes that are right for every row, whatever its order and its equal values, for the rows in which gather() finds too
// many (512 rows of 131072 equal bf16 logits: k 20 250 us, k 50 drawn 290, top-p 0.9 drawn 550; rows that have more than CAP
// logits and not much more than 8 k: 256 x 8192 bf16, k 1000, 38 us, 15 with k 600).  Thread t takes elements
// [8 t, 8 t + 8) of tiles of 8 * BLK, so that tiles, waves and lanes follow each other in the order of the ids.
// ---------------------------------------------------------------------------
// A row's order as integers: larger logits have larger keys, -0 equals 0, NaN is largest.  bf16 needs 16 bits.
template <int DT>
__device__ __forceinline__ uint32_t top_key(float x) {
  return DT == SF_DTYPE_BF16 ? ordered_key(x) >> 16 : ordered_key(x);
}

// f(first id, how many, elements) over a thread's elements, the next 8 on their way.
template <int DT, int BLK, typename F>
__device__ __forceinline__ void each_any(const void* row, int vocab, F&& f) {
  const auto fetch = [&](Raw8<DT>& to, int i) SF_INLINE {
    if (i + 8 <= vocab)
      to.load(row, i);
    else
      to.load_some(row, i, vocab - i);
  };
  Raw8<DT> next;
  fetch(next, threadIdx.x * 8);
#pragma unroll 1
  for (int i = threadIdx.x * 8; i < vocab; i += BLK * 8) {
    float v[8];
    next.get(v);
    fetch(next, i + BLK * 8);
    f(i, vocab - i < 8 ? vocab - i : 8, v);
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
// (1 .. total): passes of 8 bits from the top, each over the elements whose higher bits are the border's.  Afterwards
// sh.mass and sh.count hold the border's own key's at its last 8 bits.
template <int DT, int BLK, typename W>
__device__ __forceinline__ Border radix_border(const void* row, int vocab, bool by_weight, u64 target, W&& weight,
                                               AnyShared& sh) {
  constexpr int kBits = DT == SF_DTYPE_BF16 ? 16 : 32;
  uint32_t prefix = 0;
  u64 above = 0;
#pragma unroll 1
  for (int shift = kBits - 8; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += BLK) sh.mass[i] = 0, sh.count[i] = 0;
    if (threadIdx.x == 0) sh.shared[0] = 0, sh.shared[1] = target, sh.shared[2] = above;
    __syncthreads();
    // elements with the same bits in a row are added as one
    each_any<DT, BLK>(row, vocab, [&](int, int n, const float (&v)[8]) SF_INLINE {
      uint32_t at = 0, count = 0;
      u64 mass = 0;
      const auto add = [&]() SF_INLINE {
        if (count == 0) return;
        atomicAdd(&sh.count[at], count);
        if (mass) atomicAdd(&sh.mass[at], mass);
      };
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t key = top_key<DT>(v[k]);
        if (k < n && (static_cast<u64>(key) >> (shift + 8)) == prefix) {
          if ((key >> shift & 255) != at) {
            add();
            at = key >> shift & 255;
            count = 0;
            mass = 0;
          }
          ++count;
          mass += weight(v[k]);
        }
      }
      add();
    });
    __syncthreads();
    if (threadIdx.x < 64) {  // from the largest down, four to a lane
      u64 here[4], own = 0, mass = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int b = 255 - threadIdx.x * 4 - i;
        own += here[i] = by_weight ? sh.mass[b] : sh.count[b];
        mass += sh.mass[b];
      }
      u64 upto = wave_scan(own) - own, over = above + wave_scan(mass) - mass;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int b = 255 - threadIdx.x * 4 - i;
        if (upto < target && target <= upto + here[i]) {
          sh.shared[0] = b;
          sh.shared[1] = target - upto;
          sh.shared[2] = over;
        }
        upto += here[i];
        over += sh.mass[b];
      }
    }
    __syncthreads();
    prefix = prefix << 8 | static_cast<uint32_t>(sh.shared[0]);
    target = sh.shared[1];
    above = sh.shared[2];
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
  constexpr int kWaves = BLK / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tiles = (vocab + BLK * 8 - 1) / (BLK * 8);
  const auto sum_of = [&](int i, int n, const float (&v)[8]) SF_INLINE {
    u64 s = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += k < n ? weight(v[k], i + k) : 0;
    return s;
  };
  for (int j = threadIdx.x; j < tiles * kWaves; j += BLK) sh.sums[j] = 0;
  if (threadIdx.x == 0) sh.shared[0] = tiles * kWaves, sh.shared[1] = 0;
  __syncthreads();
  each_any<DT, BLK>(row, vocab, [&](int i, int n, const float (&v)[8]) SF_INLINE {
    const u64 s = sum_of(i, n, v);
    if (s) atomicAdd(&sh.sums[i / 512], s);  // a wave's tile is 512 elements
  });
  __syncthreads();
  // the tile in which the sum passes what at() says, by one wave
  if (wave == 0) {
    const int each = (tiles * kWaves + 63) / 64, from = lane * each;
    u64 own = 0;
    for (int j = from; j < from + each && j < tiles * kWaves; ++j) own += sh.sums[j];
    const u64 upto = wave_scan(own), total = last_lane(upto), target = at(total);
    if (lane == 0) sh.shared[2] = total;
    if (upto - own <= target && target < upto) {
      u64 left = target - (upto - own);
      int j = from;
      for (; sh.sums[j] <= left; ++j) left -= sh.sums[j];
      sh.shared[0] = j;
      sh.shared[1] = left;
    }
  }
  __syncthreads();
  const int j = static_cast<int>(sh.shared[0]);
  const u64 left = sh.shared[1], total = sh.shared[2];
  __syncthreads();
  if (j >= tiles * kWaves) return {-1, total};
  if (wave == 0) {
    const int i = j * 512 + lane * 8;
    Raw8<DT> raw;
    float v[8];
    if (i + 8 <= vocab)
      raw.load(row, i);
    else
      raw.load_some(row, i, vocab - i);
    raw.get(v);
    const u64 s = sum_of(i, vocab - i < 8 ? vocab - i : 8, v), upto = wave_scan(s);
    u64 before = upto - s;
    if (before <= left && left < upto) {
#pragma unroll 1
      for (int k = i; k < i + 8 && k < vocab; ++k) {
        const u64 w = weight(load_as_f32(row, k, DT), k);
        if (before <= left && left < before + w) sh.shared[0] = k;
        before += w;
      }
    }
  }
  __syncthreads();
  const int id = static_cast<int>(sh.shared[0]);
  __syncthreads();
  return {id, total};
}

}  // namespace
}  // namespace sf
