// A token for every row from given random numbers.  For a row x with maximum m, at temperature T, the tokens ordered by
// falling logit (equal ones by rising id):
//   w_i = exp((x_i - m) / T)
//   top-k keeps the first k; top-p of these the fewest first tokens that hold p of their weight; min-p those of at least
//   min_p times the largest weight.  All three keep a first part of that order.
//   the token is the first, by id, at which the weight of the kept tokens up to it exceeds u times their whole weight.
// Weights are formed in f64 and summed as integers of 2^-F, F = 44 (43 above 65536 tokens, 42 above 131072), so that no
// sum depends on its order.  A cumulative share is off by 2e-12 (the exponential's polynomial) at most, which decides one
// draw in 4e6 from 131072 equal tokens; shares from f32 exponentials, off by 1e-7, would decide one in a hundred.
//
// One workgroup per row.  With top-k up to 1024 the row is read once, for the maxima of its pieces; the pieces above the
// bound that follows from these are taken again, their largest gathered in LDS, and the rest happens among them.  Without
// it, top-p's border is the place in a histogram of weights by logit where their sum reaches p, resolved among the tokens
// of that bin, which are gathered while the weight above the bin is summed; the draw finds the wave's part of the row,
// then the thread's.
//
// Few rows are bound by their chain of passes and barriers (4 x 32000 bf16, k 50: 9.8 us; 48 x 50257 f32 with settings of
// their own: 17), many without top-k by the vector unit, which forms a weight in 23 instructions for 64 elements: 1024 x
// 32000 bf16 without limits 41 us (vector unit 0.72 busy), 256 x 131072 f32 with top-p 104 us (three passes, 0.60
// busy, half of the cycles of LDS lost to bins that collide).  1024 x 32000 bf16 with k 100: 28 us, 2.3 TB/s, as the rows of a
// CU read together and then stand in the same chain together.  With top-k above 1024 and the k-th logit more than 31 T below
// the largest its border lies in the last bin, beside thousands, and the row is looked through by its bits: 256 x 32000 bf16,
// k 2000, T 0.3 102 us, 28 with T 1.  Tried for top-p: a
// histogram with f32 exponentials that the next pass's exact sums confirm, 117 us with sums of 64 bits, 256 with the float
// additions of LDS.
#include <type_traits>

#include "sf_mfma.hpp"
#include "sf_top.hpp"

namespace sf {
namespace {

constexpr int kSpBins = 2048, kSpCandidates = 2048;

struct SampleArgs {
  const void* x;
  int64_t xs;
  int vocab;
  const float* u;
  int64_t* tokens;
  float* logprobs;
  const float* temp;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temp1, top_p1, min_p1;
  int top_k1, bits;  // bits: F
  double round;      // 1.5 * 2^52 + F
  double poly[8];    // (2^f - 1) / f, the polynomial of degree 7 through its values at the Chebyshev points
};

// A row's settings.
struct Settings {
  float top;     // the largest logit
  float temp;    // above 0
  float u;
  int64_t k;     // 1 .. vocab
  double p;      // 1: all
  double one;    // 2^F
  double least;  // the smallest weight that min-p keeps

  __device__ __forceinline__ Settings(const SampleArgs& a, int64_t r) : top(0.0f) {
    const float T = a.temp ? a.temp[r] : a.temp1, top_p = a.top_p ? a.top_p[r] : a.top_p1;
    const float min_p = a.min_p ? a.min_p[r] : a.min_p1;
    const int top_k = a.top_k ? a.top_k[r] : a.top_k1;
    const bool greedy = !(T > 0.0f);
    u = a.u[r];
    temp = greedy ? 1.0f : T;
    k = greedy ? 1 : top_k <= 0 || top_k > a.vocab ? a.vocab : top_k;
    p = !greedy && top_p < 1.0f ? static_cast<double>(top_p) : 1.0;
    one = ldexp(1.0, a.bits);
    least = (min_p > 1.0f ? 1.0 : min_p > 0.0f ? static_cast<double>(min_p) : 0.0) * one;
  }
};

// Weights exp((x - top) / T) as integers of 2^-F (F <= 44); 2^F exactly for the largest logit, which is finite.  The
// constants come from the kernel's arguments, that is in scalar registers.
struct Weight {
  double top, c;  // c: log2(e) / T
  const double& round;
  const double (&poly)[8];
  // before it is rounded
  __device__ __forceinline__ double scaled(float x) const {
    // 2^z = 2^n 2^f, f in [-1/2, 1/2]: n + F is in the low bits of the sum with 1.5 * 2^52 + F.  -inf ends at the smallest
    // z.  The last bit, 2^-8 of a unit at most, is set: nothing lies half way between integers, where a sum would round
    // another way than the weight alone.
    const double z = fmax((static_cast<double>(x) - top) * c, -64.0);
    const double rounded = z + round;
    const double f = z - (rounded - round);
    double p = poly[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) p = fma(p, f, poly[i]);
    p = fma(p, f, 1.0);
    const u64 as = static_cast<u64>(__double_as_longlong(p));
    const uint32_t n = static_cast<uint32_t>(__double_as_longlong(rounded));
    return __longlong_as_double(static_cast<u64>(static_cast<uint32_t>(as >> 32) + (n << 20)) << 32 |
                                (static_cast<uint32_t>(as) | 1u));
  }
  __device__ __forceinline__ u64 operator()(float x) const { return whole(scaled(x) + kWhole); }

  // A number added to 2^52 is rounded to an integer, which is in the sum's low bits; so are the sums of up to 2^52 / 2^bits
  // weights that start there.
  static constexpr double kWhole = 4503599627370496.0;
  static __device__ __forceinline__ u64 whole(double x) {
    return static_cast<u64>(__double_as_longlong(x)) & 0xfffffffffffffull;
  }
};

// What a share of the weight comes to, as a number of units: cumulative sums of at most `total` are compared with it.
__device__ __forceinline__ u64 share_down(float share, u64 total) {  // below total
  const double want = floor((share > 0.0f ? static_cast<double>(share) : 0.0) * static_cast<double>(total));
  return want < static_cast<double>(total) && static_cast<u64>(want) < total ? static_cast<u64>(want) : total - 1;
}
__device__ __forceinline__ u64 share_up(double share, u64 total) {  // 1 .. total
  const double want = ceil(share * static_cast<double>(total));
  return !(want >= 1.0) ? 1 : want < static_cast<double>(total) && static_cast<u64>(want) < total
                                  ? static_cast<u64>(want)
                                  : total;
}

__device__ __forceinline__ void put_token(const SampleArgs& a, const Settings& s, int64_t r, int id, float x, u64 total) {
  a.tokens[r] = id;
  if (!a.logprobs) return;
  const double d = x == s.top ? 0.0 : (static_cast<double>(x) - s.top) / static_cast<double>(s.temp);
  a.logprobs[r] = static_cast<float>(d - log(static_cast<double>(total) / s.one));
}

// A row that holds a NaN, or nothing above -inf.
__device__ __forceinline__ void put_none(const SampleArgs& a, int64_t r, float m) {
  if (threadIdx.x != 0) return;
  a.tokens[r] = -1;
  if (a.logprobs) a.logprobs[r] = m;
}

// Any row, by passes over the bits of its logits.
template <int DT, int BLK>
__device__ __forceinline__ void sample_any(const SampleArgs& a, const Settings& s, int64_t r, const void* row,
                                           const Weight& finite, AnyShared& any) {
  const int V = a.vocab;
  // below a largest logit of inf nothing has weight
  const auto weight = [&](float x) { return x == s.top ? 1ull << a.bits : finite(x); };
  Border border{0, ~0ull, 0};
  u64 z = 0;
  if (s.k < V) {
    border = radix_border<DT, BLK>(row, V, false, s.k, weight, any);
    // count and weight of the border's own key are in the last pass's bins
    z = border.above + border.keep * (any.mass[border.key & 255] / any.count[border.key & 255]);
    __syncthreads();
  } else if (s.p < 1.0) {
    z = locate<DT, BLK>(row, V, [&](float x, int) { return weight(x); }, [](u64 t) { return t; }, any).total;
  }
  if (s.p < 1.0) {
    border = radix_border<DT, BLK>(row, V, true, share_up(s.p, z), weight, any);
    const u64 each = any.mass[border.key & 255] / any.count[border.key & 255];
    border.keep = (border.keep + each - 1) / each;
    __syncthreads();
  }
  int last = V;  // the last id of those at the border that is kept
  if (border.keep != ~0ull)
    last = locate<DT, BLK>(
               row, V, [&](float x, int) { return static_cast<u64>(top_key<DT>(x) == border.key); },
               [&](u64) { return border.keep - 1; }, any)
               .id;
  const auto kept = [&](float x, int id) -> u64 {
    const uint32_t key = top_key<DT>(x);
    if (key < border.key || (key == border.key && id > last)) return 0;
    const u64 w = weight(x);
    return static_cast<double>(w) >= s.least ? w : 0;
  };
  const Place at = locate<DT, BLK>(row, V, kept, [&](u64 total) { return share_down(s.u, total); }, any);
  if (threadIdx.x == 0) put_token(a, s, r, at.id, load_as_f32(row, at.id, DT), at.total);
}

// CAP: candidates, BINS: bins of weight, or tokens that are drawn from.
template <int CAP, int BINS>
struct SampleLds {
  TopShared<CAP> top;
  u64 weight[BINS + 64];  // by place, or by bin; in the end a bin for each lane of what has no weight
  u64 before[BINS];
  u64 part[2][16];
  u64 base, last;
  int count, bin;
};
using SampleShared = SampleLds<kSpCandidates, kSpBins>;

// The draw by one wave among the row's n <= 64 largest, which sh.top.found holds in any order: top-k, top-p, min-p and the
// token.
template <typename S>
__device__ __forceinline__ void sample_few(const SampleArgs& a, const Settings& s, int64_t r, const Weight& weight, int n,
                                           S& sh) {
  const int t = threadIdx.x;
  const u64 own = t < n ? sh.top.found[t] : 0;
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j < n; ++j) rank += sh.top.found[j] > own ? 1 : 0;
  if (t < n) sh.top.mixed[rank] = own;
  wave_lds_fence();
  const int k = s.k < n ? static_cast<int>(s.k) : n;
  const u64 c = t < k ? sh.top.mixed[t] : 0;
  const float x = candidate_logit(c);
  const int id = candidate_id(c);
  const u64 w = t < k ? weight(x) : 0, upto = wave_scan(w);
  const bool kept = t < k && (s.p >= 1.0 || upto - w < share_up(s.p, last_lane(upto))) && static_cast<double>(w) >= s.least;
  const int count = __popcll(__ballot(kept));
  const u64 total = __shfl(upto, count - 1, 64), want = share_down(s.u, total);
  sh.weight[t] = w;
  wave_lds_fence();
  u64 sum = 0;
#pragma unroll 4
  for (int i = 0; i < count; ++i) sum += candidate_id(sh.top.mixed[i]) <= id ? sh.weight[i] : 0;
  if (kept && sum - w <= want && want < sum) put_token(a, s, r, id, x, total);
}

// The same by the workgroup among the n largest in order.  Ids are drawn from by ranges: the range in which the sum passes
// the drawn share, then the token among the kept ones of that range.
template <int BLK, typename S>
__device__ __forceinline__ void sample_sorted(const SampleArgs& a, const Settings& s, int64_t r, const Weight& weight,
                                              int n, S& sh) {
  const int t = threadIdx.x, k = s.k < n ? static_cast<int>(s.k) : n;  // k <= BLK
  const u64 c = t < k ? sh.top.found[t] : 0;
  const float x = candidate_logit(c);
  const int id = candidate_id(c);
  const u64 w = t < k ? weight(x) : 0;
  sh.weight[t] = 0;
  if (t == 0) sh.count = 0;
  const u64 upto = block_scan<BLK>(w, sh.part[0]);
  u64 all = 0;
  for (int i = 0; i < BLK / 64; ++i) all += sh.part[0][i];
  const bool kept = t < k && (s.p >= 1.0 || upto - w < share_up(s.p, all)) && static_cast<double>(w) >= s.least;
  const int width = (a.vocab + BLK - 1) / BLK, range = id / width;
  if (kept) atomicAdd(&sh.weight[range], w);
  __syncthreads();
  const u64 mine = sh.weight[t], end = block_scan<BLK>(mine, sh.part[1]);
  u64 total = 0;
  for (int i = 0; i < BLK / 64; ++i) total += sh.part[1][i];
  const u64 want = share_down(s.u, total);
  if (end - mine <= want && want < end) sh.bin = t, sh.base = end - mine;
  __syncthreads();
  if (kept && range == sh.bin) {
    const int at = atomicAdd(&sh.count, 1);
    sh.top.mixed[at] = c;
    sh.before[at] = w;
  }
  __syncthreads();
  if (kept && range == sh.bin) {
    u64 sum = sh.base;
    for (int i = 0; i < sh.count; ++i) sum += candidate_id(sh.top.mixed[i]) <= id ? sh.before[i] : 0;
    if (sum - w <= want && want < sum) put_token(a, s, r, id, x, total);
  }
}

template <int BLK, typename S>
__device__ __forceinline__ void sample_found(const SampleArgs& a, const Settings& s, int64_t r, const Weight& weight,
                                             const Bound& bound, int n, S& sh) {
  if (n > 64) {
    sort_found<BLK>(bound, s.top, n, sh.top);
    sample_sorted<BLK>(a, s, r, weight, n, sh);
  } else if (threadIdx.x < 64) {
    sample_few(a, s, r, weight, n, sh);
  }
}

// Every row with top-k, of at most BLK and less than CAP (or at temperature 0): the row is read once.
template <int DT, int BLK, int G, int CAP>
__global__ void __launch_bounds__(BLK) sample_top_k_kernel(SampleArgs a) {
  __shared__ union {
    SampleLds<CAP, BLK> sh;
    AnyShared any;
  } lds;
  auto& sh = lds.sh;
  const int64_t r = blockIdx.x;
  const RowAt<DT, BLK> row(static_cast<const char*>(a.x) + r * a.xs * (DT == SF_DTYPE_BF16 ? 2 : 4), a.vocab);
  Settings s(a, r);
  float best[G];
  read_row(row, best, [](const float (&)[8]) {});
  float m = best[0];
#pragma unroll
  for (int g = 1; g < G; ++g) m = nan_max(m, best[g]);
  m = s.top = row_max<BLK>(m, sh.top.edge[1]);
  if (!(m > -INFINITY)) {
    put_none(a, r, m);
    return;
  }
  const Weight weight{m, 1.4426950408889634 / static_cast<double>(s.temp), a.round, a.poly};
  int n = 0;
  if (m < INFINITY) {
    const Bound bound = bound_of<BLK>(best, m, static_cast<int>(s.k), sh.top);
    n = gather<G>(row, bound, hits_of(best, bound), sh.top);
    if (n > 0 && n <= CAP) sample_found<BLK>(a, s, r, weight, bound, n, sh);
  }
  if (n == 0 || n > CAP) {
    __syncthreads();
    sample_any<DT, BLK>(a, s, r, row.row, weight, lds.any);
  }
}

// Places of logits in a histogram from the largest down; what has no weight ends in the last bin.
struct Bins {
  float top, scale;
  __device__ __forceinline__ int of(float x) const {
    return static_cast<int>(fminf((top - x) * scale, static_cast<float>(kSpBins - 1)));
  }
  // The logits of a bin lie between these (and a few beside it).
  __device__ __forceinline__ void range(int bin, float& low, float& high) const {
    const float a = (static_cast<float>(bin) - 0.01f) / scale, b = (static_cast<float>(bin) + 1.01f) / scale;
    const float off = 1e-6f * (fabsf(top) + b);
    high = fminf(top - a + off, -kTopLow);
    low = bin == kSpBins - 1 ? kTopLow : fmaxf(top - b - off, kTopLow);
  }
};

// The last element, in the order of logits, that top-k and top-p keep.
struct Last {
  float x = -INFINITY;
  int id = INT32_MAX;
  __device__ __forceinline__ bool keeps(float y, int i) const { return (y > x) | ((y == x) & (i <= id)); }
};

// Adds the elements' weights (KIND 1), those that `last` keeps (KIND 2), or their number (KIND 0) to the bins.
template <int KIND, int DT, int BLK, int H>
__device__ __forceinline__ void fill_bins(Row<DT, BLK, H>& row, const Bins& bins, const Last& last, const Weight& weight,
                                          SampleShared& sh) {
  // what is added has no branch around it, so that several elements are on their way at a time
  const int none = kSpBins + (threadIdx.x & 63);
  row.each_looped([&](int, int i, const float (&v)[8]) SF_INLINE {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const u64 w = KIND == 0 ? 1 : weight(v[k]);
      const bool counts = KIND == 2 ? last.keeps(v[k], i + k) & (v[k] > -INFINITY) : v[k] > -INFINITY;
      atomicAdd(&sh.weight[counts ? bins.of(v[k]) : none], w);
      if (k % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // four at a time: eight take more registers than there are
    }
  });
}

// The float above x, which is not inf.
__device__ __forceinline__ float float_above(float x) { return key_float(ordered_key(x) + 1); }

// The weight of the thread's elements from `from` up (ALL: of every one), as a sum that starts at 2^52.  Those of
// [low, high], which is below, are gathered in sh.top.found.
template <bool ALL, int DT, int BLK, int H>
__device__ __forceinline__ double sum_from(Row<DT, BLK, H>& row, float from, float low, float high,
                                           const Weight& weight, SampleShared& sh) {
  double sum = Weight::kWhole;
  row.each_looped([&](int, int i, const float (&v)[8]) SF_INLINE {
    const float largest = max8(v);
    if (!ALL && largest >= low) {
      bool in[8], any = false;
#pragma unroll
      for (int k = 0; k < 8; ++k) any |= in[k] = (v[k] >= low) & (v[k] <= high);
      if (any) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (in[k]) {
            const int at = atomicAdd(&sh.top.n, 1);
            if (at < kSpCandidates) sh.top.found[at] = candidate(v[k], i + k);
          }
      }
    }
    if (ALL || largest >= from) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        sum += weight.scaled(ALL || v[k] >= from ? v[k] : -INFINITY);  // 2^-20, which the sum of integers does not see
        if (k % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
  });
  return sum;
}

// The place in the bins (see fill_bins) at which the sum of what they hold reaches want(whole sum): sh.bin and the sum
// before it in sh.base, which comes back with the target.  -1: the sum stays below.
template <int BLK, typename W>
__device__ __forceinline__ u64 bin_of_sum(W&& want, SampleShared& sh) {
  constexpr int kEach = kSpBins / BLK;
  const int t = threadIdx.x;
  u64 own[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += own[i] = sh.weight[t * kEach + i];
  u64 upto = block_scan<BLK>(sum, sh.part[0]) - sum, total = 0;
  for (int i = 0; i < BLK / 64; ++i) total += sh.part[0][i];
  const u64 target = want(total);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (upto < target && target <= upto + own[i]) sh.bin = t * kEach + i, sh.base = upto;
    upto += own[i];
  }
  __syncthreads();
  return target;
}

// Among the n gathered elements, which hold all of the bin, the last one before which the sum is below target: up to 512 by
// each one's sum over the others, more by sorting them (us for 1024 x 32000 bf16 with top-p 0.9: logits that spread 87 and
// 94; within 3 of 12, where 2000 share a bin, 518 and 174).
template <int BLK, typename M>
__device__ __forceinline__ Last last_of(const Bins& bins, int n, u64 target, M&& amount, SampleShared& sh) {
  const int t = threadIdx.x, bin = sh.bin;
  const auto own_of = [&](u64 c) -> u64 {  // nothing for those beside the bin
    const float x = candidate_logit(c);
    return bins.of(x) == bin ? amount(x, candidate_id(c)) : 0;
  };
  if (n <= 512) {
    for (int i = t; i < n; i += BLK) {
      sh.weight[i] = own_of(sh.top.found[i]);
      sh.before[i] = sh.base;
    }
    __syncthreads();
    // every candidate's sum before it, its terms shared by as many threads as there are
    const int parts = n < BLK ? BLK / n : 1, size = (n + parts - 1) / parts;
    for (int at = t; at < n * parts; at += BLK) {
      const int i = at % n, from = at / n * size, to = from + size < n ? from + size : n;
      const u64 c = sh.top.found[i];
      u64 sum = 0;
#pragma unroll 4
      for (int j = from; j < to; ++j) sum += sh.top.found[j] > c ? sh.weight[j] : 0;
      atomicAdd(&sh.before[i], sum);
    }
    __syncthreads();
    for (int i = t; i < n; i += BLK)
      if (sh.before[i] < target && target <= sh.before[i] + sh.weight[i]) sh.last = sh.top.found[i];
  } else {
    constexpr int kEach = kSpCandidates / BLK;
    sort_all<BLK>(sh.top.found, n);
    u64 own[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += own[i] = t * kEach + i < n ? own_of(sh.top.found[t * kEach + i]) : 0;
    u64 upto = sh.base + block_scan<BLK>(sum, sh.part[0]) - sum;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (upto < target && target <= upto + own[i]) sh.last = sh.top.found[t * kEach + i];
      upto += own[i];
    }
  }
  __syncthreads();
  return {candidate_logit(sh.last), candidate_id(sh.last)};
}

// The draw among the elements that `last` keeps, whose weight by wave is in sh.part[1]: the wave whose part of the row it
// falls in, then the thread.
template <int DT, int BLK, int H>
__device__ __forceinline__ void draw(const SampleArgs& a, const Settings& s, int64_t r, const Row<DT, BLK, H>& row,
                                     const Last& last, const Weight& weight, SampleShared& sh) {
  const int t = threadIdx.x;
  u64 total = 0;
  for (int w = 0; w < BLK / 64; ++w) total += sh.part[1][w];
  u64 left = share_down(s.u, total);
  int wave = 0;
  for (; wave < BLK / 64 - 1 && sh.part[1][wave] <= left; ++wave) left -= sh.part[1][wave];
  // the wave's ids, one range for each thread
  const int each = (row.pieces * 64 + BLK - 1) / BLK, from = row.wave_at(wave) + t * each * 8,
            end = row.wave_at(wave + 1);
  const auto amount = [&](float x, int id) { return last.keeps(x, id) ? weight(x) : 0; };
  u64 mine = 0;
#pragma unroll 1
  for (int i = from; i < from + each * 8 && i < end; i += 8) {
    Raw8<DT> raw;
    float v[8];
    row.fetch(raw, i);
    raw.get(v);
#pragma unroll
    for (int k = 0; k < 8; ++k) mine += amount(v[k], i + k);
  }
  u64 before = block_scan<BLK>(mine, sh.part[0]) - mine;
  if (before <= left && left < before + mine) {
#pragma unroll 1
    for (int i = from; i < from + each * 8 && i < row.vocab; ++i) {
      const float x = load_as_f32(row.row, i, DT);
      const u64 w = amount(x, i);
      if (before <= left && left < before + w) put_token(a, s, r, i, x, total);
      before += w;
    }
  }
}

// The smallest logit whose weight min-p keeps, for s.least above 0.  It lies between a float that is not kept and one that is,
// in the order of their keys: 64 floats around m + T ln((ceil(least) - 1/2) / 2^F), where a weight rounds to what is asked for,
// nearly always hold both; next to 0, where floats lie closer than weights differ, the gap between the two is cut by 65 until
// they are neighbours, six times more at most.
__device__ __forceinline__ float least_logit(const Settings& s, const Weight& weight) {
  const int lane = threadIdx.x & 63;
  uint32_t low = ordered_key(-INFINITY), high = __builtin_amdgcn_readfirstlane(ordered_key(s.top));
  const double near = s.top + s.temp * log((ceil(s.least) - 0.5) / s.one);
  uint32_t from = ordered_key(static_cast<float>(fmax(near, static_cast<double>(kTopLow)))) - 32, step = 1;
#pragma unroll 1
  while (high - low > 1) {
    const int64_t at = static_cast<int64_t>(from) + static_cast<int64_t>(step) * lane;
    const uint32_t key = at <= low ? low : at >= high ? high : static_cast<uint32_t>(at);
    const u64 kept = __ballot(key == high || (key > low && static_cast<double>(weight(key_float(key))) >= s.least));
    const int first = kept ? __ffsll(kept) - 1 : 64;
    if (first > 0) low = __builtin_amdgcn_readlane(key, first - 1);
    if (first < 64) high = __builtin_amdgcn_readlane(key, first);
    step = (high - low + 64) / 65;
    from = low + step;
  }
  return key_float(high);
}

// WHOLE: without top-k and top-p.
template <int DT, int BLK, int H, bool WHOLE>
__global__ void __launch_bounds__(BLK, 4) sample_kernel(SampleArgs a) {
  __shared__ union {
    SampleShared sh;
    AnyShared any;
  } lds;
  SampleShared& sh = lds.sh;
  const int64_t r = blockIdx.x;
  Row<DT, BLK, H> row(static_cast<const char*>(a.x) + r * a.xs * (DT == SF_DTYPE_BF16 ? 2 : 4), a.vocab);
  Settings s(a, r);
  const bool among = !WHOLE && s.k <= BLK && s.k < a.vocab;  // few enough to be gathered
  const bool binned = !WHOLE && !among && (s.k < a.vocab || s.p < 1.0);
  float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, low = INFINITY;
  row.each([&](int p, int, const float (&v)[8]) SF_INLINE {
    const float x = max8(v);
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (p % 4 == g) best[g] = nan_max(best[g], x);
    if (binned) {
#pragma unroll
      for (int k = 0; k < 8; ++k) low = fminf(low, v[k] == -INFINITY ? INFINITY : v[k]);
    }
  });
  const float m = s.top = row_max<BLK>(nan_max(nan_max(best[0], best[1]), nan_max(best[2], best[3])), sh.top.edge[1]);
  if (!(m > -INFINITY)) {
    put_none(a, r, m);
    return;
  }
  const Weight weight{m, 1.4426950408889634 / static_cast<double>(s.temp), a.round, a.poly};
  bool done = m < INFINITY;
  if (done && among) {
    const Bound bound = bound_of<BLK>(best, m, static_cast<int>(s.k), sh.top);
    const int n = gather<4>(row, bound, hits_of(best, bound), sh.top);
    done = n > 0 && n <= kSpCandidates;
    if (done) sample_found<BLK>(a, s, r, weight, bound, n, sh);
  } else if (done) {
    Last last;
    const float least = s.least > 0.0 ? least_logit(s, weight) : -INFINITY;
    double sum = 0.0;
    if (WHOLE && least == -INFINITY) {
      sum = sum_from<true>(row, 0.0f, 0.0f, 0.0f, weight, sh);
    } else {
      Bins bins{m, 0.0f};
      if (binned) {
        low = last_lane(wave_scan(low, INFINITY, [](float a, float b) { return fminf(a, b); }));
        if ((threadIdx.x & 63) == 0) sh.top.edge[0][threadIdx.x >> 6] = low;
        __syncthreads();
        for (int w = 0; w < BLK / 64; ++w) low = fminf(low, sh.top.edge[0][w]);
        // 2^-(F + 1) of the largest weight is 0
        const float range = fminf(m - low, static_cast<float>((a.bits + 1) * 0.6931471805599453 * s.temp));
        bins.scale = fminf(kSpBins / range, 1e30f);
      }
      // by number for top-k, by weight among these for top-p
      const bool cut = s.k < a.vocab, among_p = s.p < 1.0;
      bool by_weight = !cut;
      while (true) {
        u64 target = 0;
        float low = INFINITY, high = -INFINITY;
        if (binned) {
          for (int i = threadIdx.x; i < kSpBins; i += BLK) sh.weight[i] = 0;
          if (threadIdx.x == 0) sh.bin = -1, sh.top.n = 0;
          __syncthreads();
          if (!by_weight)
            fill_bins<0>(row, bins, last, weight, sh);
          else if (!cut)
            fill_bins<1>(row, bins, last, weight, sh);
          else
            fill_bins<2>(row, bins, last, weight, sh);
          __syncthreads();
          target = bin_of_sum<BLK>(
              [&](u64 total) { return by_weight ? share_up(s.p, total) : static_cast<u64>(s.k); }, sh);
          if (sh.bin >= 0) bins.range(sh.bin, low, high);
        }
        // the weight above the bin, for the draw, in the pass that gathers the bin
        const bool at_end = by_weight || !among_p;
        sum = sum_from<false>(row, at_end ? fmaxf(float_above(high), least) : INFINITY, low, high, weight, sh);
        if (!binned) break;
        __syncthreads();
        const int n = sh.top.n;
        done = n <= kSpCandidates;
        if (done && n > 0)
          last = last_of<BLK>(
              bins, n, target,
              [&](float x, int id) -> u64 { return !last.keeps(x, id) ? 0 : by_weight ? weight(x) : 1; }, sh);
        if (!done || at_end) break;
        by_weight = true;
      }
    }
    if (done) {
      const u64 part = wave_scan(Weight::whole(sum));
      if ((threadIdx.x & 63) == 63) sh.part[1][threadIdx.x >> 6] = part;
      __syncthreads();
      if (least > last.x) last = {least, INT32_MAX};
      if (binned) {
        for (int i = threadIdx.x; i < sh.top.n; i += BLK) {
          const u64 c = sh.top.found[i];
          const float x = candidate_logit(c);
          const int id = candidate_id(c);
          if (last.keeps(x, id)) atomicAdd(&sh.part[1][id / (row.pieces * 512)], weight(x));
        }
        __syncthreads();
      }
      draw(a, s, r, row, last, weight, sh);
    }
  }
  if (!done) {
    __syncthreads();
    sample_any<DT, BLK>(a, s, r, row.row, weight, lds.any);
  }
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" int sf_sample_logits(const sf_sample_desc* desc, void* stream) {
  SF_CHECK_ARG(desc, "sf_sample_logits: null descriptor");
  const sf_sample_desc& d = *desc;
  SF_CHECK_ARG(d.dtype == SF_DTYPE_F32 || d.dtype == SF_DTYPE_BF16, "sf_sample_logits: unknown dtype %d", d.dtype);
  SF_CHECK_ARG(d.rows >= 0 && d.rows < SF_TOP_MAX_ROWS && d.vocab > 0 && d.vocab <= SF_TOP_MAX_VOCAB,
               "sf_sample_logits: %lld rows (fewer than %d) of %lld (at most %d)", (long long)d.rows, SF_TOP_MAX_ROWS,
               (long long)d.vocab, SF_TOP_MAX_VOCAB);
  if (d.rows == 0) return SF_OK;
  SF_CHECK_ARG(d.logits && d.uniform && d.tokens, "sf_sample_logits: null pointer");
  SF_CHECK_ARG(d.logits_stride >= 0, "sf_sample_logits: stride %lld", (long long)d.logits_stride);
  SF_CHECK_ARG(d.temperature || d.temperature_all >= 0.0f, "sf_sample_logits: a temperature of %g", d.temperature_all);
  SampleArgs a;
  a.x = d.logits, a.xs = d.logits_stride, a.vocab = static_cast<int>(d.vocab);
  a.u = d.uniform, a.tokens = d.tokens, a.logprobs = d.logprobs;
  a.temp = d.temperature, a.top_k = d.top_k, a.top_p = d.top_p, a.min_p = d.min_p;
  a.temp1 = d.temperature_all, a.top_k1 = d.top_k_all, a.top_p1 = d.top_p_all, a.min_p1 = d.min_p_all;
  // 2e-12 of 2^f
  constexpr double kPoly[8] = {0x1.62e42fef9cc69p-1,  0x1.ebfbdff82a734p-3,  0x1.c6b08da70cce3p-5,
                               0x1.3b2ab70ad2565p-7,  0x1.5d877598350dep-10, 0x1.4308c7183d6a2p-13,
                               0x1.00c0e4e15189cp-16, 0x1.63b2d7971923fp-20};
  memcpy(a.poly, kPoly, sizeof(kPoly));
  // The sums of a thread, which has at most vocab / 512 weights of at most 2^bits, stay below 2^52.
  a.bits = 60;
  for (int64_t n = 1; n < d.vocab; n *= 2) --a.bits;
  if (a.bits > 44) a.bits = 44;
  a.round = 6755399441055744.0 + a.bits;
  const dim3 grid(static_cast<unsigned>(d.rows));
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto with = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    // Pieces that stay in registers: with the code of every setting half as many, as more are spilled (us with 12, 8, 4
    // and 2 of bf16 and half of that of f32, top-p 0.9: 1024 x 32000 bf16 108, 87, 86 and 86; 1024 x 50257 f32 171, 155,
    // 147 and 154).
    constexpr int H = DT == SF_DTYPE_BF16 ? 8 : 4, kFew = H / 2;
    // Threads to a row: 1024 where a CU has at most one row, 512 where two cover each other's waits (us: 64 x 50257 f32 k
    // 50 17 and 20, 64 x 131072 bf16 top-p 0.9 80 and 96; 300 x 32000 bf16 k 400 31 and 22, 1024 x 50257 f32 top-p 0.9 178
    // and 149, 1024 x 131072 f32 k 400 164 and 150, without limits 209 and 209; 300 x 262144 bf16 without limits 141 and
    // 148).
    const bool narrow = d.rows > 256;
    const bool whole = !a.temp && a.temp1 > 0.0f && !a.top_k && (a.top_k1 <= 0 || a.top_k1 >= a.vocab) && !a.top_p &&
                       !(a.top_p1 < 1.0f);
    const int k = !a.temp && !(a.temp1 > 0.0f) ? 1 : a.top_k || a.top_k1 <= 0 ? INT32_MAX : a.top_k1;
    // 256 where many rows each give few candidates (us, k 100, with 512 and 256: 3000 x 8192 bf16 63 and 34, 600 x 32000
    // bf16 27 and 23, 3000 x 32000 f32 103 and 85, 1024 x 65536 bf16 44 and 43, 300 x 65536 bf16 23 and 28, 1024 x 131072
    // bf16 74 and 78).
    if (d.rows > 512 && k <= 128 && a.vocab <= 65536)
      sample_top_k_kernel<DT, 256, 16, 512><<<grid, 256, 0, st>>>(a);
    else if (narrow && k <= 512)
      sample_top_k_kernel<DT, 512, 16, 2048><<<grid, 512, 0, st>>>(a);
    else if (!narrow && k <= 1024)
      sample_top_k_kernel<DT, 1024, 8, 2048><<<grid, 1024, 0, st>>>(a);
    else if (narrow && whole)
      sample_kernel<DT, 512, H, true><<<grid, 512, 0, st>>>(a);
    else if (narrow)
      sample_kernel<DT, 512, kFew, false><<<grid, 512, 0, st>>>(a);
    else if (whole)
      sample_kernel<DT, 1024, H, true><<<grid, 1024, 0, st>>>(a);
    else
      sample_kernel<DT, 1024, kFew, false><<<grid, 1024, 0, st>>>(a);
  };
  if (d.dtype == SF_DTYPE_BF16)
    with(std::integral_constant<int, SF_DTYPE_BF16>{});
  else
    with(std::integral_constant<int, SF_DTYPE_F32>{});
  return launch_status("sf_sample_logits");
}
