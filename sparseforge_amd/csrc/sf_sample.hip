// A token for every row from given random numbers.  For a row x with maximum m, at temperature T, the tokens ordered by
// falling logit (equal ones by rising id):
//   w_i = exp((x_i - m) / T)
//   top-k keeps the first k; top-p of these the fewest first tokens that hold p of their weight; min-p those of at least
//   min_p times the largest weight.  All three keep a first part of that order.
//   the token is the first, by id, at which the weight of the kept tokens up to it exceeds u times their whole weight.
// Weights are formed in f64 and summed as integers of 2^-F, F = 62 - log2 of the vocabulary (45 for 131072 tokens): sums
// do not depend on their order, and what a cumulative sum is off by (about 2^-F of the largest weight) decides a draw
// once in 1e8 draws; sums of f32 exponentials would decide one in thousands over large vocabularies.
//
// One workgroup per row, which it holds in registers if it fits.  With top-k up to 1024 the row's largest are gathered in
// LDS (gather_top) and the rest happens among them.  Without it, top-p's border is the place in a histogram of weights by
// logit where their sum reaches p, resolved among the tokens of that bin; the draw finds the wave's part of the row, then
// the thread's.
#include <type_traits>

#include "sf_top.hpp"

namespace sf {
namespace {

constexpr int kSpBlock = 1024;
constexpr int kSpBins = 2048;

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
};

// Weights exp((x - top) / T) as integers of 2^-bits (bits <= 51); 2^bits exactly for the largest logit, which is finite.
struct Weight {
  double top, c;  // c: log2(e) / T
  int bits;
  __device__ __forceinline__ u64 operator()(float x) const {
    // 2^z = 2^n 2^f, f in [-1/2, 1/2]: n is in the low bits of the sum with 1.5 * 2^52.  -inf ends at the smallest z.
    constexpr double kRound = 6755399441055744.0;
    const double z = fmax((static_cast<double>(x) - top) * c, -64.0);
    const double rounded = z + kRound;
    const double f = z - (rounded - kRound);
    // (2^f - 1) / f, the polynomial of degree 8 through its values at the Chebyshev points: 4e-14 of 2^f
    double p = 0x1.b63880a30e9ffp-24;
    p = fma(p, f, 0x1.63d136366db24p-20);
    p = fma(p, f, 0x1.ffcb9515a8016p-17);
    p = fma(p, f, 0x1.4308ac85aa947p-13);
    p = fma(p, f, 0x1.5d87fe86fe88ep-10);
    p = fma(p, f, 0x1.3b2ab7181b755p-7);
    p = fma(p, f, 0x1.c6b08d7047e52p-5);
    p = fma(p, f, 0x1.ebfbdff823cedp-3);
    p = fma(p, f, 0x1.62e42fefa39efp-1);
    p = fma(p, f, 1.0);
    const u64 scaled = static_cast<u64>(__double_as_longlong(p)) +
                       (static_cast<u64>(static_cast<uint32_t>(__double_as_longlong(rounded)) + bits) << 52);
    // with 2^52 added the low bits are the rounded integer
    return static_cast<u64>(__double_as_longlong(__longlong_as_double(scaled) + 4503599627370496.0)) & 0xfffffffffffffull;
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

struct SampleShared {
  TopShared top;
  u64 weight[kSpBins];  // of the found in their order, or of bins
  u64 before[kTopCandidates];
  int id[SF_TOP_MAX_K];
  float logit[SF_TOP_MAX_K];
  u64 part[2][kSpBlock / 64];
  u64 total, base, last;
  int count, bin;
};

// Among the row's n largest, which sh.top.found holds: top-k, top-p, min-p and the draw.
__device__ __forceinline__ void sample_found(const SampleArgs& a, const Settings& s, int64_t r, const Weight& weight,
                                             int n, SampleShared& sh) {
  const int t = threadIdx.x;
  for (int i = t; i < n; i += kSpBlock) {
    const u64 own = sh.top.found[i];
    const int rank = rank_of(own, sh.top.found, n);
    if (rank < s.k) {
      sh.logit[rank] = candidate_logit(own);
      sh.weight[rank] = weight(sh.logit[rank]);
      sh.id[rank] = candidate_id(own);
    }
  }
  if (t == 0) sh.total = 0, sh.count = 0;
  __syncthreads();
  const int k = s.k < n ? static_cast<int>(s.k) : n;
  const u64 w = t < k ? sh.weight[t] : 0;
  const u64 upto = block_scan<kSpBlock>(w, sh.part[0]);
  u64 all = 0;
  for (int i = 0; i < kSpBlock / 64; ++i) all += sh.part[0][i];
  const bool kept = t < k && (s.p >= 1.0 || upto - w < share_up(s.p, all)) && static_cast<double>(w) >= s.least;
  if (kept) {
    atomicMax(&sh.total, upto);
    atomicMax(&sh.count, t + 1);
  }
  __syncthreads();
  if (!kept) return;
  const int id = sh.id[t], count = sh.count;
  const u64 total = sh.total, want = share_down(s.u, total);
  u64 sum = 0;
  for (int i = 0; i < count; ++i) sum += sh.id[i] <= id ? sh.weight[i] : 0;
  if (sum - w <= want && want < sum) put_token(a, s, r, id, sh.logit[t], total);
}

// Places of logits in a histogram from the largest down; what has no weight ends in the last bin.
struct Bins {
  float top, scale;
  __device__ __forceinline__ int of(float x) const {
    const float y = (top - x) * scale;
    return y < kSpBins - 1 ? static_cast<int>(y) : kSpBins - 1;
  }
};

// What top-k and top-p keep: up to this candidate in the order of logits.
struct Last {
  u64 c;
  __device__ __forceinline__ bool keeps(float x, int id) const { return candidate(x, id) >= c; }
};

// The last element, in the order of logits, at which the sum of amount(x, id) before it is below want(whole sum): found in
// last.  False: more than kTopCandidates are in the bin where that happens.  A sum that stays below takes in everything.
template <int DT, int H, typename M, typename A>
__device__ __forceinline__ bool border_of(const Row<DT, kSpBlock, H>& row, const Bins& bins, M&& amount, A&& want,
                                          Last& last, SampleShared& sh) {
  constexpr int kEach = kSpBins / kSpBlock;
  const int t = threadIdx.x;
  for (int i = t; i < kSpBins; i += kSpBlock) sh.weight[i] = 0;
  if (t == 0) sh.bin = -1, sh.top.n = 0;
  __syncthreads();
  row.each([&](int, int i, const float (&v)[8]) SF_INLINE {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const u64 w = amount(v[k], i + k);
      if (w) atomicAdd(&sh.weight[bins.of(v[k])], w);
    }
  });
  __syncthreads();
  u64 own[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += own[i] = sh.weight[t * kEach + i];
  u64 upto = block_scan<kSpBlock>(sum, sh.part[0]) - sum, total = 0;
  for (int i = 0; i < kSpBlock / 64; ++i) total += sh.part[0][i];
  const u64 target = want(total);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (upto < target && target <= upto + own[i]) sh.bin = t * kEach + i, sh.base = upto;
    upto += own[i];
  }
  __syncthreads();
  const int bin = sh.bin;
  if (bin < 0) return true;
  uint32_t hits = 0;
  row.each([&](int p, int i, const float (&v)[8]) SF_INLINE {
    bool any = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) any |= bins.of(v[k]) == bin;
    if (any) hits |= 1u << p;
  });
  const int n = gather(row, [&](float x) { return bins.of(x) == bin; }, hits, sh.top);
  if (n > kTopCandidates) return false;
  for (int i = t; i < n; i += kSpBlock) {
    const u64 c = sh.top.found[i];
    sh.weight[i] = amount(candidate_logit(c), candidate_id(c));
    sh.before[i] = sh.base;
  }
  __syncthreads();
  // every candidate's sum before it, its terms shared by as many threads as there are
  const int parts = n < kSpBlock ? kSpBlock / n : 1, size = (n + parts - 1) / parts;
  for (int at = t; at < n * parts; at += kSpBlock) {
    const int i = at % n, from = at / n * size, to = from + size < n ? from + size : n;
    const u64 c = sh.top.found[i];
    u64 sum = 0;
    for (int j = from; j < to; ++j) sum += sh.top.found[j] > c ? sh.weight[j] : 0;
    atomicAdd(&sh.before[i], sum);
  }
  __syncthreads();
  for (int i = t; i < n; i += kSpBlock)
    if (sh.before[i] < target && target <= sh.before[i] + sh.weight[i]) sh.last = sh.top.found[i];
  __syncthreads();
  last.c = sh.last;
  return true;
}

// The draw among the elements with amount(x, id): the wave whose part of the row it falls in, then the thread.
template <int DT, int H, typename M>
__device__ __forceinline__ void draw(const SampleArgs& a, const Settings& s, int64_t r, const Row<DT, kSpBlock, H>& row,
                                     float cut, M&& amount, SampleShared& sh) {
  const int t = threadIdx.x;
  u64 sum = 0;
  row.each([&](int, int i, const float (&v)[8]) SF_INLINE {
    if (max8(v) >= cut) {
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += amount(v[k], i + k);
    }
  });
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if ((t & 63) == 0) sh.part[1][t >> 6] = sum;
  __syncthreads();
  u64 total = 0;
  for (int w = 0; w < kSpBlock / 64; ++w) total += sh.part[1][w];
  u64 left = share_down(s.u, total);
  int wave = 0;
  for (; wave < kSpBlock / 64 - 1 && sh.part[1][wave] <= left; ++wave) left -= sh.part[1][wave];
  // the wave's ids, one range for each thread
  const int each = (row.pieces * 64 + kSpBlock - 1) / kSpBlock, from = row.wave_at(wave) + t * each * 8,
            end = row.wave_at(wave + 1);
  u64 mine = 0;
  for (int i = from; i < from + each * 8 && i < end; i += 8) {
    Raw8<DT> raw;
    float v[8];
    row.fetch(raw, i);
    raw.get(v);
    for (int k = 0; k < 8; ++k) mine += amount(v[k], i + k);
  }
  u64 before = block_scan<kSpBlock>(mine, sh.part[0]) - mine;
  if (before <= left && left < before + mine)
    for (int i = from; i < from + each * 8 && i < row.vocab; ++i) {
      const float x = load_as_f32(row.row, i, DT);
      const u64 w = amount(x, i);
      if (before <= left && left < before + w) put_token(a, s, r, i, x, total);
      before += w;
    }
}

template <int DT, int H>
__global__ void __launch_bounds__(kSpBlock) sample_kernel(SampleArgs a) {
  __shared__ union {
    SampleShared sh;
    AnyShared any;
  } lds;
  SampleShared& sh = lds.sh;
  const int64_t r = blockIdx.x;
  const Row<DT, kSpBlock, H> row(static_cast<const char*>(a.x) + r * a.xs * (DT == SF_DTYPE_BF16 ? 2 : 4), a.vocab);
  const float T = a.temp ? a.temp[r] : a.temp1, top_p = a.top_p ? a.top_p[r] : a.top_p1;
  const float min_p = a.min_p ? a.min_p[r] : a.min_p1;
  const int top_k = a.top_k ? a.top_k[r] : a.top_k1;
  const bool greedy = !(T > 0.0f);
  Settings s;
  s.u = a.u[r];
  s.temp = greedy ? 1.0f : T;
  s.k = greedy ? 1 : top_k <= 0 || top_k > a.vocab ? a.vocab : top_k;
  s.p = !greedy && top_p < 1.0f ? static_cast<double>(top_p) : 1.0;
  s.one = ldexp(1.0, a.bits);
  s.least = (min_p > 1.0f ? 1.0 : min_p > 0.0f ? static_cast<double>(min_p) : 0.0) * s.one;
  float best[2];
  const float m = s.top = row_max(row, best, sh.top.edge[1]);
  if (m != m || m == -INFINITY) {
    if (threadIdx.x == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = m;
    }
    return;
  }
  const Weight weight{m, 1.4426950408889634 / static_cast<double>(s.temp), a.bits};
  bool done = m < INFINITY;
  if (done && s.k <= SF_TOP_MAX_K && s.k < a.vocab) {
    const Bound bound = top_bound<kSpBlock>(best, m, static_cast<int>(s.k), sh.top);
    uint32_t hits = 0;
    row.each([&](int p, int, const float (&v)[8]) SF_INLINE {
      if (bound.holds(max8(v))) hits |= 1u << p;
    });
    const int n = gather(row, [&](float x) { return bound.holds(x); }, hits, sh.top);
    done = n > 0 && n <= kTopCandidates;
    if (done) sample_found(a, s, r, weight, n, sh);
  } else if (done) {
    Last last{0};
    if (s.k < a.vocab || s.p < 1.0) {
      float low = INFINITY;
      row.each([&](int, int, const float (&v)[8]) SF_INLINE {
#pragma unroll
        for (int k = 0; k < 8; ++k) low = fminf(low, v[k] == -INFINITY ? INFINITY : v[k]);
      });
      for (int off = 32; off > 0; off >>= 1) low = fminf(low, __shfl_xor(low, off, 64));
      if ((threadIdx.x & 63) == 0) sh.top.edge[0][threadIdx.x >> 6] = low;
      __syncthreads();
      for (int w = 0; w < kSpBlock / 64; ++w) low = fminf(low, sh.top.edge[0][w]);
      // 2^-(F + 1) of the largest weight is 0
      const float range = fminf(m - low, static_cast<float>((a.bits + 1) * 0.6931471805599453 * s.temp));
      const Bins bins{m, fminf(kSpBins / range, 1e30f)};
      if (s.k < a.vocab)
        done = border_of(
            row, bins, [&](float x, int) -> u64 { return x > -INFINITY; },
            [&](u64) { return static_cast<u64>(s.k); }, last, sh);
      if (done && s.p < 1.0) {
        __syncthreads();
        done = border_of(
            row, bins, [&](float x, int id) -> u64 { return last.keeps(x, id) ? weight(x) : 0; },
            [&](u64 total) { return share_up(s.p, total); }, last, sh);
      }
    }
    if (done) {
      // no element below this one is kept
      float cut = last.c ? candidate_logit(last.c) : -INFINITY;
      if (s.least > 0.0) {
        const double d = s.temp * log(s.least / s.one);
        cut = fmaxf(cut, static_cast<float>(m + d - 1e-6 * (fabs(m) + fabs(d))));
      }
      draw(
          a, s, r, row, cut,
          [&](float x, int id) -> u64 {
            if (x < cut || !last.keeps(x, id)) return 0;
            const u64 w = weight(x);
            return static_cast<double>(w) >= s.least ? w : 0;
          },
          sh);
    }
  }
  if (!done) {
    __syncthreads();
    sample_any<DT, kSpBlock>(a, s, r, row.row, weight, lds.any);
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
  a.bits = 62;  // sums of vocab weights of at most 2^bits stay below 2^62; the weights below 2^52
  for (int64_t n = 1; n < d.vocab; n *= 2) --a.bits;
  if (a.bits > 50) a.bits = 50;
  const dim3 grid(static_cast<unsigned>(d.rows));
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto with = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (a.vocab <= kSpBlock * 8 * 4)
      sample_kernel<DT, 4><<<grid, kSpBlock, 0, st>>>(a);
    else
      sample_kernel<DT, 8><<<grid, kSpBlock, 0, st>>>(a);
  };
  if (d.dtype == SF_DTYPE_BF16)
    with(std::integral_constant<int, SF_DTYPE_BF16>{});
  else
    with(std::integral_constant<int, SF_DTYPE_F32>{});
  return launch_status("sf_sample_logits");
}
