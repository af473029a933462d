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
// One workgroup per row.
#include "sf_top.hpp"

namespace sf {
namespace {

constexpr int kSpBlock = 1024;
constexpr int kSpTiles = SF_TOP_MAX_VOCAB / (kSpBlock * 8);

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

// 2^f for |f| <= 1/2 by its series, to 2^-52.
__device__ __forceinline__ double exp2_frac(double f) {
  constexpr double kLn2 = 0.693147180559945309417232121458;
  const double y = f * kLn2;
  double p = 1.0 / 6227020800.0;
  p = fma(p, y, 1.0 / 479001600.0);
  p = fma(p, y, 1.0 / 39916800.0);
  p = fma(p, y, 1.0 / 3628800.0);
  p = fma(p, y, 1.0 / 362880.0);
  p = fma(p, y, 1.0 / 40320.0);
  p = fma(p, y, 1.0 / 5040.0);
  p = fma(p, y, 1.0 / 720.0);
  p = fma(p, y, 1.0 / 120.0);
  p = fma(p, y, 1.0 / 24.0);
  p = fma(p, y, 1.0 / 6.0);
  p = fma(p, y, 0.5);
  p = fma(p, y, 1.0);
  return fma(p, y, 1.0);
}

// Weights as integers of 2^-bits.
struct Weight {
  float top;
  double c;  // log2(e) / T
  int bits;
  __device__ __forceinline__ u64 operator()(float x) const {
    if (x == top) return 1ull << bits;
    const double z = (static_cast<double>(x) - static_cast<double>(top)) * c;
    if (!(z > -bits - 1.0)) return 0;  // also -inf, and everything below a maximum of +inf
    const double n = rint(z);
    // 2^52 added: the sum's low bits are the rounded integer
    const double w = ldexp(exp2_frac(z - n), static_cast<int>(n) + bits) + 4503599627370496.0;
    return __double_as_longlong(w) & 0xfffffffffffffull;
  }
};

template <int DT>
__global__ void __launch_bounds__(kSpBlock) sample_kernel(SampleArgs a) {
  __shared__ u64 mass[256];
  __shared__ uint32_t count[256];
  __shared__ u64 sums[kSpTiles * (kSpBlock / 64)];
  __shared__ u64 shared[3];
  __shared__ float part[kSpBlock / 64];
  const int64_t r = blockIdx.x, base = r * a.xs;
  const int t = threadIdx.x, V = a.vocab;
  float m = -INFINITY;
  int nan = 0;
  top_scan<DT, kSpBlock>(a.x, base, V, [&](int, int, int n, const float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) {
        nan |= v[k] != v[k];
        m = fmaxf(m, v[k]);
      }
  });
  m = block_max_f<kSpBlock>(m, part);
  nan = __syncthreads_or(nan);
  if (nan || m == -INFINITY) {
    if (t == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = nan ? NAN : -INFINITY;
    }
    return;
  }
  const float T = a.temp ? a.temp[r] : a.temp1;
  const bool greedy = !(T > 0.0f);
  int64_t top_k = a.top_k ? a.top_k[r] : a.top_k1;
  const float top_p = a.top_p ? a.top_p[r] : a.top_p1, min_p = a.min_p ? a.min_p[r] : a.min_p1;
  const Weight weight{m, greedy ? 0.0 : 1.4426950408889634 / static_cast<double>(T), a.bits};
  const double one = ldexp(1.0, a.bits);
  if (greedy || top_k <= 0 || top_k > V) top_k = greedy ? 1 : V;
  Border border{0, ~0ull, 0};
  u64 z = 0;
  if (top_k < V) {
    border = radix_border<DT, kSpBlock>(a.x, base, V, false, top_k, weight, mass, count, shared);
    // count and weight of the border's own key are in the last pass's bins
    z = border.above + border.keep * (mass[border.key & 255] / count[border.key & 255]);
    __syncthreads();
  } else if (top_p < 1.0f) {
    const auto all = [&](float x, int) { return weight(x); };
    z = locate<DT, kSpBlock, kSpTiles>(a.x, base, V, all, [](u64 s) { return s; }, sums, shared).total;
  }
  if (top_p < 1.0f && !greedy) {
    const double want = ceil(static_cast<double>(top_p) * static_cast<double>(z));
    const u64 target = want < 1.0 ? 1 : static_cast<u64>(want) < z ? static_cast<u64>(want) : z;
    border = radix_border<DT, kSpBlock>(a.x, base, V, true, target, weight, mass, count, shared);
    const u64 each = mass[border.key & 255] / count[border.key & 255];
    border.keep = (border.keep + each - 1) / each;
    __syncthreads();
  }
  int last = V;  // the last id of those at the border that is kept
  if (border.keep != ~0ull)
    last = locate<DT, kSpBlock, kSpTiles>(
               a.x, base, V, [&](float x, int) { return static_cast<u64>(top_key<DT>(x) == border.key); },
               [&](u64) { return border.keep - 1; }, sums, shared)
               .id;
  const double least = (min_p > 1.0f ? 1.0 : min_p > 0.0f ? static_cast<double>(min_p) : 0.0) * one;
  const auto kept = [&](float x, int id) -> u64 {
    const uint32_t key = top_key<DT>(x);
    if (key < border.key || (key == border.key && id > last)) return 0;
    const u64 w = weight(x);
    return static_cast<double>(w) >= least ? w : 0;
  };
  const float uf = a.u[r];
  const Place at = locate<DT, kSpBlock, kSpTiles>(
      a.x, base, V, kept,
      [&](u64 total) {
        const double u = uf > 0.0f ? static_cast<double>(uf) : 0.0;
        const double want = floor(u * static_cast<double>(total));
        return want < static_cast<double>(total) && static_cast<u64>(want) < total ? static_cast<u64>(want) : total - 1;
      },
      sums, shared);
  if (t == 0) {
    a.tokens[r] = at.id;
    if (a.logprobs) {
      const double x = load_as_f32(a.x, base + at.id, DT);
      const double z1 = log(static_cast<double>(at.total) / one);
      a.logprobs[r] = static_cast<float>((x == m || greedy ? 0.0 : (x - m) / static_cast<double>(T)) - z1);
    }
  }
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" int sf_sample_logits(const sf_sample_desc* desc, void* stream) {
  SF_CHECK_ARG(desc, "sf_sample_logits: null descriptor");
  const sf_sample_desc& d = *desc;
  SF_CHECK_ARG(d.dtype == SF_DTYPE_F32 || d.dtype == SF_DTYPE_BF16, "sf_sample_logits: unknown dtype %d", d.dtype);
  SF_CHECK_ARG(d.rows >= 0 && d.rows < (1ll << 31) && d.vocab > 0 && d.vocab <= SF_TOP_MAX_VOCAB,
               "sf_sample_logits: %lld rows of %lld (at most %d)", (long long)d.rows, (long long)d.vocab,
               SF_TOP_MAX_VOCAB);
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
  if (d.dtype == SF_DTYPE_BF16)
    sample_kernel<SF_DTYPE_BF16><<<grid, kSpBlock, 0, st>>>(a);
  else
    sample_kernel<SF_DTYPE_F32><<<grid, kSpBlock, 0, st>>>(a);
  return launch_status("sf_sample_logits");
}
