// The k largest logits of every row in falling order (equal ones by rising id), their ids, and the row's log-sum-exp at a
// temperature: what is kept of a teacher for distillation, or answered as log-probabilities.
//
// One workgroup per row: it finds the k-th largest key, gathers what lies above it and the first of its equals, and sorts
// these in LDS.
#include "sf_top.hpp"

namespace sf {
namespace {

constexpr int kTlBlock = 1024;
constexpr int kTlTiles = SF_TOP_MAX_VOCAB / (kTlBlock * 8);

struct TopLogitsArgs {
  const void* x;
  int64_t s0, s1, inner;
  int vocab, k, dt;
  double inv_t;
  void* values;
  int32_t* ids;
  float* lse;
};

template <int DT>
__global__ void __launch_bounds__(kTlBlock) top_logits_kernel(TopLogitsArgs a) {
  __shared__ u64 mass[256];
  __shared__ uint32_t count[256];
  __shared__ u64 sums[kTlTiles * (kTlBlock / 64)];
  __shared__ u64 shared[3];
  __shared__ float part[kTlBlock / 64];
  __shared__ double partd[kTlBlock / 64];
  __shared__ u64 found[SF_TOP_MAX_K];
  __shared__ int at;
  const int64_t r = blockIdx.x, base = (r / a.inner) * a.s0 + (r % a.inner) * a.s1;
  const int t = threadIdx.x, V = a.vocab;
  float m = -INFINITY;
  top_scan<DT, kTlBlock>(a.x, base, V, [&](int, int, int n, const float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) m = fmaxf(m, v[k]);
  });
  m = block_max_f<kTlBlock>(m, part);
  const float c = static_cast<float>(a.inv_t * 1.4426950408889634);
  const float ref = m == -INFINITY || m == INFINITY ? 0.0f : m;
  float sum = 0.0f;
  top_scan<DT, kTlBlock>(a.x, base, V, [&](int, int, int n, const float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) sum += __builtin_amdgcn_exp2f((v[k] - ref) * c);
  });
  double total = sum;
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
  if ((t & 63) == 0) partd[t >> 6] = total;
  if (t == 0) at = 0;
  const Border border = radix_border<DT, kTlBlock>(a.x, base, V, false, a.k, [](float) { return 0ull; }, mass, count,
                                                   shared);
  const int last = locate<DT, kTlBlock, kTlTiles>(
                       a.x, base, V, [&](float x, int) { return static_cast<u64>(top_key<DT>(x) == border.key); },
                       [&](u64) { return border.keep - 1; }, sums, shared)
                       .id;
  int size = 1;
  while (size < a.k) size *= 2;
  for (int i = t; i < size; i += kTlBlock) found[i] = 0;
  __syncthreads();
  top_scan<DT, kTlBlock>(a.x, base, V, [&](int, int i, int n, const float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t key = top_key<DT>(v[k]);
      if (k < n && (key > border.key || (key == border.key && i + k <= last)))
        found[atomicAdd(&at, 1)] = static_cast<u64>(key) << 32 | static_cast<uint32_t>(~(i + k));
    }
  });
  __syncthreads();
  // bitonic sort, falling
  for (int step = 2; step <= size; step *= 2)
    for (int d = step / 2; d > 0; d /= 2) {
      for (int i = t; i < size; i += kTlBlock) {
        const int j = i ^ d;
        if (j > i && (found[i] < found[j]) == ((i & step) == 0)) {
          const u64 x = found[i];
          found[i] = found[j];
          found[j] = x;
        }
      }
      __syncthreads();
    }
  for (int i = t; i < a.k; i += kTlBlock) {
    const int id = static_cast<int>(~static_cast<uint32_t>(found[i]));
    a.ids[r * a.k + i] = id;
    if (DT == SF_DTYPE_F32)
      static_cast<float*>(a.values)[r * a.k + i] = static_cast<const float*>(a.x)[base + id];
    else
      static_cast<uint16_t*>(a.values)[r * a.k + i] = static_cast<const uint16_t*>(a.x)[base + id];
  }
  if (t == 0 && a.lse) {
    total = 0.0;
    for (int w = 0; w < kTlBlock / 64; ++w) total += partd[w];
    a.lse[r] = static_cast<float>(ref * a.inv_t + log(total));
  }
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" int sf_top_logits(const sf_top_logits_desc* desc, void* stream) {
  SF_CHECK_ARG(desc, "sf_top_logits: null descriptor");
  const sf_top_logits_desc& d = *desc;
  SF_CHECK_ARG(d.dtype == SF_DTYPE_F32 || d.dtype == SF_DTYPE_BF16, "sf_top_logits: unknown dtype %d", d.dtype);
  SF_CHECK_ARG(d.rows >= 0 && d.rows < (1ll << 31) && d.vocab > 0 && d.vocab <= SF_TOP_MAX_VOCAB,
               "sf_top_logits: %lld rows of %lld (at most %d)", (long long)d.rows, (long long)d.vocab,
               SF_TOP_MAX_VOCAB);
  SF_CHECK_ARG(d.k >= 1 && d.k <= d.vocab && d.k <= SF_TOP_MAX_K, "sf_top_logits: the %lld largest of %lld (at most %d)",
               (long long)d.k, (long long)d.vocab, SF_TOP_MAX_K);
  SF_CHECK_ARG(d.inner > 0 && d.rows % d.inner == 0 && d.outer_stride >= 0 && d.row_stride >= 0,
               "sf_top_logits: rows in groups of %lld, strides %lld, %lld", (long long)d.inner,
               (long long)d.outer_stride, (long long)d.row_stride);
  SF_CHECK_ARG(d.temperature > 0.0f && d.temperature <= 3.0e38f, "sf_top_logits: temperature %g", d.temperature);
  if (d.rows == 0) return SF_OK;
  SF_CHECK_ARG(d.logits && d.values && d.ids, "sf_top_logits: null pointer");
  TopLogitsArgs a;
  a.x = d.logits, a.s0 = d.outer_stride, a.s1 = d.row_stride, a.inner = d.inner;
  a.vocab = static_cast<int>(d.vocab), a.k = static_cast<int>(d.k);
  a.inv_t = 1.0 / static_cast<double>(d.temperature);
  a.values = d.values, a.ids = d.ids, a.lse = d.lse;
  const dim3 grid(static_cast<unsigned>(d.rows));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (d.dtype == SF_DTYPE_BF16)
    top_logits_kernel<SF_DTYPE_BF16><<<grid, kTlBlock, 0, st>>>(a);
  else
    top_logits_kernel<SF_DTYPE_F32><<<grid, kTlBlock, 0, st>>>(a);
  return launch_status("sf_top_logits");
}
