// The k largest logits of every row in falling order (equal ones by rising id), their ids, and the row's log-sum-exp at a
// temperature: what is kept of a teacher for distillation, or answered as log-probabilities.
//
// One workgroup per row reads it once, for the sum of exponentials and the maxima of the threads' pieces.  From these follows
// a bound above which the k largest and few others lie (top_bound), whose pieces are taken again from the caches.  The
// candidates are ordered in LDS: counted into bins, placed, ranked among those of their bin.  Rows in which that finds too
// many or too few (equal values, infinities, NaN, hardly more than 8 k logits where these do not fit) are looked through by
// the bits of their logits instead.
//
// 4096 x 32000 bf16, k 64: 60 us (262 MB at 4.4 TB/s; the vector unit is 0.86 busy: an exponential and a fourth of a
// compensated sum for each element beside the maxima); 509 x 131072 f32, k 500: 63 us (267 MB at 4.2 TB/s); 16 x 32000
// bf16, k 20: 10 us, a chain of some ten barriers.  With four passes over the bits of every row's logits: 589, 404 and 71
// us.
#include <type_traits>

#include "sf_top.hpp"

namespace sf {
namespace {

struct TopLogitsArgs {
  const void* x;
  int64_t s0, s1, inner;
  int vocab, k;
  double inv_t;
  void* values;
  int32_t* ids;
  float* lse;
};

// Entry `rank` of row r.
template <int DT>
__device__ __forceinline__ void put(const TopLogitsArgs& a, const void* row, int64_t r, int rank, int id) {
  a.ids[r * a.k + rank] = id;
  if constexpr (DT == SF_DTYPE_F32)
    static_cast<float*>(a.values)[r * a.k + rank] = static_cast<const float*>(row)[id];
  else
    static_cast<uint16_t*>(a.values)[r * a.k + rank] = static_cast<const uint16_t*>(row)[id];
}

// Any row: the k-th largest key by its bits, then the elements above it and the first of its equals.
template <int DT, int BLK, int CAP>
__device__ __forceinline__ void top_of_any(const TopLogitsArgs& a, const void* row, int64_t r, AnyShared& any,
                                           TopShared<CAP>& sh) {
  const int t = threadIdx.x, V = a.vocab;
  const Border border = radix_border<DT, BLK>(row, V, false, a.k, [](float) { return 0ull; }, any);
  const int last = locate<DT, BLK>(
                       row, V, [&](float x, int) { return static_cast<u64>(top_key<DT>(x) == border.key); },
                       [&](u64) { return border.keep - 1; }, any)
                       .id;
  if (t == 0) sh.n = 0;
  __syncthreads();
  each_any<DT, BLK>(row, V, [&](int i, int n, const float (&v)[8]) SF_INLINE {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t key = top_key<DT>(v[k]);
      if (k < n && (key > border.key || (key == border.key && i + k <= last)))
        sh.found[atomicAdd(&sh.n, 1)] = candidate(v[k], i + k);
    }
  });
  __syncthreads();
  sort_all<BLK>(sh.found, a.k);
  for (int i = t; i < a.k; i += BLK) put<DT>(a, row, r, i, candidate_id(sh.found[i]));
}

// k is at most BLK (two groups' maxima a thread) and below CAP.
// Registers for as many workgroups on a CU as its LDS holds (1024 threads: two, 2000 x 131072 f32 191 us, 225 with one).
template <int DT, int BLK, int G, int CAP>
__global__ void __launch_bounds__(BLK, BLK == 1024 ? 8 : 6) top_logits_kernel(TopLogitsArgs a) {
  __shared__ TopShared<CAP> sh;
  __shared__ AnyShared any;
  __shared__ double sums[BLK / 64];
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  const RowAt<DT, BLK> row(static_cast<const char*>(a.x) + ((r / a.inner) * a.s0 + (r % a.inner) * a.s1) *
                                                               (DT == SF_DTYPE_BF16 ? 2 : 4),
                           a.vocab);
  const float c = static_cast<float>(a.inv_t * 1.4426950408889634);
  float top = kTopLow, sum = 0.0f, lost = 0.0f, best[G];
  read_row(row, best, [&](const float (&v)[8]) SF_INLINE {
    float x = top;
#pragma unroll
    for (int k = 0; k < 8; ++k) x = fmaxf(x, v[k]);
    if (x > top) {
      const float f = __builtin_amdgcn_exp2f((top - x) * c);
      sum *= f;
      lost *= f;
      top = x;
    }
    float e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = __builtin_amdgcn_exp2f((v[k] - top) * c);
    // hundreds of small terms beside a large one: what an addition rounds off is carried along
    const float s = (((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]))) - lost, upto = sum + s;
    lost = (upto - sum) - s;
    sum = upto;
  });
  float m = best[0];
#pragma unroll
  for (int g = 1; g < G; ++g) m = nan_max(m, best[g]);
  m = row_max<BLK>(m, sh.edge[1]);
  const bool plain = m > -INFINITY && m < INFINITY;
  int n = 0;
  double total = sum == 0.0f || !plain ? 0.0 : static_cast<double>(sum * __builtin_amdgcn_exp2f((top - m) * c));
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
  if ((t & 63) == 0) sums[t >> 6] = total;
  Bound bound;
  if (plain) {
    bound = bound_of<BLK>(best, m, a.k, sh);
    n = gather<G>(row, bound, hits_of(best, bound), sh);
  } else {
    __syncthreads();
  }
  if (t == 0 && a.lse) {
    total = 0.0;
    for (int w = 0; w < BLK / 64; ++w) total += sums[w];
    a.lse[r] = plain ? static_cast<float>(m * a.inv_t + log(total)) : m;
  }
  if (n < a.k || n > CAP) {  // -inf, inf or NaN among the k, or too many
    top_of_any<DT, BLK>(a, row.row, r, any, sh);
  } else {
    sort_found<BLK>(bound, m, n, sh);
    for (int i = t; i < a.k; i += BLK) put<DT>(a, row.row, r, i, candidate_id(sh.found[i]));
  }
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" int sf_top_logits(const sf_top_logits_desc* desc, void* stream) {
  SF_CHECK_ARG(desc, "sf_top_logits: null descriptor");
  const sf_top_logits_desc& d = *desc;
  SF_CHECK_ARG(d.dtype == SF_DTYPE_F32 || d.dtype == SF_DTYPE_BF16, "sf_top_logits: unknown dtype %d", d.dtype);
  SF_CHECK_ARG(d.rows >= 0 && d.rows < SF_TOP_MAX_ROWS && d.vocab > 0 && d.vocab <= SF_TOP_MAX_VOCAB,
               "sf_top_logits: %lld rows (fewer than %d) of %lld (at most %d)", (long long)d.rows, SF_TOP_MAX_ROWS,
               (long long)d.vocab, SF_TOP_MAX_VOCAB);
  SF_CHECK_ARG(d.k >= 1 && d.k <= d.vocab && d.k <= SF_TOP_MAX_K, "sf_top_logits: the %lld largest of %lld (at most %d)",
               (long long)d.k, (long long)d.vocab, SF_TOP_MAX_K);
  SF_CHECK_ARG(d.inner > 0 && d.rows % d.inner == 0 && d.outer_stride >= 0 && d.row_stride >= 0,
               "sf_top_logits: rows in groups of %lld, strides %lld, %lld", (long long)d.inner,
               (long long)d.outer_stride, (long long)d.row_stride);
  SF_CHECK_ARG(d.temperature >= 1.0e-30f && d.temperature <= 1.0e30f, "sf_top_logits: temperature %g", d.temperature);
  if (d.rows == 0) return SF_OK;
  SF_CHECK_ARG(d.logits && d.values && d.ids, "sf_top_logits: null pointer");
  TopLogitsArgs a;
  a.x = d.logits, a.s0 = d.outer_stride, a.s1 = d.row_stride, a.inner = d.inner;
  a.vocab = static_cast<int>(d.vocab), a.k = static_cast<int>(d.k);
  a.inv_t = 1.0 / static_cast<double>(d.temperature);
  a.values = d.values, a.ids = d.ids, a.lse = d.lse;
  const dim3 grid(static_cast<unsigned>(d.rows));
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto with = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    // Threads to a row: many where a CU has at most one row, fewer where rows can cover each other's waits (us with 1024,
    // 512 and 256 threads, k 20: bf16 100 x 32000 14, 14 and 17; 1024 x 32000 31, 27 and 24; 3000 x 32000 71, 55 and 49;
    // f32 3000 x 50257 112, 110 and 117; 509 x 131072 with k 500 70 and 75).
    if (DT == SF_DTYPE_BF16 && d.rows > 512 && d.k <= 128 && d.vocab <= 256 * 8 * 32)
      top_logits_kernel<SF_DTYPE_BF16, 256, 16, 512><<<grid, 256, 0, st>>>(a);
    else if (d.rows > 256 && d.k <= 512 && d.vocab <= (DT == SF_DTYPE_BF16 ? 131072 : 65536))
      top_logits_kernel<DT, 512, 16, 2048><<<grid, 512, 0, st>>>(a);
    else
      top_logits_kernel<DT, 1024, 8, 2048><<<grid, 1024, 0, st>>>(a);
  };
  if (d.dtype == SF_DTYPE_BF16)
    with(std::integral_constant<int, SF_DTYPE_BF16>{});
  else
    with(std::integral_constant<int, SF_DTYPE_F32>{});
  return launch_status("sf_top_logits");
}
