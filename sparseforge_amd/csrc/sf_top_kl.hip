// Distillation from a teacher's recorded top logits: KL of a student's whole softmax from the listed tokens (and, with
// the teacher's log-sum-exp, from the rest taken together), its gradient, and the product of its second derivative with a
// direction.  At temperature T, for a row with listed ids i_k, teacher logits t_k, student logits s over the vocabulary:
//   a = s / T,  Z = log sum_V exp a_j,  q_j = exp(a_j - Z),  b_k = t_k / T,  p_k = exp(b_k - N)
//   N = log sum_k exp b_k (then the row is renormalised, r = 0), or the given lse (then r = 1 - sum p, not below 0)
//   KL = sum_k p_k (log p_k - log q_(i_k)) + r (log r - log q_rest),   q_rest = sum over unlisted j of q_j
//   dKL/da_j = P q_j - p_j - r q_j / q_rest [j unlisted],              P = sum p + r
// With Z_r the log-sum-exp of the unlisted tokens and kappa = exp(Z - Z_r) the gradient of an unlisted token is
// (P - r kappa) q_j: one exponential.  Its derivative along u: with U = sum u_j q_j and U_r = the same over the unlisted,
//   h_j = q_j ((P - r kappa) u_j - (P U - r kappa^2 U_r))  [unlisted],   P q_j (u_j - U)  [listed].
// The rest's sums are formed without the listed tokens (one bit for each of the vocabulary in LDS), not as a difference.
//
// One workgroup per row streams it once.  Listed tokens (at most a few hundred) are gathered and handled in f64.
#include "sf_common.hpp"

namespace sf {
namespace {

constexpr int kTkBlock = 256;
constexpr int kTkStats = 6;  // f64 of a row that the backward needs
constexpr float kTkLow = -3.0e38f;  // start of a running maximum: finite, so that -inf minus it is -inf and not NaN

struct TopKlArgs {
  const void* s;
  int64_t s0, s1, inner;  // row r lies at (r / inner) s0 + (r % inner) s1
  const void* values;
  const void* ids;
  const float* lse;      // null: renormalised
  const float* weights;  // null: all 1
  int64_t vocab;
  int k, vdt, id_bytes;
  double inv_t;
};

struct RowStats {
  double z, zr, n, p, r;  // Z, Z_r, N, P, r; in units of a
  double twice;           // an id is listed more than once
};

__device__ __forceinline__ int64_t tk_id(const TopKlArgs& a, int64_t at) {
  const int64_t id = a.id_bytes == 8 ? static_cast<const int64_t*>(a.ids)[at] : static_cast<const int32_t*>(a.ids)[at];
  return id >= 0 && id < a.vocab ? id : -1;
}

// n (at most 8) elements from any element's address.
template <int DT>
__device__ __forceinline__ void tk_load8(const void* p, int64_t i, int n, float (&v)[8]) {
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
    for (int k = 0; k < 8; ++k) v[k] = k < n ? load_as_f32(p, i + k, DT) : -INFINITY;
  }
}
template <int DT>
__device__ __forceinline__ void tk_store8(void* p, int64_t i, int n, const float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) store_from_f32(p, i + k, DT, v[k]);
}

__device__ __forceinline__ double wave_sum(double x) {
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// Sum of N numbers of every thread, in an order that does not vary; the result is in every thread.
template <int N, int BLK>
__device__ __forceinline__ void block_sum(double (&x)[N], double (&part)[BLK / 64][N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = wave_sum(x[i]);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
    for (int i = 0; i < N; ++i) part[threadIdx.x >> 6][i] = x[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = 0.0;
    for (int w = 0; w < BLK / 64; ++w) x[i] += part[w][i];
  }
}
template <int BLK>
__device__ __forceinline__ double block_max(double x, double (&part)[BLK / 64]) {
  for (int off = 32; off > 0; off >>= 1) x = fmax(x, __shfl_xor(x, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  x = part[0];
  for (int w = 1; w < BLK / 64; ++w) x = fmax(x, part[w]);
  return x;
}

// Marks the row's listed ids; in every thread 1 if some are, 3 if one is listed twice.
template <int BLK>
__device__ __forceinline__ int mark_listed(const TopKlArgs& a, int64_t r, uint32_t* bits) {
  for (int64_t i = threadIdx.x; i < a.vocab / 32 + 1; i += BLK) bits[i] = 0;
  __syncthreads();
  int any = 0, twice = 0;
  for (int k = threadIdx.x; k < a.k; k += BLK) {
    const int64_t id = tk_id(a, r * a.k + k);
    if (id < 0) continue;
    any = 1;
    twice |= atomicOr(&bits[id / 32], 1u << (id % 32)) >> (id % 32) & 1;
  }
  any = __syncthreads_or(any) ? 1 : 0;
  return any | (__syncthreads_or(twice) ? 2 : 0);
}

// The marks of 8 tokens from i on.
__device__ __forceinline__ uint32_t marks8(const uint32_t* bits, int64_t i) {
  return static_cast<uint32_t>((static_cast<uint64_t>(bits[i / 32 + 1]) << 32 | bits[i / 32]) >> (i % 32)) & 255u;
}

template <int DT>
__global__ void __launch_bounds__(kTkBlock) top_kl_kernel(TopKlArgs a, double* __restrict__ stats,
                                                          double* __restrict__ row_kl) {
  extern __shared__ uint32_t bits[];  // vocab / 32 + 2 words
  __shared__ double part5[kTkBlock / 64][5];
  __shared__ double part1[kTkBlock / 64];
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  RowStats st{};
  if (a.weights && a.weights[r] == 0.0f) {
    if (t == 0) row_kl[r] = 0.0;
    return;
  }
  const int64_t base = (r / a.inner) * a.s0 + (r % a.inner) * a.s1;
  if (t == 0) bits[a.vocab / 32 + 1] = 0;
  const int marked = mark_listed<kTkBlock>(a, r, bits);
  if (!marked) {  // a row without entries adds nothing
    if (t == 0) {
      row_kl[r] = 0.0;
      *reinterpret_cast<RowStats*>(stats + r * kTkStats) = st;
    }
    return;
  }
  st.twice = marked >> 1;
  // the unlisted tokens: running maximum and sum of exponentials
  const float c = static_cast<float>(a.inv_t * 1.4426950408889634);
  float m = kTkLow, sum = 0.0f;
  for (int64_t i = t * 8; i < a.vocab; i += kTkBlock * 8) {
    const int n = a.vocab - i < 8 ? static_cast<int>(a.vocab - i) : 8;
    float v[8];
    tk_load8<DT>(a.s, base + i, n, v);
    const uint32_t out = marks8(bits, i);
    float top = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (out >> k & 1) v[k] = -INFINITY;
      top = fmaxf(top, v[k]);
    }
    if (top > m) {
      sum *= __builtin_amdgcn_exp2f((m - top) * c);
      m = top;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += __builtin_amdgcn_exp2f((v[k] - m) * c);
  }
  // the listed ones, and the teacher's side
  double bm = -INFINITY, am = -INFINITY;
  for (int k = t; k < a.k; k += kTkBlock) {
    const int64_t id = tk_id(a, r * a.k + k);
    if (id < 0) continue;
    bm = fmax(bm, load_as_f32(a.values, r * a.k + k, a.vdt) * a.inv_t);
    am = fmax(am, static_cast<double>(load_as_f32(a.s, base + id, DT)));
  }
  const double top = block_max<kTkBlock>(fmax(am, m), part1);
  if (!a.lse) bm = block_max<kTkBlock>(bm, part1);
  double x[5] = {0.0, 0.0, 0.0, 0.0, 0.0};  // sum e, sum e (b - N0), sum e a, exponentials of the listed, of the rest
  const double n0 = a.lse ? static_cast<double>(a.lse[r]) : bm;
  for (int k = t; k < a.k; k += kTkBlock) {
    const int64_t id = tk_id(a, r * a.k + k);
    if (id < 0) continue;
    const double b = load_as_f32(a.values, r * a.k + k, a.vdt) * a.inv_t;
    const double s = load_as_f32(a.s, base + id, DT);
    const double e = n0 == -INFINITY ? 0.0 : exp(b - n0);
    if (!(e <= 0.0)) {
      x[0] += e;
      x[1] += e * (b - n0);
      x[2] += e * (s * a.inv_t);
    }
    bool first = true;
    if (st.twice != 0.0)
      for (int j = 0; j < k && first; ++j) first = tk_id(a, r * a.k + j) != id;
    if (first) x[3] += s == -INFINITY ? 0.0 : exp((s - top) * a.inv_t);
  }
  x[4] = sum == 0.0f ? 0.0 : static_cast<double>(sum) * exp((static_cast<double>(m) - top) * a.inv_t);
  block_sum<5, kTkBlock>(x, part5);
  if (t != 0) return;
  st.z = top * a.inv_t + log(x[3] + x[4]);
  st.zr = top * a.inv_t + log(x[4]);
  double kl = 0.0;
  if (a.lse) {
    st.n = n0;
    st.r = x[0] > 1.0 ? 0.0 : 1.0 - x[0];
    int64_t listed = 0;  // with nothing left to hold the rest there is none
    if (a.k >= a.vocab)
      for (int64_t i = 0; i <= a.vocab / 32; ++i) listed += __popc(bits[i]);
    if (listed >= a.vocab) st.r = 0.0;
    st.p = x[0] + st.r;
    kl = x[1] - x[2] + x[0] * st.z;
    if (st.r != 0.0) kl += st.r * (log(st.r) - (st.zr - st.z));
  } else if (x[0] != 0.0) {
    st.n = n0 + log(x[0]);
    st.p = 1.0;
    kl = (x[1] - x[2]) / x[0] - log(x[0]) + st.z;
  }
  row_kl[r] = kl;
  *reinterpret_cast<RowStats*>(stats + r * kTkStats) = st;
}

constexpr int kTkFinal = 1024;

// loss = T^2 sum w KL / sum w; norm = T / sum w (0 where nothing has weight).
__global__ void __launch_bounds__(kTkFinal) top_kl_final_kernel(const double* __restrict__ row_kl,
                                                                const float* __restrict__ weights, int64_t rows,
                                                                double temperature, float* __restrict__ loss,
                                                                double* __restrict__ norm) {
  __shared__ double part[kTkFinal / 64][2];
  double x[2] = {0.0, 0.0};
  for (int64_t i = threadIdx.x; i < rows; i += kTkFinal) {
    const double w = weights ? static_cast<double>(weights[i]) : 1.0;
    if (w == 0.0) continue;
    x[0] += w;
    x[1] += w * row_kl[i];
  }
  block_sum<2, kTkFinal>(x, part);
  if (threadIdx.x != 0) return;
  *norm = x[0] == 0.0 ? 0.0 : temperature / x[0];
  *loss = x[0] == 0.0 ? 0.0f : static_cast<float>(temperature * temperature * (x[1] / x[0]));
}

__global__ void __launch_bounds__(kTkFinal) top_kl_dot_kernel(const double* __restrict__ row_dot, int64_t rows,
                                                              float* __restrict__ dot) {
  __shared__ double part[kTkFinal / 64][1];
  double x[1] = {0.0};
  for (int64_t i = threadIdx.x; i < rows; i += kTkFinal) x[0] += row_dot[i];
  block_sum<1, kTkFinal>(x, part);
  if (threadIdx.x == 0) *dot = static_cast<float>(x[0]);
}

// What the gradient of a row needs of its sums: coefficients in f32 and Z in two parts, in the logits' units, so that
// (s - hi) c - lo has the rounding of the difference only.
struct RowGrad {
  double factor;  // dL/da scale: g w T / sum w, of the logits: dL/ds
  float hi, lo, c;
  __device__ __forceinline__ RowGrad(const TopKlArgs& a, const RowStats& st, double f) : factor(f) {
    const double z = st.z / a.inv_t;
    hi = static_cast<float>(z);
    lo = static_cast<float>((z - static_cast<double>(hi)) * a.inv_t * 1.4426950408889634);
    c = static_cast<float>(a.inv_t * 1.4426950408889634);
  }
  __device__ __forceinline__ float q(float s) const { return __builtin_amdgcn_exp2f(fmaf(s - hi, c, -lo)); }
};

// Probability that the row's record gives to the id of entry k: p_k, and those of entries with the same id.
__device__ __forceinline__ double listed_p(const TopKlArgs& a, const RowStats& st, int64_t r, int k, int64_t id) {
  if (st.twice == 0.0) return exp(load_as_f32(a.values, r * a.k + k, a.vdt) * a.inv_t - st.n);
  double p = 0.0;
  for (int j = 0; j < a.k; ++j)
    if (tk_id(a, r * a.k + j) == id) p += exp(load_as_f32(a.values, r * a.k + j, a.vdt) * a.inv_t - st.n);
  return p;
}

template <int DT>
__global__ void __launch_bounds__(kTkBlock) top_kl_backward_kernel(TopKlArgs a, const double* __restrict__ stats,
                                                                   const double* __restrict__ norm,
                                                                   const float* __restrict__ grad_out,
                                                                   void* __restrict__ gs) {
  const int64_t r = blockIdx.x, out = r * a.vocab;
  const int t = threadIdx.x;
  const double w = a.weights ? static_cast<double>(a.weights[r]) : 1.0, f = *norm * w * static_cast<double>(*grad_out);
  RowStats st{};
  if (w != 0.0) st = *reinterpret_cast<const RowStats*>(stats + r * kTkStats);
  if (f == 0.0 || st.p == 0.0) {
    const float zero[8] = {};
    for (int64_t i = t * 8; i < a.vocab; i += kTkBlock * 8)
      tk_store8<DT>(gs, out + i, a.vocab - i < 8 ? static_cast<int>(a.vocab - i) : 8, zero);
    return;
  }
  const int64_t base = (r / a.inner) * a.s0 + (r % a.inner) * a.s1;
  const RowGrad g(a, st, f);
  const float coef = static_cast<float>(f * (st.p - (st.r != 0.0 ? st.r * exp(st.z - st.zr) : 0.0)));
  for (int64_t i = t * 8; i < a.vocab; i += kTkBlock * 8) {
    const int n = a.vocab - i < 8 ? static_cast<int>(a.vocab - i) : 8;
    float v[8];
    tk_load8<DT>(a.s, base + i, n, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = coef * g.q(v[k]);
    tk_store8<DT>(gs, out + i, n, v);
  }
  __syncthreads();  // the listed tokens are written again, with their own gradient
  for (int k = t; k < a.k; k += kTkBlock) {
    const int64_t id = tk_id(a, r * a.k + k);
    if (id < 0) continue;
    const double q = exp(load_as_f32(a.s, base + id, DT) * a.inv_t - st.z);
    store_from_f32(gs, out + id, DT, static_cast<float>(f * (st.p * q - listed_p(a, st, r, k, id))));
  }
}

// Along u (rows contiguous): h_j, and the row's u . dL/ds at an upstream gradient of 1.
template <int DT>
__global__ void __launch_bounds__(kTkBlock) top_kl_second_kernel(TopKlArgs a, const double* __restrict__ stats,
                                                                 const double* __restrict__ norm,
                                                                 const float* __restrict__ grad_out,
                                                                 const void* __restrict__ u, void* __restrict__ hs,
                                                                 double* __restrict__ row_dot) {
  extern __shared__ uint32_t bits[];
  __shared__ double part[kTkBlock / 64][3];
  const int64_t r = blockIdx.x, out = r * a.vocab;
  const int t = threadIdx.x;
  const double share = *norm * (a.weights ? static_cast<double>(a.weights[r]) : 1.0);
  RowStats st{};
  if (share != 0.0) st = *reinterpret_cast<const RowStats*>(stats + r * kTkStats);
  if (share == 0.0 || st.p == 0.0) {
    const float zero[8] = {};
    for (int64_t i = t * 8; i < a.vocab; i += kTkBlock * 8)
      tk_store8<DT>(hs, out + i, a.vocab - i < 8 ? static_cast<int>(a.vocab - i) : 8, zero);
    if (t == 0) row_dot[r] = 0.0;
    return;
  }
  const double f = share * static_cast<double>(*grad_out) * a.inv_t;
  const int64_t base = (r / a.inner) * a.s0 + (r % a.inner) * a.s1;
  const RowGrad g(a, st, f);
  if (t == 0) bits[a.vocab / 32 + 1] = 0;
  mark_listed<kTkBlock>(a, r, bits);
  float rest = 0.0f;
  for (int64_t i = t * 8; i < a.vocab; i += kTkBlock * 8) {
    const int n = a.vocab - i < 8 ? static_cast<int>(a.vocab - i) : 8;
    float v[8], w[8];
    tk_load8<DT>(a.s, base + i, n, v);
    tk_load8<DT>(u, out + i, n, w);
    const uint32_t skip = marks8(bits, i);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n && !(skip >> k & 1)) rest = fmaf(w[k], g.q(v[k]), rest);
  }
  double x[3] = {static_cast<double>(rest), 0.0, 0.0};  // u . q unlisted, listed; u . p
  for (int k = t; k < a.k; k += kTkBlock) {
    const int64_t id = tk_id(a, r * a.k + k);
    if (id < 0) continue;
    const double w = load_as_f32(u, out + id, DT);
    x[2] += w * exp(load_as_f32(a.values, r * a.k + k, a.vdt) * a.inv_t - st.n);
    bool first = true;
    if (st.twice != 0.0)
      for (int j = 0; j < k && first; ++j) first = tk_id(a, r * a.k + j) != id;
    if (first) x[1] += w * exp(load_as_f32(a.s, base + id, DT) * a.inv_t - st.z);
  }
  block_sum<3, kTkBlock>(x, part);
  const double kappa = st.r != 0.0 ? exp(st.z - st.zr) : 0.0, uq = x[0] + x[1];
  if (t == 0) row_dot[r] = share * (st.p * uq - x[2] - st.r * kappa * x[0]);
  const float A = static_cast<float>(f * (st.p - st.r * kappa));
  const float B = static_cast<float>(f * (st.p * uq - st.r * kappa * kappa * x[0]));
  for (int64_t i = t * 8; i < a.vocab; i += kTkBlock * 8) {
    const int n = a.vocab - i < 8 ? static_cast<int>(a.vocab - i) : 8;
    float v[8], w[8];
    tk_load8<DT>(a.s, base + i, n, v);
    tk_load8<DT>(u, out + i, n, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = g.q(v[k]) * fmaf(A, w[k], -B);
    tk_store8<DT>(hs, out + i, n, v);
  }
  __syncthreads();
  for (int k = t; k < a.k; k += kTkBlock) {
    const int64_t id = tk_id(a, r * a.k + k);
    if (id < 0) continue;
    const double q = exp(load_as_f32(a.s, base + id, DT) * a.inv_t - st.z);
    const double w = load_as_f32(u, out + id, DT);
    store_from_f32(hs, out + id, DT, static_cast<float>(f * st.p * q * (w - uq)));
  }
}

int top_kl_args(const sf_top_kl_desc* desc, const char* what, TopKlArgs& a) {
  SF_CHECK_ARG(desc, "%s: null descriptor", what);
  const sf_top_kl_desc& d = *desc;
  SF_CHECK_ARG((d.dtype == SF_DTYPE_F32 || d.dtype == SF_DTYPE_BF16) &&
                   (d.value_dtype == SF_DTYPE_F32 || d.value_dtype == SF_DTYPE_BF16),
               "%s: unknown dtype %d / %d", what, d.dtype, d.value_dtype);
  SF_CHECK_ARG(d.rows > 0 && d.rows < (1ll << 31) && d.vocab > 0 && d.vocab <= SF_TOP_MAX_VOCAB,
               "%s: %lld rows of %lld (at most %d)", what, (long long)d.rows, (long long)d.vocab, SF_TOP_MAX_VOCAB);
  SF_CHECK_ARG(d.inner > 0 && d.rows % d.inner == 0 && d.outer_stride >= 0 && d.row_stride >= 0,
               "%s: rows in groups of %lld, strides %lld, %lld", what, (long long)d.inner, (long long)d.outer_stride,
               (long long)d.row_stride);
  SF_CHECK_ARG(d.k >= 0 && d.k <= d.vocab, "%s: %lld entries of %lld", what, (long long)d.k, (long long)d.vocab);
  SF_CHECK_ARG(d.id_bytes == 4 || d.id_bytes == 8, "%s: ids must be int32 or int64", what);
  SF_CHECK_ARG(d.logits && ((d.values && d.ids) || d.k == 0) && d.stats && d.norm, "%s: null pointer", what);
  SF_CHECK_ARG(d.temperature > 0.0f && d.temperature <= 3.0e38f, "%s: temperature %g", what, d.temperature);
  a.s = d.logits, a.s0 = d.outer_stride, a.s1 = d.row_stride, a.inner = d.inner;
  a.values = d.values, a.ids = d.ids, a.lse = d.lse, a.weights = d.weights;
  a.vocab = d.vocab, a.k = static_cast<int>(d.k), a.vdt = d.value_dtype, a.id_bytes = d.id_bytes;
  a.inv_t = 1.0 / static_cast<double>(d.temperature);
  return SF_OK;
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" size_t sf_top_kl_stats_size(int64_t rows) {
  return rows > 0 ? static_cast<size_t>(rows) * kTkStats * sizeof(double) : 0;
}
extern "C" size_t sf_top_kl_workspace_size(int64_t rows) {
  return rows > 0 ? static_cast<size_t>(rows) * sizeof(double) : 0;
}

extern "C" int sf_top_kl_forward(const sf_top_kl_desc* desc, float* loss, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  TopKlArgs a;
  if (int rc = top_kl_args(desc, "sf_top_kl_forward", a)) return rc;
  SF_CHECK_ARG(loss, "sf_top_kl_forward: null pointer");
  SF_CHECK_ARG(workspace && workspace_bytes >= sf_top_kl_workspace_size(desc->rows),
               "sf_top_kl_forward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(desc->rows));
  const size_t lds = (static_cast<size_t>(a.vocab) / 32 + 2) * 4;
  double* row_kl = static_cast<double*>(workspace);
  if (desc->dtype == SF_DTYPE_F32)
    top_kl_kernel<SF_DTYPE_F32><<<grid, kTkBlock, lds, st>>>(a, desc->stats, row_kl);
  else
    top_kl_kernel<SF_DTYPE_BF16><<<grid, kTkBlock, lds, st>>>(a, desc->stats, row_kl);
  top_kl_final_kernel<<<1, kTkFinal, 0, st>>>(row_kl, a.weights, desc->rows, desc->temperature, loss, desc->norm);
  return launch_status("sf_top_kl_forward");
}

extern "C" int sf_top_kl_backward(const sf_top_kl_desc* desc, const float* grad_out, void* grad_logits, void* stream) {
  TopKlArgs a;
  if (int rc = top_kl_args(desc, "sf_top_kl_backward", a)) return rc;
  SF_CHECK_ARG(grad_out && grad_logits, "sf_top_kl_backward: null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(desc->rows));
  if (desc->dtype == SF_DTYPE_F32)
    top_kl_backward_kernel<SF_DTYPE_F32><<<grid, kTkBlock, 0, st>>>(a, desc->stats, desc->norm, grad_out, grad_logits);
  else
    top_kl_backward_kernel<SF_DTYPE_BF16><<<grid, kTkBlock, 0, st>>>(a, desc->stats, desc->norm, grad_out, grad_logits);
  return launch_status("sf_top_kl_backward");
}

extern "C" int sf_top_kl_double_backward(const sf_top_kl_desc* desc, const float* grad_out, const void* grad_grad,
                                         void* grad2_logits, float* dot, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  TopKlArgs a;
  if (int rc = top_kl_args(desc, "sf_top_kl_double_backward", a)) return rc;
  SF_CHECK_ARG(grad_out && grad_grad && grad2_logits, "sf_top_kl_double_backward: null pointer");
  SF_CHECK_ARG(workspace && workspace_bytes >= sf_top_kl_workspace_size(desc->rows),
               "sf_top_kl_double_backward: workspace too small");
  double* row_dot = static_cast<double*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(desc->rows));
  const size_t lds = (static_cast<size_t>(a.vocab) / 32 + 2) * 4;
  if (desc->dtype == SF_DTYPE_F32)
    top_kl_second_kernel<SF_DTYPE_F32><<<grid, kTkBlock, lds, st>>>(a, desc->stats, desc->norm, grad_out, grad_grad,
                                                                    grad2_logits, row_dot);
  else
    top_kl_second_kernel<SF_DTYPE_BF16><<<grid, kTkBlock, lds, st>>>(a, desc->stats, desc->norm, grad_out, grad_grad,
                                                                     grad2_logits, row_dot);
  if (dot) top_kl_dot_kernel<<<1, kTkFinal, 0, st>>>(row_dot, desc->rows, dot);
  return launch_status("sf_top_kl_double_backward");
}
