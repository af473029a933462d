// Distillation from a teacher's recorded top logits: KL of a student's whole softmax from the listed tokens (and, with
// the teacher's log-sum-exp, from the rest taken together), its gradient, and the product of its second derivative with a
// direction.  At temperature T, for a row with listed ids i_k, teacher logits t_k, student logits s over the vocabulary:
//   a = s / T,  Z = log sum_V exp a_j,  q_j = exp(a_j - Z),  b_k = t_k / T,  p_k = exp(b_k - N)
//   N = log sum_k exp b_k (then the row is renormalised, r = 0), or the given lse (then r = 1 - sum p, not below 0)
//   KL = sum_k p_k (log p_k - log q_(i_k)) + r (log r - log q_rest),   q_rest = sum over unlisted j of q_j
//   dKL/da_j = P q_j - p_j - r q_j / q_rest [j unlisted],              P = sum p + r
// With Z_r the log-sum-exp of the unlisted tokens, rho_j = exp(a_j - Z_r) and G = exp(Z_r - Z) the gradient of an unlisted
// token is (P G - r) rho_j: one exponential, and no factor above 1, however little probability the rest has (of q_j and exp(Z -
// Z_r) float32 holds neither from a gap of 88 on).  Its derivative along u: with U = sum u_j q_j over the vocabulary and U_r =
// sum u_j rho_j over the unlisted,
//   h_j = rho_j ((P G - r) u_j - (P G U - r U_r))  [unlisted],   P q_j (u_j - U)  [listed].
// The rest's sums are formed without the listed tokens (one bit for each of the vocabulary in LDS), not as a difference, and
// from the rest's own maximum.
//
// One workgroup per row streams it once forward and once backward (twice along u); listed tokens are gathered and handled
// in f64 while the row is on its way.  Row sums are f32 exponentials in compensated sums, joined in f64; stats and losses
// are f64.  Bound by memory: forward and backward by turns 4096 x 32000 bf16, k 64, 143 us (two reads and a write of 262
// MB: 5.5 TB/s, what a copy reaches), 2048 x 131072 333 (4.8 TB/s; with a fifth of the rows of weight 0, whose zeros are
// written alone, 270), 2046 x 50257 f32 with rows of odd alignment 248 (5.0 TB/s; 202 with three rows in ten of weight 0);
// along u 1024 x 32000 46 (two rows read, one written, 4.3 TB/s).  64 x 32000 forward 7 us and 3 for the sum over the rows.
// Two products of log-softmax over the vocabulary, as the formula stands, take ten passes and more.
#include <type_traits>

#include "sf_top.hpp"

namespace sf {
namespace {

// Pieces of a row that a thread loads before it uses them: bytes on their way against registers.  Forward and backward by
// turns, us: 4096 x 32000 bf16 142 with 3 and 4 pieces, 146 with 2 and 2; 2046 x 50257 f32, whose pieces are twice as
// long, three rows in ten of weight 0, 212 and 202.
template <int DT>
constexpr int kTkForwardU = DT == SF_DTYPE_BF16 ? 3 : 2;
template <int DT>
constexpr int kTkBackwardU = DT == SF_DTYPE_BF16 ? 4 : 2;
constexpr int kTkSecond = 512;
constexpr int kTkStats = 9;  // f64 of a row's RowStats

struct TopKlArgs {
  const void* s;
  int64_t s0, s1, inner;  // row r lies at (r / inner) s0 + (r % inner) s1
  const void* values;
  const void* ids;
  const float* lse;      // null: renormalised
  const float* weights;  // null: all 1
  int vocab;
  int k, vdt, id_bytes;
  double inv_t;
};

// What the backward needs of a row.  Z = top / T + lz and Z_r = rest_top / T + lzr, N = nb + ln: in two parts, so that rows of
// huge logits (all at the type's lowest value, say) keep their differences.
struct RowStats {
  double top, lz, rest_top, lzr;
  double nb, ln;
  double p, r;
  double twice;  // an id is listed more than once
};
static_assert(sizeof(RowStats) == kTkStats * sizeof(double), "stats of a row");

// Z_r - Z
__device__ __forceinline__ double rest_gap(const TopKlArgs& a, const RowStats& st) {
  return (st.rest_top - st.top) * a.inv_t + (st.lzr - st.lz);
}

// Words of a row's marks.
__host__ __device__ __forceinline__ int mark_words(int vocab) { return (vocab + 8) / 32 + 1; }

__device__ __forceinline__ int tk_id(const TopKlArgs& a, int64_t at) {
  const int64_t id = a.id_bytes == 8 ? static_cast<const int64_t*>(a.ids)[at] : static_cast<const int32_t*>(a.ids)[at];
  return id >= 0 && id < a.vocab ? static_cast<int>(id) : -1;
}

// PAST: past the caches.
template <int DT, bool PAST>
__device__ __forceinline__ void tk_store8(void* row, int i, int n, const float (&v)[8]) {
  typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
  if (n == 8) {
    u32x4u* to = reinterpret_cast<u32x4u*>(static_cast<char*>(row) +
                                           static_cast<int64_t>(i) * (DT == SF_DTYPE_BF16 ? 2 : 4));
    const auto put = [](u32x4u* q, const u32x4u& w) {
      if constexpr (PAST)
        __builtin_nontemporal_store(w, q);
      else
        *q = w;
    };
    if constexpr (DT == SF_DTYPE_BF16) {
      const auto two = [&](int k) {
        return static_cast<uint32_t>(f32_to_bf16(v[k])) | static_cast<uint32_t>(f32_to_bf16(v[k + 1])) << 16;
      };
      put(to, u32x4u{two(0), two(2), two(4), two(6)});
    } else {
#pragma unroll
      for (int k = 0; k < 8; k += 4)
        put(to + k / 4, u32x4u{__float_as_uint(v[k]), __float_as_uint(v[k + 1]), __float_as_uint(v[k + 2]),
                               __float_as_uint(v[k + 3])});
    }
  } else {
    for (int k = 0; k < n; ++k) store_from_f32(row, i + k, DT, v[k]);
  }
}

// How a row is cut: `head` tokens before its first 16-byte boundary, pieces of 8, and the last few.  Thread t takes pieces
// t, t + BLK, ..; n of them; the last threads take the odd tokens.
struct Cut {
  int vocab, head, n;
  template <int DT, int BLK>
  static __device__ __forceinline__ Cut of(const void* row, int vocab) {
    constexpr int kBytes = DT == SF_DTYPE_BF16 ? 2 : 4;
    Cut c;
    c.vocab = vocab;
    c.head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16) / kBytes;
    if (c.head > vocab) c.head = vocab;
    const int pieces = (vocab - c.head) / 8, t = threadIdx.x;
    c.n = pieces > t ? (pieces - t - 1) / BLK + 1 : 0;
    return c;
  }
  template <int BLK>
  __device__ __forceinline__ int at(int p) const {
    return head + (static_cast<int>(threadIdx.x) + p * BLK) * 8;
  }
  // Place of a token's mark: a piece's marks are a byte.
  __device__ __forceinline__ int mark(int id) const { return id + 8 - head; }
};

// f(first id, number of elements, elements of each of N rows) over the odd tokens; what is missing of 8 is -inf.
template <int DT, int BLK, int N, typename F>
__device__ __forceinline__ void tk_odd(const void* const (&rows)[N], const Cut& c, F&& f) {
  const int done = c.head + (c.vocab - c.head) / 8 * 8, t = threadIdx.x;
  const int i = t == BLK - 1 ? 0 : done, n = t == BLK - 1 ? c.head : t == BLK - 2 ? c.vocab - done : 0;
  if (n == 0) return;
  float v[N][8];
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) v[j][k] = k < n ? load_as_f32(rows[j], i + k, DT) : -INFINITY;
  f(i, n, v);
}

// The same over the pieces from piece `from` of each thread on, and the odd tokens: U pieces are loaded before the first
// is used; before() runs, in every thread, between the first loads and their use.
template <int DT, int BLK, int U, int N, typename B, typename F>
__device__ __forceinline__ void tk_stream(const void* const (&rows)[N], const Cut& c, int from, B&& before, F&& f) {
  Raw8<DT> raw[U][N];
  float v[N][8];
  const auto load = [&](int p) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u < c.n)
#pragma unroll
        for (int j = 0; j < N; ++j) raw[u][j].load(rows[j], c.at<BLK>(p + u));
  };
  load(from);
  before();
  for (int p = from; p < c.n; p += U) {
    if (p > from) load(p);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u < c.n) {
#pragma unroll
        for (int j = 0; j < N; ++j) raw[u][j].get(v[j]);
        f(c.at<BLK>(p + u), 8, v);
      }
  }
  tk_odd<DT, BLK>(rows, c, f);
}

template <int DT>
__device__ __forceinline__ const void* row_at(const void* p, int64_t at) {
  return static_cast<const char*>(p) + at * (DT == SF_DTYPE_BF16 ? 2 : 4);
}

// Sums of N numbers over groups of W lanes, and maxima.
template <int W = 64, int N>
__device__ __forceinline__ void lanes_sum(double (&x)[N]) {
#pragma unroll
  for (int off = W / 2; off > 0; off >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += __shfl_xor(x[i], off, 64);
}
template <int W = 64, int N>
__device__ __forceinline__ void lanes_max(double (&x)[N]) {
#pragma unroll
  for (int off = W / 2; off > 0; off >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = fmax(x[i], __shfl_xor(x[i], off, 64));
}

// Sum of N numbers of every thread, in an order that does not vary; the result is in every thread.
template <int N, int BLK>
__device__ __forceinline__ void block_sum(double (&x)[N], double (&part)[BLK / 64][N]) {
  lanes_sum(x);
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
// Marks the row's listed ids in bits that are 0; per wave in flags: 1 if some are listed, 3 if one was marked already.
template <int BLK>
__device__ __forceinline__ void mark_listed(const TopKlArgs& a, int64_t r, const Cut& c, uint32_t* bits, int* flags) {
  int any = 0, twice = 0;
  for (int k = threadIdx.x; k < a.k; k += BLK) {
    const int id = tk_id(a, r * a.k + k);
    if (id < 0) continue;
    any = 1;
    const int at = c.mark(id);
    twice |= atomicOr(&bits[at / 32], 1u << (at % 32)) >> (at % 32) & 1;
  }
  const int f = (__ballot(any) ? 1 : 0) | (__ballot(twice) ? 2 : 0);
  if ((threadIdx.x & 63) == 0) flags[threadIdx.x >> 6] = f;
}
template <int BLK>
__device__ __forceinline__ int all_flags(const int* flags) {
  int f = 0;
  for (int w = 0; w < BLK / 64; ++w) f |= flags[w];
  return f;
}

// The marks of the up to 8 tokens from i on: of a piece, or of the odd ones.
__device__ __forceinline__ uint32_t marks8(const uint32_t* bits, const Cut& c, int i) {
  const int at = c.mark(i);
  return reinterpret_cast<const uint8_t*>(bits)[at / 8] >> (at % 8);
}

// Whether entry k of the row is the first with its id.
__device__ __forceinline__ bool first_of_id(const TopKlArgs& a, int64_t r, int k, int id) {
  for (int j = 0; j < k; ++j)
    if (tk_id(a, r * a.k + j) == id) return false;
  return true;
}

// What a wave finds of a row.
struct WavePart {
  double nb, e0, e1, e2;  // listed: sums of e = exp(b - nb), of e (b - nb), of e (s - ml)
  double ml, sl;          // listed students: maximum and sum of exponentials
  float m, sum;           // tokens of the stream: maximum and sum of exponentials
};

// exp((x - top) / T) for sums whose maximum is top; nothing counts 0.
__device__ __forceinline__ double exp_from(double x, double top, double inv_t) {
  return x == -INFINITY ? 0.0 : exp((x - top) * inv_t);
}

// REST: with the teacher's log-sum-exp; the stream then leaves out the listed tokens.
template <int DT, int BLK, bool REST>
__global__ void __launch_bounds__(BLK) top_kl_kernel(TopKlArgs a, double* __restrict__ stats,
                                                     double* __restrict__ row_kl) {
  extern __shared__ uint32_t bits[];  // mark_words(vocab)
  __shared__ WavePart parts[BLK / 64];
  __shared__ int flags[BLK / 64];
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  if (a.weights && a.weights[r] == 0.0f) {
    if (t == 0) row_kl[r] = 0.0;
    return;
  }
  const void* rows[1] = {row_at<DT>(a.s, (r / a.inner) * a.s0 + (r % a.inner) * a.s1)};
  const Cut cut = Cut::of<DT, BLK>(rows[0], a.vocab);
  const float c = static_cast<float>(a.inv_t * 1.4426950408889634);
  float m = kTopLow, sum = 0.0f, lost = 0.0f;
  WavePart part{REST ? static_cast<double>(a.lse[r]) : -INFINITY, 0.0, 0.0, 0.0, -INFINITY, 0.0, 0.0f, 0.0f};
  // The row's first loads are on their way while the listed tokens are marked and summed: the latter by the waves that
  // have some, each with its own maxima, so that no wave waits for another before the row's end.
  const auto listed = [&] {
    for (int i = t; i < mark_words(a.vocab); i += BLK) bits[i] = 0;
    __syncthreads();
    mark_listed<BLK>(a, r, cut, bits, flags);
    __syncthreads();
    if (wave * 64 >= a.k) return;
    const bool twice = all_flags<BLK>(flags) & 2;
    for (int k = t; k < a.k; k += BLK) {
      const int id = tk_id(a, r * a.k + k);
      if (id < 0) continue;
      if (!REST) part.nb = fmax(part.nb, load_as_f32(a.values, r * a.k + k, a.vdt) * a.inv_t);
      part.ml = fmax(part.ml, static_cast<double>(load_as_f32(rows[0], id, DT)));
    }
    double most[2] = {part.nb, part.ml};
    lanes_max(most);
    if (!REST) part.nb = most[0];
    part.ml = most[1];
    for (int k = t; k < a.k; k += BLK) {
      const int id = tk_id(a, r * a.k + k);
      if (id < 0) continue;
      const double b = load_as_f32(a.values, r * a.k + k, a.vdt) * a.inv_t, s = load_as_f32(rows[0], id, DT);
      const double e = !REST && b == -INFINITY ? 0.0 : exp(b - part.nb);  // NaN where b is, whatever the maximum says
      if (!(e <= 0.0)) {
        part.e0 += e;
        part.e1 += e * (b - part.nb);
        part.e2 += s == -INFINITY ? -INFINITY : e * (s - part.ml);
      }
      if (REST && (!twice || first_of_id(a, r, k, id))) part.sl += exp_from(s, part.ml, a.inv_t);
    }
    double x[4] = {part.e0, part.e1, part.e2, part.sl};
    lanes_sum(x);
    part.e0 = x[0], part.e1 = x[1], part.e2 = x[2], part.sl = x[3];
  };
  tk_stream<DT, BLK, kTkForwardU<DT>>(rows, cut, 0, listed, [&](int i, int, float (&x)[1][8]) {
    float(&v)[8] = x[0];
    float top = m;
    const uint32_t out = REST ? marks8(bits, cut, i) : 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (REST) {  // -inf where the bit is set
        const uint32_t mask = static_cast<uint32_t>(static_cast<int32_t>(out << (31 - k)) >> 31);
        v[k] = __uint_as_float((__float_as_uint(v[k]) & ~mask) | (mask & 0xff800000u));
      }
      top = fmaxf(top, v[k]);
    }
    if (top > m) {
      const float f = __builtin_amdgcn_exp2f((m - top) * c);
      sum *= f;
      lost *= f;
      m = top;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __builtin_amdgcn_exp2f((v[k] - m) * c);
    // hundreds of small terms beside a large one: what an addition rounds off is carried along
    const float add = (((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]))) - lost, upto = sum + add;
    lost = (upto - sum) - add;
    sum = upto;
  });
  part.m = m;
  for (int off = 32; off > 0; off >>= 1) part.m = fmaxf(part.m, __shfl_xor(part.m, off, 64));
  part.sum = sum == 0.0f ? 0.0f : sum * __builtin_amdgcn_exp2f((m - part.m) * c);
  for (int off = 32; off > 0; off >>= 1) part.sum += __shfl_xor(part.sum, off, 64);
  if (lane == 0) parts[wave] = part;
  __syncthreads();
  if (wave != 0) return;
  // the waves' parts, one to a lane
  constexpr int W = BLK / 64;
  part = parts[lane % W];
  double most[3] = {part.nb, part.ml, static_cast<double>(part.m)};
  lanes_max<W>(most);
  const double nb = most[0], rest_top = most[2], top = fmax(most[1], rest_top);
  if (part.e0 != 0.0) part.e2 += part.e0 * (part.ml == -INFINITY ? 0.0 : part.ml - top);
  if (!REST && part.nb != nb) {
    const double f = exp_from(part.nb, nb, 1.0), d = part.nb - nb, none = 0.0 * part.e0;  // 0, or NaN
    part.e1 = f == 0.0 ? none : f * (part.e1 + d * part.e0);
    part.e2 = f == 0.0 ? none : f * part.e2;
    part.e0 = f == 0.0 ? none : f * part.e0;
  }
  double x[5] = {part.e0, part.e1, part.e2,
                 part.sum == 0.0f ? 0.0 : part.sum * exp((static_cast<double>(part.m) - rest_top) * a.inv_t),
                 part.sl == 0.0 ? 0.0 : part.sl * exp_from(part.ml, top, a.inv_t)};
  lanes_sum<W>(x);
  const double e0 = x[0], e1 = x[1], e2 = x[2] * a.inv_t, rest = x[3];
  const double all = rest * exp((rest_top - top) * a.inv_t) + x[4];
  RowStats st{};
  if (REST) {
    st.r = e0 > 1.0 ? 0.0 : 1.0 - e0;
    if (a.k >= a.vocab) {  // with every token listed there is no rest
      int marked = 0;
      for (int i = lane; i < mark_words(a.vocab); i += 64) marked += __popc(bits[i]);
      for (int off = 32; off > 0; off >>= 1) marked += __shfl_xor(marked, off, 64);
      if (marked == a.vocab) st.r = 0.0;
    }
  }
  const double l = log(lane == 0 ? all : lane == 1 ? rest : REST ? st.r : e0);
  if (!REST && e0 != 0.0) st.p = 1.0;
  if (REST) st.p = e0 + st.r;
  st.top = top;
  st.rest_top = rest_top;
  st.lz = __shfl(l, 0, 64);
  st.lzr = __shfl(l, 1, 64);
  st.nb = nb;
  st.ln = REST ? 0.0 : __shfl(l, 2, 64);
  double kl;
  if (REST) {
    kl = e1 - e2 + e0 * st.lz;
    if (st.r != 0.0) kl += st.r * (__shfl(l, 2, 64) - rest_gap(a, st));
  } else {
    kl = e0 == 0.0 ? 0.0 : (e1 - e2) / e0 - st.ln + st.lz;
  }
  const int marked = all_flags<BLK>(flags);
  if (!marked) {  // a row without entries adds nothing
    st = RowStats{};
    kl = 0.0;
  }
  st.twice = marked >> 1;
  if (lane == 0) {
    row_kl[r] = kl;
    *reinterpret_cast<RowStats*>(stats + r * kTkStats) = st;
  }
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

// Of a row's unlisted tokens: with a rest rho = exp(s / T - Z_r) and `share` = G, else q = exp(s / T - Z) and 1.  The exponent
// in base 2, (s - top) c - lo, rounds in f32 by up to 2^-24 of itself: 1e-6 of q for a token of probability 1e-7, nothing
// beside bf16's 2^-9; for f32 its whole part is split off and what s - top and c round is carried along.  Of listed tokens it
// may be inf.
template <int DT>
struct RowGrad {
  double share;
  float hi, lo, c, c_lo, whole, part;  // lo = whole + part
  __device__ __forceinline__ RowGrad(const TopKlArgs& a, const RowStats& st) {
    const bool rest = st.r != 0.0;
    const double k = a.inv_t * 1.4426950408889634, l = (rest ? st.lzr : st.lz) * 1.4426950408889634;
    share = rest ? exp(rest_gap(a, st)) : 1.0;
    hi = static_cast<float>(rest ? st.rest_top : st.top);
    lo = static_cast<float>(l);
    c = static_cast<float>(k);
    c_lo = static_cast<float>(k - static_cast<double>(c));
    whole = static_cast<float>(rint(l));
    part = static_cast<float>(l - rint(l));
  }
  __device__ __forceinline__ float q(float s) const {
    const float d = s - hi;
    if constexpr (DT == SF_DTYPE_BF16) return __builtin_amdgcn_exp2f(fmaf(d, c, -lo));
    const float back = d - s;  // d + e = s - hi exactly
    const float e = (s - (d - back)) - (hi + back);
    const float n = rintf(d * c);
    const float f = fmaf(d, c, -n) + fmaf(e, c, fmaf(d, c_lo, -part));
    // below 2^-126 nothing is left to be exact about, and -inf has no parts
    return n - whole > -126.0f ? ldexpf(__builtin_amdgcn_exp2f(f), static_cast<int>(n - whole))
                               : __builtin_amdgcn_exp2f(fmaf(d, c, -lo));
  }
};

// The same in f64, and the listed probability of entry k's own value.
__device__ __forceinline__ double q_of(const TopKlArgs& a, const RowStats& st, float s) {
  return exp((static_cast<double>(s) - st.top) * a.inv_t - st.lz);
}
__device__ __forceinline__ double p_of(const TopKlArgs& a, const RowStats& st, int64_t at) {
  return exp((load_as_f32(a.values, at, a.vdt) * a.inv_t - st.nb) - st.ln);
}

// Probability that the row's record gives to the id of entry k: p_k, and those of entries with the same id.
__device__ __forceinline__ double listed_p(const TopKlArgs& a, const RowStats& st, int64_t r, int k, int id) {
  if (st.twice == 0.0) return p_of(a, st, r * a.k + k);
  double p = 0.0;
  for (int j = 0; j < a.k; ++j)
    if (tk_id(a, r * a.k + j) == id) p += p_of(a, st, r * a.k + j);
  return p;
}

template <int DT, int BLK, bool PAST>
__global__ void __launch_bounds__(BLK) top_kl_backward_kernel(TopKlArgs a, const double* __restrict__ stats,
                                                                   const double* __restrict__ norm,
                                                                   const float* __restrict__ grad_out,
                                                                   void* __restrict__ gs) {
  // from the last row on: the forward read these last, and the caches hold them
  const int64_t r = gridDim.x - 1 - blockIdx.x;
  const int t = threadIdx.x;
  void* out = const_cast<void*>(row_at<DT>(gs, r * a.vocab));
  const double w = a.weights ? static_cast<double>(a.weights[r]) : 1.0, f = *norm * w * static_cast<double>(*grad_out);
  RowStats st{};
  if (w != 0.0) st = *reinterpret_cast<const RowStats*>(stats + r * kTkStats);
  if (f == 0.0 || st.p == 0.0) {
    const float zero[8] = {};
    for (int i = t * 8; i < a.vocab; i += BLK * 8) tk_store8<DT, PAST>(out, i, a.vocab - i < 8 ? a.vocab - i : 8, zero);
    return;
  }
  const RowGrad<DT> g(a, st);
  const float coef = static_cast<float>(f * (st.p * g.share - st.r));
  const void* rows[1] = {row_at<DT>(a.s, (r / a.inner) * a.s0 + (r % a.inner) * a.s1)};
  const Cut cut = Cut::of<DT, BLK>(out, a.vocab);  // whole 16 bytes are written rather than read
  // the listed tokens' own gradient, formed while the row is on its way and written when the row is
  const auto listed = [&](int k, int id) {
    const double q = q_of(a, st, load_as_f32(rows[0], id, DT));
    return static_cast<float>(f * (st.p * q - listed_p(a, st, r, k, id)));
  };
  int id0 = -1;
  float g0 = 0.0f;
  const auto first = [&] {
    if (t < a.k) id0 = tk_id(a, r * a.k + t);
    if (id0 >= 0) g0 = listed(t, id0);
  };
  tk_stream<DT, BLK, kTkBackwardU<DT>>(rows, cut, 0, first, [&](int i, int n, float (&x)[1][8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[0][k] = coef * g.q(x[0][k]);
    tk_store8<DT, PAST>(out, i, n, x[0]);
  });
  __syncthreads();
  if (id0 >= 0) store_from_f32(out, id0, DT, g0);
  for (int k = t + BLK; k < a.k; k += BLK) {
    const int id = tk_id(a, r * a.k + k);
    if (id >= 0) store_from_f32(out, id, DT, listed(k, id));
  }
}

// Along u (rows contiguous): h_j, and the row's u . dL/ds at an upstream gradient of 1.  Of the pieces that both passes need
// the first H of a thread stay in registers: 4096 x 32000 bf16 167 us with 6, 185 with 2; 2046 x 50257 f32, three rows in
// ten of weight 0, 248 with 3, 259 with 1 (every row: 307 with 3).
template <int DT, bool PAST>
__global__ void __launch_bounds__(kTkSecond) top_kl_second_kernel(TopKlArgs a, const double* __restrict__ stats,
                                                                  const double* __restrict__ norm,
                                                                  const float* __restrict__ grad_out,
                                                                  const void* __restrict__ u, void* __restrict__ hs,
                                                                  double* __restrict__ row_dot) {
  constexpr int BLK = kTkSecond, H = DT == SF_DTYPE_BF16 ? 6 : 3;
  extern __shared__ uint32_t bits[];
  __shared__ double part[BLK / 64][3];
  __shared__ int flags[BLK / 64];
  const int64_t r = gridDim.x - 1 - blockIdx.x;
  const int t = threadIdx.x;
  void* out = const_cast<void*>(row_at<DT>(hs, r * a.vocab));
  const double w = a.weights ? static_cast<double>(a.weights[r]) : 1.0, share = *norm * w;
  RowStats st{};
  if (w != 0.0) st = *reinterpret_cast<const RowStats*>(stats + r * kTkStats);
  if (share == 0.0 || st.p == 0.0) {
    const float zero[8] = {};
    for (int i = t * 8; i < a.vocab; i += BLK * 8) tk_store8<DT, PAST>(out, i, a.vocab - i < 8 ? a.vocab - i : 8, zero);
    if (t == 0) row_dot[r] = 0.0;
    return;
  }
  const double f = share * static_cast<double>(*grad_out) * a.inv_t;
  const RowGrad<DT> g(a, st);
  const void* rows[2] = {row_at<DT>(a.s, (r / a.inner) * a.s0 + (r % a.inner) * a.s1), row_at<DT>(u, r * a.vocab)};
  const Cut cut = Cut::of<DT, BLK>(rows[0], a.vocab);
  Raw8<DT> raw[H][2];  // the thread's first pieces stay in registers
#pragma unroll
  for (int p = 0; p < H; ++p)
    if (p < cut.n) {
      raw[p][0].load(rows[0], cut.at<BLK>(p));
      raw[p][1].load(rows[1], cut.at<BLK>(p));
    }
  for (int i = t; i < mark_words(a.vocab); i += BLK) bits[i] = 0;
  __syncthreads();
  mark_listed<BLK>(a, r, cut, bits, flags);
  __syncthreads();
  // the listed tokens, while the row is on its way
  double x[3] = {0.0, 0.0, 0.0};  // u . rho unlisted (see RowGrad), u . q listed; u . p
  int id0 = -1;
  double q0 = 0.0, u0 = 0.0;
  for (int k = t; k < a.k; k += BLK) {
    const int id = tk_id(a, r * a.k + k);
    if (id < 0) continue;
    const double q = q_of(a, st, load_as_f32(rows[0], id, DT)), y = load_as_f32(rows[1], id, DT);
    if (k == t) id0 = id, q0 = q, u0 = y;
    x[2] += y * p_of(a, st, r * a.k + k);
    if (st.twice == 0.0 || first_of_id(a, r, k, id)) x[1] += y * q;
  }
  float rest = 0.0f;
  const auto dot = [&](int i, int m, float (&x)[2][8]) {
    const uint32_t skip = marks8(bits, cut, i);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < m && !(skip >> k & 1)) rest = fmaf(x[1][k], g.q(x[0][k]), rest);
  };
  const auto kept = [&](auto&& use) {
#pragma unroll
    for (int p = 0; p < H; ++p)
      if (p < cut.n) {
        float x[2][8];
        raw[p][0].get(x[0]);
        raw[p][1].get(x[1]);
        use(cut.at<BLK>(p), 8, x);
      }
  };
  kept(dot);
  tk_stream<DT, BLK, 1>(rows, cut, H, [] {}, dot);
  x[0] = static_cast<double>(rest);
  block_sum<3, BLK>(x, part);
  const double uq = g.share * x[0] + x[1];
  if (t == 0) row_dot[r] = share * (st.p * uq - x[2] - st.r * x[0]);
  const float A = static_cast<float>(f * (st.p * g.share - st.r));
  const float B = static_cast<float>(f * (st.p * g.share * uq - st.r * x[0]));
  const auto write = [&](int i, int m, float (&x)[2][8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[0][k] = g.q(x[0][k]) * fmaf(A, x[1][k], -B);
    tk_store8<DT, PAST>(out, i, m, x[0]);
  };
  kept(write);
  tk_stream<DT, BLK, 1>(rows, cut, H, [] {}, write);
  __syncthreads();
  if (id0 >= 0) store_from_f32(out, id0, DT, static_cast<float>(f * st.p * q0 * (u0 - uq)));
  for (int k = t + BLK; k < a.k; k += BLK) {
    const int id = tk_id(a, r * a.k + k);
    if (id < 0) continue;
    const double q = q_of(a, st, load_as_f32(rows[0], id, DT)), y = load_as_f32(rows[1], id, DT);
    store_from_f32(out, id, DT, static_cast<float>(f * st.p * q * (y - uq)));
  }
}

// With at most one row for each CU a row takes 1024 threads; with more, 256 forward and 512 backward, whose waits cover each
// other.  Forward and backward by turns, us: 64 x 32000 bf16 15.8 and 17.9, 256 x 50257 f32 35 and 39; 400 x 32000 bf16
// 30.6 and 26.3, 400 x 50257 f32 53 and 50, 4096 x 32000 bf16 193 and 143 (256 threads backward too: 150).
constexpr int64_t kTkFewRows = 256;

// launch(data type, whether what it writes passes the caches).  A gradient that the last-level cache (256 MB) does not hold
// beside the logits is not found there by who reads it next, and what of it stays there has to be written back while the
// next pass reads: forward and backward by turns, 4096 x 32000 bf16 143 us past the caches and 167 through them, 2048 x
// 131072, a fifth of the rows of weight 0, 270 and 314; 1024 x 32000 (66 MB) 45 and 43.
template <typename F>
void tk_dispatch(const sf_top_kl_desc& d, F&& launch) {
  const bool past = d.rows * d.vocab * (d.dtype == SF_DTYPE_F32 ? 4 : 2) > (128ll << 20);
  const auto with = [&](auto dt) {
    if (past)
      launch(dt, std::true_type{});
    else
      launch(dt, std::false_type{});
  };
  if (d.dtype == SF_DTYPE_F32)
    with(std::integral_constant<int, SF_DTYPE_F32>{});
  else
    with(std::integral_constant<int, SF_DTYPE_BF16>{});
}

int top_kl_args(const sf_top_kl_desc* desc, const char* what, TopKlArgs& a) {
  SF_CHECK_ARG(desc, "%s: null descriptor", what);
  const sf_top_kl_desc& d = *desc;
  SF_CHECK_ARG((d.dtype == SF_DTYPE_F32 || d.dtype == SF_DTYPE_BF16) &&
                   (d.value_dtype == SF_DTYPE_F32 || d.value_dtype == SF_DTYPE_BF16),
               "%s: unknown dtype %d / %d", what, d.dtype, d.value_dtype);
  SF_CHECK_ARG(d.rows > 0 && d.rows < SF_TOP_MAX_ROWS && d.vocab > 0 && d.vocab <= SF_TOP_MAX_VOCAB,
               "%s: %lld rows (fewer than %d) of %lld (at most %d)", what, (long long)d.rows, SF_TOP_MAX_ROWS,
               (long long)d.vocab, SF_TOP_MAX_VOCAB);
  SF_CHECK_ARG(d.inner > 0 && d.rows % d.inner == 0 && d.outer_stride >= 0 && d.row_stride >= 0,
               "%s: rows in groups of %lld, strides %lld, %lld", what, (long long)d.inner, (long long)d.outer_stride,
               (long long)d.row_stride);
  SF_CHECK_ARG(d.k >= 0 && d.k <= d.vocab && d.k <= SF_TOP_MAX_ENTRIES, "%s: %lld entries of %lld (at most %d)", what,
               (long long)d.k, (long long)d.vocab, SF_TOP_MAX_ENTRIES);
  SF_CHECK_ARG(d.id_bytes == 4 || d.id_bytes == 8, "%s: ids must be int32 or int64", what);
  SF_CHECK_ARG(d.logits && ((d.values && d.ids) || d.k == 0) && d.stats && d.norm, "%s: null pointer", what);
  SF_CHECK_ARG(d.temperature >= 1.0e-30f && d.temperature <= 1.0e30f, "%s: temperature %g", what, d.temperature);
  a.s = d.logits, a.s0 = d.outer_stride, a.s1 = d.row_stride, a.inner = d.inner;
  a.values = d.values, a.ids = d.ids, a.lse = d.lse, a.weights = d.weights;
  a.vocab = static_cast<int>(d.vocab), a.k = static_cast<int>(d.k), a.vdt = d.value_dtype, a.id_bytes = d.id_bytes;
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
  const size_t lds = static_cast<size_t>(mark_words(a.vocab)) * 4;
  double* row_kl = static_cast<double*>(workspace);
  tk_dispatch(*desc, [&](auto dt, auto) {
    constexpr int DT = decltype(dt)::value;
    auto with = [&](auto blk) {
      constexpr int BLK = decltype(blk)::value;
      if (a.lse)
        top_kl_kernel<DT, BLK, true><<<grid, BLK, lds, st>>>(a, desc->stats, row_kl);
      else
        top_kl_kernel<DT, BLK, false><<<grid, BLK, lds, st>>>(a, desc->stats, row_kl);
    };
    if (desc->rows <= kTkFewRows)
      with(std::integral_constant<int, 1024>{});
    else
      with(std::integral_constant<int, 256>{});
  });
  top_kl_final_kernel<<<1, kTkFinal, 0, st>>>(row_kl, a.weights, desc->rows, desc->temperature, loss, desc->norm);
  return launch_status("sf_top_kl_forward");
}

extern "C" int sf_top_kl_backward(const sf_top_kl_desc* desc, const float* grad_out, void* grad_logits, void* stream) {
  TopKlArgs a;
  if (int rc = top_kl_args(desc, "sf_top_kl_backward", a)) return rc;
  SF_CHECK_ARG(grad_out && grad_logits, "sf_top_kl_backward: null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(desc->rows));
  tk_dispatch(*desc, [&](auto dt, auto past) {
    constexpr int DT = decltype(dt)::value;
    constexpr bool PAST = decltype(past)::value;
    if (desc->rows <= kTkFewRows)
      top_kl_backward_kernel<DT, 1024, PAST><<<grid, 1024, 0, st>>>(a, desc->stats, desc->norm, grad_out, grad_logits);
    else
      top_kl_backward_kernel<DT, 512, PAST><<<grid, 512, 0, st>>>(a, desc->stats, desc->norm, grad_out, grad_logits);
  });
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
  const size_t lds = static_cast<size_t>(mark_words(a.vocab)) * 4;
  tk_dispatch(*desc, [&](auto dt, auto past) {
    top_kl_second_kernel<decltype(dt)::value, decltype(past)::value><<<grid, kTkSecond, lds, st>>>(
        a, desc->stats, desc->norm, grad_out, grad_grad, grad2_logits, row_dot);
  });
  if (dot) top_kl_dot_kernel<<<1, kTkFinal, 0, st>>>(row_dot, desc->rows, dot);
  return launch_status("sf_top_kl_double_backward");
}
