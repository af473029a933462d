// Logits before a token is drawn: penalties for tokens that a sequence already holds, a bias, a mask of the tokens that
// may follow.  For token t of row b, in this order and in f32, rounded once to the output's type:
//   x = logit;  if t occurs c > 0 times in the row's history: x = x > 0 ? x / repetition : x * repetition,
//   x -= frequency * c, x -= presence;  x += bias[t];  x = -inf where t is not allowed.
//
// A workgroup takes a slice of a row's vocabulary: it counts the row's history that falls into the slice in LDS
// (integer atomics: the order does not matter), then streams over the slice.  Bound by memory: the logits are read and
// written once; the history is read by every slice of the row, from the L2 after the first.  Measured: 512 rows of
// 131072 f32 with histories up to 4096, a shared bias and bits, 113 us (562 MB, 4.95 TB/s, what a copy reaches); 64 rows
// of 50257 f32 with a byte mask 8.6 us; one row of 32000 bf16 2.9 us.  256 threads: 163 us for the first, slices of 4096:
// 123 us, 1024 threads: 118 us.
#include "sf_mfma.hpp"

namespace sf {
namespace {

constexpr int kLgBlock = 512;
constexpr int kLgMaxSlice = 8192;  // tokens whose counts fit 32 KB

struct LogitsArgs {
  const void* x;
  void* y;
  int64_t xs, ys;  // row strides in elements
  int64_t V, slice;
  const void* hist;
  int64_t hs, hlen;
  int hist_bytes;
  const int32_t* lengths;  // null: hlen for every row
  const float* rep;        // per row, or null: the number
  const float* pres;
  const float* freq;
  float rep1, pres1, freq1;
  const float* bias;
  int64_t bs;           // row stride, 0: shared
  const uint8_t* mask;  // bits (mask_bits) or bytes
  int64_t ms;           // row stride in bytes, 0: shared
  int mask_bits;
};

// 8 elements from any element's address (a dword's alignment is enough for the wide loads, and HSA allows less).
template <int DT>
__device__ __forceinline__ void lg_load8(const void* p, int64_t i, float (&v)[8]) {
  if constexpr (DT == SF_DTYPE_BF16) {
    uint32_t w[4];
    __builtin_memcpy(w, static_cast<const uint16_t*>(p) + i, 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = lo_f(w[k]);
      v[2 * k + 1] = hi_f(w[k]);
    }
  } else {
    __builtin_memcpy(v, static_cast<const float*>(p) + i, 32);
  }
}
template <int DT, bool PAST>
__device__ __forceinline__ void lg_store8(void* p, int64_t i, const float (&v)[8]) {
  typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
  auto put = [](u32x4u* q, const u32x4u& w) {
    if constexpr (PAST)
      __builtin_nontemporal_store(w, q);
    else
      *q = w;
  };
  if constexpr (DT == SF_DTYPE_BF16) {
    put(reinterpret_cast<u32x4u*>(static_cast<uint16_t*>(p) + i),
        u32x4u{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])});
  } else {
#pragma unroll
    for (int k = 0; k < 8; k += 4)
      put(reinterpret_cast<u32x4u*>(static_cast<float*>(p) + i + k),
          u32x4u{__float_as_uint(v[k]), __float_as_uint(v[k + 1]), __float_as_uint(v[k + 2]), __float_as_uint(v[k + 3])});
  }
}

struct Penalty {
  float rep, pres, freq;
  __device__ __forceinline__ float operator()(float x, uint32_t count) const {
    if (count == 0) return x;
    x = x > 0.0f ? x / rep : x * rep;
    x = x - freq * static_cast<float>(count);
    return x - pres;
  }
};

// PAST: the output is written past the caches.
template <int DT, bool PAST>
__global__ void __launch_bounds__(kLgBlock) logits_kernel(LogitsArgs a) {
  extern __shared__ __align__(16) uint32_t counts[];
  const int64_t b = blockIdx.y, lo = blockIdx.x * a.slice, hi = lo + a.slice < a.V ? lo + a.slice : a.V;
  const int t = threadIdx.x;
  int64_t len = 0;
  if (a.hist) {
    len = a.lengths ? a.lengths[b] : a.hlen;
    len = len < 0 ? 0 : len > a.hlen ? a.hlen : len;
  }
  if (len > 0) {
    for (int i = t * 4; i < a.slice; i += kLgBlock * 4) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int64_t i = t; i < len; i += kLgBlock) {
      const int64_t id = a.hist_bytes == 8 ? static_cast<const int64_t*>(a.hist)[b * a.hs + i]
                                           : static_cast<const int32_t*>(a.hist)[b * a.hs + i];
      if (id >= lo && id < hi) atomicAdd(&counts[id - lo], 1u);
    }
    __syncthreads();
  }
  const Penalty pen{a.rep ? a.rep[b] : a.rep1, a.pres ? a.pres[b] : a.pres1, a.freq ? a.freq[b] : a.freq1};
  const uint8_t* mask = a.mask ? a.mask + b * a.ms : nullptr;
  for (int64_t i = lo + t * 8; i < hi; i += kLgBlock * 8) {
    const int at = static_cast<int>(i - lo);
    if (i + 8 <= hi) {
      float v[8];
      lg_load8<DT>(a.x, b * a.xs + i, v);
      if (len > 0) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = pen(v[k], counts[at + k]);
      }
      if (a.bias) {
        float w[8];
        lg_load8<SF_DTYPE_F32>(a.bias, b * a.bs + i, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = v[k] + w[k];
      }
      if (mask) {
        uint32_t bits = 0;
        if (a.mask_bits) {
          bits = mask[i / 8];
        } else {
          uint32_t w[2];
          __builtin_memcpy(w, mask + i, 8);
#pragma unroll
          for (int k = 0; k < 8; ++k) bits |= (w[k / 4] >> (8 * (k & 3)) & 255u) ? 1u << k : 0u;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (!(bits >> k & 1)) v[k] = -INFINITY;
      }
      lg_store8<DT, PAST>(a.y, b * a.ys + i, v);
    } else {
      for (int k = 0; i + k < hi; ++k) {
        float x = load_as_f32(a.x, b * a.xs + i + k, DT);
        if (len > 0) x = pen(x, counts[at + k]);
        if (a.bias) x = x + a.bias[b * a.bs + i + k];
        if (mask && !(a.mask_bits ? mask[(i + k) / 8] >> ((i + k) % 8) & 1 : mask[i + k] != 0)) x = -INFINITY;
        store_from_f32(a.y, b * a.ys + i + k, DT, x);
      }
    }
  }
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" int sf_process_logits(const sf_logits_desc* desc, void* stream) {
  SF_CHECK_ARG(desc, "sf_process_logits: null descriptor");
  const sf_logits_desc& d = *desc;
  const int64_t rows = d.rows, vocab = d.vocab;
  SF_CHECK_ARG(d.dtype == SF_DTYPE_F32 || d.dtype == SF_DTYPE_BF16, "sf_process_logits: unknown dtype %d", d.dtype);
  SF_CHECK_ARG(rows >= 0 && rows < 65536 && vocab >= 0 && vocab < (1ll << 31), "sf_process_logits: %lld rows of %lld",
               (long long)rows, (long long)vocab);
  if (rows == 0 || vocab == 0) return SF_OK;
  SF_CHECK_ARG(d.logits && d.out, "sf_process_logits: null pointer");
  SF_CHECK_ARG(d.logits_stride >= 0 && d.out_stride >= vocab, "sf_process_logits: strides %lld, %lld for rows of %lld",
               (long long)d.logits_stride, (long long)d.out_stride, (long long)vocab);
  SF_CHECK_ARG(!d.history || ((d.history_bytes == 4 || d.history_bytes == 8) && d.history_len >= 0),
               "sf_process_logits: the history must be int32 or int64");
  SF_CHECK_ARG(d.repetition || d.repetition_all > 0.0f, "sf_process_logits: a repetition penalty of %g",
               d.repetition_all);
  LogitsArgs a;
  a.x = d.logits, a.y = d.out, a.xs = d.logits_stride, a.ys = d.out_stride;
  a.V = vocab;
  a.hist = d.history, a.hs = d.history_stride, a.hlen = d.history_len, a.hist_bytes = d.history_bytes;
  a.lengths = d.history_lengths;
  a.rep = d.repetition, a.pres = d.presence, a.freq = d.frequency;
  a.rep1 = d.repetition_all, a.pres1 = d.presence_all, a.freq1 = d.frequency_all;
  a.bias = d.bias, a.bs = d.bias_stride;
  a.mask = static_cast<const uint8_t*>(d.allowed), a.ms = d.allowed_stride, a.mask_bits = d.allowed_bits;
  // slices small enough that the rows fill the card, not so small that reading the history again outweighs a slice
  int64_t slices = ceil_div(1024, rows);
  const int64_t fewest = ceil_div(vocab, kLgMaxSlice), most = ceil_div(vocab, 8 * kLgBlock);
  slices = slices > most ? most : slices;
  slices = slices < fewest ? fewest : slices;
  a.slice = ceil_div(ceil_div(vocab, slices), 32) * 32;
  slices = ceil_div(vocab, a.slice);
  const dim3 grid(static_cast<unsigned>(slices), static_cast<unsigned>(rows));
  const size_t lds = d.history ? static_cast<size_t>(a.slice) * 4 : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  // An output that the last-level cache (256 MB) does not hold beside the logits only pushes out of it what else is read,
  // and is not found there by who reads it next. 512 rows of 131072 f32: 88 us past the caches, 101 through them, with an
  // argmax of the result after it 162 and 166; 1024 of 50257 bf16 (103 MB): 50 and 51, 83 and 82; 256 of 131072 bf16 (67
  // MB): 31 and 31, 82 and 72.
  const bool past = rows * vocab * (d.dtype == SF_DTYPE_BF16 ? 2 : 4) > (128ll << 20);
  if (d.dtype == SF_DTYPE_BF16) {
    if (past)
      logits_kernel<SF_DTYPE_BF16, true><<<grid, kLgBlock, lds, st>>>(a);
    else
      logits_kernel<SF_DTYPE_BF16, false><<<grid, kLgBlock, lds, st>>>(a);
  } else {
    if (past)
      logits_kernel<SF_DTYPE_F32, true><<<grid, kLgBlock, lds, st>>>(a);
    else
      logits_kernel<SF_DTYPE_F32, false><<<grid, kLgBlock, lds, st>>>(a);
  }
  return launch_status("sf_process_logits");
}
