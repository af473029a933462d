// Rotary positions of queries and keys: each pair (a, b) of a head's first `rotary` elements turns by the angle of
// its position and pair,
//   a' = a c - b s,  b' = b c + a s,   c, s = cos, sin [position][pair]  (f32 tables, any scaling in them),
// the rest of the head is copied.  Pairs are (i, i + rotary / 2), or (2 i, 2 i + 1) when interleaved.  The adjoint,
// which carries gradients back, is the same turn the other way: s -> -s.  Products and sums in f32, one rounding
// to the tensors' type (the model's own attention rounds each product to bf16, as HuggingFace's eager form does).
//
// Bound by memory: every element is read once and written once, and the 8 bytes of cos and sin per pair, which the
// heads of a token share, come from the caches.  One launch takes queries and keys.  A thread turns two chunks of V
// elements (one, of V / 2 pairs, when interleaved) or copies one, the widest of 8, 4, 2, 1 that sizes, strides and
// addresses allow, 16 bytes at most (`chunk_width`).  Measured: 2 x 2048 tokens of 32 + 32 bf16 heads of 64, columns of a
// fused projection, 12.6 us a pass (67 MB, 5.3 TB/s); 32749 tokens of 32 + 8 f32 heads of 80, 20 of them turning,
// interleaved, 177 us (840 MB, 4.7 TB/s; chunks of 8 bytes: 279 us); 4 tokens of 32 + 32 heads of 128, 3.2 us.
#include "sf_common.hpp"

namespace sf {
namespace {

constexpr int kRotBlock = 256;

// n / d for n < 2^31 as one multiply and a shift.
struct FastDiv {
  uint32_t d, m, l;
};
inline FastDiv fast_div(uint32_t d) {
  FastDiv f{d, 0, 0};
  while ((1ull << f.l) < d) ++f.l;
  f.m = static_cast<uint32_t>((((1ull << f.l) - d) << 32) / d + 1);
  return f;
}
__device__ __forceinline__ uint32_t quot(uint32_t n, const FastDiv& f) { return (__umulhi(n, f.m) + n) >> f.l; }

struct RotTensor {
  const void* x;
  void* y;             // contiguous [B, S, heads, D]
  int64_t sb, ss, sh;  // strides of x in elements
  int heads;
};
struct RotArgs {
  RotTensor t[2];
  const float* cos;  // [table_rows, rotary / 2]
  const float* sin;
  const void* pos;   // null: the position is s
  int pos_bytes;     // 4 or 8
  int64_t pos_sb;    // stride of a batch entry in pos (0: shared)
  int64_t table_rows;
  int64_t first;     // this launch's first token
  uint32_t items;
  int D, half, turn_units;  // units that turn pairs; the others copy
  int copy_width;
  float sign;
  FastDiv per_token, per_head, seq;
};

template <int DT, int V>
struct Chunk {
  float v[V];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (DT == SF_DTYPE_BF16) {
      const uint16_t* q = static_cast<const uint16_t*>(p) + i;
      uint32_t w[V / 2 ? V / 2 : 1];
      if constexpr (V == 8) {
        const uint4 x = *reinterpret_cast<const uint4*>(q);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
      } else if constexpr (V == 4) {
        const uint2 x = *reinterpret_cast<const uint2*>(q);
        w[0] = x.x; w[1] = x.y;
      } else if constexpr (V == 2) {
        w[0] = *reinterpret_cast<const uint32_t*>(q);
      } else {
        w[0] = *q;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = __uint_as_float(k & 1 ? w[k / 2] & 0xffff0000u : w[k / 2] << 16);
    } else {
      const float* q = static_cast<const float*>(p) + i;
      if constexpr (V % 4 == 0) {
#pragma unroll
        for (int k = 0; k < V; k += 4) {
          const float4 x = *reinterpret_cast<const float4*>(q + k);
          v[k] = x.x; v[k + 1] = x.y; v[k + 2] = x.z; v[k + 3] = x.w;
        }
      } else if constexpr (V == 2) {
        const float2 x = *reinterpret_cast<const float2*>(q);
        v[0] = x.x; v[1] = x.y;
      } else {
        v[0] = *q;
      }
    }
  }
  __device__ __forceinline__ void store(void* p, int64_t i) const {
    if constexpr (DT == SF_DTYPE_BF16) {
      uint16_t* q = static_cast<uint16_t*>(p) + i;
      uint32_t w[V / 2 ? V / 2 : 1];
      if constexpr (V == 1) {
        *q = f32_to_bf16(v[0]);
      } else {
#pragma unroll
        for (int k = 0; k < V / 2; ++k)
          w[k] = static_cast<uint32_t>(f32_to_bf16(v[2 * k])) | static_cast<uint32_t>(f32_to_bf16(v[2 * k + 1])) << 16;
        if constexpr (V == 8)
          *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (V == 4)
          *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
        else
          *reinterpret_cast<uint32_t*>(q) = w[0];
      }
    } else {
      float* q = static_cast<float*>(p) + i;
      if constexpr (V % 4 == 0) {
#pragma unroll
        for (int k = 0; k < V; k += 4) *reinterpret_cast<float4*>(q + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
      } else if constexpr (V == 2) {
        *reinterpret_cast<float2*>(q) = make_float2(v[0], v[1]);
      } else {
        *q = v[0];
      }
    }
  }
};

template <int DT, int W>
__device__ __forceinline__ void copy_chunk(const void* x, int64_t src, void* y, int64_t dst) {
  Chunk<DT, W> c;
  c.load(x, src);
  c.store(y, dst);
}

// V: elements of a chunk; a unit is two of them, one when interleaved (V = 1: two single elements).
template <int DT, int V, bool ILV>
__global__ void __launch_bounds__(kRotBlock) rotary_kernel(RotArgs a) {
  const uint32_t i = blockIdx.x * kRotBlock + threadIdx.x;
  if (i >= a.items) return;
  const uint32_t tok = quot(i, a.per_token), r = i - tok * a.per_token.d;
  const uint32_t hh = quot(r, a.per_head);
  const int u = static_cast<int>(r - hh * a.per_head.d);
  const int64_t token = a.first + tok;
  const uint32_t b = quot(static_cast<uint32_t>(token), a.seq);
  const int64_t s = token - static_cast<int64_t>(b) * a.seq.d;
  const bool second = static_cast<int>(hh) >= a.t[0].heads;
  const RotTensor& t = second ? a.t[1] : a.t[0];
  const int64_t h = second ? static_cast<int>(hh) - a.t[0].heads : static_cast<int>(hh);
  const int64_t src = b * t.sb + s * t.ss + h * t.sh;
  const int64_t dst = (token * t.heads + h) * a.D;
  if (u >= a.turn_units) {  // the part of the head that does not turn
    const int d = 2 * a.half + (u - a.turn_units) * a.copy_width;
    if (a.copy_width == 8)
      copy_chunk<DT, 8>(t.x, src + d, t.y, dst + d);
    else if (a.copy_width == 4)
      copy_chunk<DT, 4>(t.x, src + d, t.y, dst + d);
    else if (a.copy_width == 2)
      copy_chunk<DT, 2>(t.x, src + d, t.y, dst + d);
    else
      copy_chunk<DT, 1>(t.x, src + d, t.y, dst + d);
    return;
  }
  int64_t p = s;
  if (a.pos) {
    const int64_t at = b * a.pos_sb + s;
    p = a.pos_bytes == 8 ? static_cast<const int64_t*>(a.pos)[at] : static_cast<const int32_t*>(a.pos)[at];
  }
  constexpr bool ONE = ILV && V > 1;      // one chunk holds whole pairs
  constexpr int PAIRS = ONE ? V / 2 : V;
  const int pair = u * PAIRS;
  Chunk<SF_DTYPE_F32, PAIRS> c, sn;
  if (p >= 0 && p < a.table_rows) {
    c.load(a.cos, p * a.half + pair);
    sn.load(a.sin, p * a.half + pair);
  } else {  // a position that the tables do not hold
#pragma unroll
    for (int k = 0; k < PAIRS; ++k) c.v[k] = sn.v[k] = __builtin_nanf("");
  }
  const int d0 = ILV ? 2 * pair : pair, d1 = ILV ? 2 * pair + 1 : pair + a.half;
  Chunk<DT, V> x0, x1, y0, y1;
  x0.load(t.x, src + d0);
  if constexpr (!ONE) x1.load(t.x, src + d1);
#pragma unroll
  for (int k = 0; k < PAIRS; ++k) {
    const float e = ONE ? x0.v[2 * k % V] : x0.v[k % V], o = ONE ? x0.v[(2 * k + 1) % V] : x1.v[k % V];
    const float ss = a.sign * sn.v[k];
    const float e2 = e * c.v[k] - o * ss, o2 = o * c.v[k] + e * ss;
    (ONE ? y0.v[2 * k % V] : y0.v[k % V]) = e2;
    (ONE ? y0.v[(2 * k + 1) % V] : y1.v[k % V]) = o2;
  }
  y0.store(t.y, dst + d0);
  if constexpr (!ONE) y1.store(t.y, dst + d1);
}

template <int DT, int V>
void launch_rotary(const RotArgs& a, bool ilv, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(ceil_div(a.items, kRotBlock)));
  if (ilv)
    rotary_kernel<DT, V, true><<<grid, kRotBlock, 0, st>>>(a);
  else
    rotary_kernel<DT, V, false><<<grid, kRotBlock, 0, st>>>(a);
}

// The widest chunk, 16 bytes at most, that divides `part` and the head and whose accesses are aligned: it starts at
// multiples of its width within a head, heads at the strides' multiples.
int chunk_width(const RotArgs& a, int size, int part) {
  int v = 16 / size;
  for (; v > 1; v /= 2) {
    bool ok = part % v == 0 && a.D % v == 0;
    for (const RotTensor& t : a.t)
      ok = ok && (t.heads == 0 || ((t.sb | t.ss | t.sh) % v == 0 && reinterpret_cast<uintptr_t>(t.x) % (v * size) == 0 &&
                                   reinterpret_cast<uintptr_t>(t.y) % (v * size) == 0));
    if (ok) break;
  }
  return v;
}
// The same for pairs of `part` elements whose V (or V / 2) cosines are read as one too.
int turn_width(const RotArgs& a, int size, bool ilv) {
  int v = chunk_width(a, size, ilv ? 2 * a.half : a.half);
  auto tables = [&] {
    const int pairs = ilv && v > 1 ? v / 2 : v, bytes = pairs < 4 ? 4 * pairs : 16;
    return a.half % pairs == 0 && reinterpret_cast<uintptr_t>(a.cos) % bytes == 0 &&
           reinterpret_cast<uintptr_t>(a.sin) % bytes == 0;
  };
  while (!tables()) v /= 2;
  return v;
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" int sf_rotary(const sf_rotary_desc* desc, void* stream) {
  SF_CHECK_ARG(desc, "sf_rotary: null descriptor");
  const sf_rotary_desc& d = *desc;
  const int64_t B = d.B, S = d.S, D = d.D;
  SF_CHECK_ARG(d.dtype == SF_DTYPE_F32 || d.dtype == SF_DTYPE_BF16, "sf_rotary: unknown dtype %d", d.dtype);
  SF_CHECK_ARG(B >= 0 && S >= 0 && d.heads >= 0 && d.kv_heads >= 0, "sf_rotary: negative size");
  SF_CHECK_ARG((B == 0 || S < (1ll << 31) / B) && d.heads < (1 << 20) && d.kv_heads < (1 << 20),
               "sf_rotary: too many tokens or heads");
  SF_CHECK_ARG(D >= 1 && D <= 4096, "sf_rotary: head dimension %lld outside 1 .. 4096", (long long)D);
  SF_CHECK_ARG(d.rotary_dim >= 2 && d.rotary_dim % 2 == 0 && d.rotary_dim <= D,
               "sf_rotary: rotary_dim %lld must be even, at least 2 and at most the head's %lld",
               (long long)d.rotary_dim, (long long)D);
  SF_CHECK_ARG(!d.positions || d.position_bytes == 4 || d.position_bytes == 8,
               "sf_rotary: positions must be int32 or int64");
  if (B == 0 || S == 0 || d.heads + d.kv_heads == 0) return SF_OK;
  SF_CHECK_ARG(d.cos && d.sin && d.table_rows >= 1, "sf_rotary: no tables");
  SF_CHECK_ARG(d.heads == 0 || (d.q && d.q_out), "sf_rotary: null pointer");
  SF_CHECK_ARG(d.kv_heads == 0 || (d.k && d.k_out), "sf_rotary: null pointer");
  SF_CHECK_ARG(d.positions || S <= d.table_rows, "sf_rotary: %lld positions, the tables hold %lld", (long long)S,
               (long long)d.table_rows);
  RotArgs a{};
  a.t[0] = {d.q, d.q_out, d.q_sb, d.q_ss, d.q_sh, static_cast<int>(d.heads)};
  a.t[1] = {d.k, d.k_out, d.k_sb, d.k_ss, d.k_sh, static_cast<int>(d.kv_heads)};
  a.cos = d.cos;
  a.sin = d.sin;
  a.pos = d.positions;
  a.pos_bytes = d.position_bytes;
  a.pos_sb = d.position_sb;
  a.table_rows = d.table_rows;
  a.D = static_cast<int>(D);
  a.half = static_cast<int>(d.rotary_dim / 2);
  a.sign = d.inverse ? -1.0f : 1.0f;
  const int size = d.dtype == SF_DTYPE_BF16 ? 2 : 4, v = turn_width(a, size, d.interleaved);
  a.copy_width = chunk_width(a, size, 2 * a.half);
  a.turn_units = d.interleaved && v > 1 ? 2 * a.half / v : a.half / v;
  const int64_t per_head = a.turn_units + (D - d.rotary_dim) / a.copy_width;
  const int64_t per_token = per_head * (d.heads + d.kv_heads);
  SF_CHECK_ARG(per_token <= (1ll << 31) - kRotBlock, "sf_rotary: a token's heads are too large");
  a.per_head = fast_div(static_cast<uint32_t>(per_head));
  a.per_token = fast_div(static_cast<uint32_t>(per_token));
  a.seq = fast_div(static_cast<uint32_t>(S));
  const int64_t most = ((1ll << 31) - kRotBlock) / per_token;  // tokens of one launch
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (a.first = 0; a.first < B * S; a.first += most) {
    const int64_t n = B * S - a.first < most ? B * S - a.first : most;
    a.items = static_cast<uint32_t>(n * per_token);
    if (d.dtype == SF_DTYPE_BF16) {
      if (v == 8) launch_rotary<SF_DTYPE_BF16, 8>(a, d.interleaved, st);
      else if (v == 4) launch_rotary<SF_DTYPE_BF16, 4>(a, d.interleaved, st);
      else if (v == 2) launch_rotary<SF_DTYPE_BF16, 2>(a, d.interleaved, st);
      else launch_rotary<SF_DTYPE_BF16, 1>(a, d.interleaved, st);
    } else {
      if (v == 4) launch_rotary<SF_DTYPE_F32, 4>(a, d.interleaved, st);
      else if (v == 2) launch_rotary<SF_DTYPE_F32, 2>(a, d.interleaved, st);
      else launch_rotary<SF_DTYPE_F32, 1>(a, d.interleaved, st);
    }
  }
  return launch_status("sf_rotary");
}
