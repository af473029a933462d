// The 8-bit cache of keys and values (layout: sf_kv8.hpp): new rows appended, and what the cache stands for.
//
// A block that the new rows complete is coded: a = max |x| over its 64 x D elements, code = rint(127 x / a) (ties to
// even), scale = a / 127; the codes are those of exact arithmetic (Coder).  Rows of an incomplete block are kept as
// they come until the block is whole: what the cache holds does not depend on how many rows came at a time.  A token
// whose key or value (of a head) holds a NaN or an infinity is a NaN token: both its rows become NaN, and the block it
// completes has NaN for its scales.
//
// Both are bound by memory: append reads 4 D bytes per token and head and writes 2 D, values reads 2 D and writes
// 8 D.  Measured, 32 heads of 128: eight prompts of 1024 to 2048 tokens, append 62 us (302 MB, 4.9 TB/s) and values of
// 8 x 2048 positions 106 us (618 MB, 5.8 TB/s); one token for each of 32 sequences, some completing a block, 8.8 us, and
// the values of the block it is in 24 us (100 MB, most of it kept rows and outputs).
#include "sf_kv8.hpp"

namespace sf {
namespace {

__global__ void __launch_bounds__(256) kv8_extend_kernel(KvCache c, int n, const int32_t* __restrict__ counts) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= c.B) return;
  const int cap = static_cast<int>(c.blocks * kKvBlock);
  const int count = counts ? min(max(counts[b], 0), n) : n;
  const int start = min(max(c.ends[b], 0), cap);
  c.starts[b] = start;
  c.ends[b] = min(start + count, cap);
}

struct AppendArgs {
  KvCache c;
  const uint16_t* k;  // [B, n, H, D]
  const uint16_t* v;
  int64_t ksb, kss, ksh, vsb, vss, vsh;
  int n;
};

__device__ __forceinline__ bool nonfinite(uint32_t w) {  // either half of two bf16
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// rint(127 x / top) without a division for each element.  `unit` is 2^k and `c` 127 / (top unit): x unit c is off by
// less than 2^-22 of itself.  The exact quotient of 15 bits by 8 is a half-integer or at least 2^-16 of itself away
// from one, so rounding to 18 bits first (t - (t - y) with t = 65 y) gives half-integers where they are exact and
// keeps the others on their side.
struct Coder {
  float unit, c;
  __device__ __forceinline__ explicit Coder(float top) {
    unit = top < 0x1p-60f ? 0x1p66f : top > 0x1p60f ? 0x1p-60f : 1.0f;
    c = top > 0.0f ? 127.0f / (top * unit) : 0.0f;
  }
  __device__ __forceinline__ uint32_t operator()(float x) const {
    const float y = x * unit * c, t = y * 65.0f;
    return static_cast<uint32_t>(static_cast<int>(rintf(t - (t - y)))) & 255u;
  }
};

// One workgroup per (block, head, sequence), a thread for 4 keys x 8 dims: its codes of values are dwords of their
// lines, its rows of keys 8 bytes; a wave has 32 keys x 64 dims, whole lines of the rows it reads.  The first block's workgroup also keeps the rows of the last, incomplete block, after
// it has read the tail that they replace.
__global__ void __launch_bounds__(2 * kKvMaxD) kv8_append_kernel(AppendArgs a) {
  __shared__ uint32_t top[2][2 * kKvMaxD / 64];
  __shared__ uint32_t bad[kKvBlock];
  const KvCache& c = a.c;
  const int h = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  int start, end;
  kv_range(c, b, a.n, start, end);
  const int blk = start / kKvBlock + blockIdx.x, last = end / kKvBlock;
  const int64_t bh = (int64_t)b * c.H + h;
  const int wave = t / 64, lane = t % 64;
  const int j0 = (wave % 2 * 8 + lane / 8) * 4, d = (wave / 2 * 8 + lane % 8) * 8;
  const uint16_t* kin = a.k + b * a.ksb + h * a.ksh + d;
  const uint16_t* vin = a.v + b * a.vsb + h * a.vsh + d;
  uint16_t* kt = c.kt + bh * kKvBlock * c.Dp;
  uint16_t* vt = c.vt + bh * kKvBlock * c.Dp;
  V4 kx[4], vx[4];
  if (start < end && blk < last) {
    uint32_t mk = 0, mv = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = blk * kKvBlock + j0 + i;
      kx[i] = vx[i] = zero16();
      if (row < start) {
        kx[i] = ld16(kt + kv_key_at(j0 + i, d));
#pragma unroll
        for (int q = 0; q < 8; ++q) vx[i].w[q / 2] |= (uint32_t)vt[kv_value_at(j0 + i, d + q)] << (16 * (q & 1));
      } else if (d < c.D) {
        kx[i] = ld16(kin + (row - start) * a.kss);
        vx[i] = ld16(vin + (row - start) * a.vss);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // magnitudes of bf16 order as integers, infinities and NaN at the top
        const uint32_t x = kx[i].w[q] & 0x7fff7fffu, y = vx[i].w[q] & 0x7fff7fffu;
        mk = max(mk, max(x & 0xffffu, x >> 16));
        mv = max(mv, max(y & 0xffffu, y >> 16));
      }
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      mk = max(mk, (uint32_t)__shfl_xor((int)mk, m, 64));
      mv = max(mv, (uint32_t)__shfl_xor((int)mv, m, 64));
    }
    if ((t & 63) == 0) {
      top[0][t >> 6] = mk;
      top[1][t >> 6] = mv;
    }
    __syncthreads();
    for (int w = 0; w < (int)blockDim.x / 64; ++w) {
      mk = max(mk, top[0][w]);
      mv = max(mv, top[1][w]);
    }
    const bool nan = mk >= 0x7f80u || mv >= 0x7f80u;
    const float ak = nan ? 0.0f : __uint_as_float(mk << 16), av = nan ? 0.0f : __uint_as_float(mv << 16);
    int8_t* kc = c.k + (bh * c.blocks + blk) * kKvBlock * c.Dp;
    int8_t* vc = c.v + (bh * c.blocks + blk) * kKvBlock * c.Dp;
    if (nan) {  // no codes: x c would be NaN
#pragma unroll
      for (int i = 0; i < 4; ++i) kx[i] = vx[i] = zero16();
    }
    const Coder ck(ak), cv(av);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int q = 0; q < 8; ++q)
        w[q / 4] |= ck(q & 1 ? hi_f(kx[i].w[q / 2]) : lo_f(kx[i].w[q / 2])) << (8 * (q & 3));
      *reinterpret_cast<uint2*>(kc + kv_key_at(j0 + i, d)) = make_uint2(w[0], w[1]);
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {  // keys j0 .. j0 + 3 lie side by side
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= cv(q & 1 ? hi_f(vx[i].w[q / 2]) : lo_f(vx[i].w[q / 2])) << (8 * i);
      *reinterpret_cast<uint32_t*>(vc + kv_value_at(j0, d + q)) = w;
    }
    if (t == 0) {
      c.ks[bh * c.blocks + blk] = nan ? __builtin_nanf("") : ak / 127.0f;
      c.vs[bh * c.blocks + blk] = nan ? __builtin_nanf("") : av / 127.0f;
    }
  }
  if (blockIdx.x != 0 || start >= end || end % kKvBlock == 0) return;
  if (t < kKvBlock) bad[t] = 0;
  __syncthreads();  // also: the tail has been read
  bool in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = last * kKvBlock + j0 + i;
    in[i] = row >= start && row < end;
    kx[i] = vx[i] = zero16();
    if (in[i] && d < c.D) {
      kx[i] = ld16(kin + (row - start) * a.kss);
      vx[i] = ld16(vin + (row - start) * a.vss);
    }
    bool any = false;
#pragma unroll
    for (int q = 0; q < 4; ++q) any |= nonfinite(kx[i].w[q]) || nonfinite(vx[i].w[q]);
    if (any) bad[j0 + i] = 1;  // every writer writes 1
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!in[i]) continue;
    V4 x = kx[i], y = vx[i];
    if (bad[j0 + i]) x.w[0] = x.w[1] = x.w[2] = x.w[3] = y.w[0] = y.w[1] = y.w[2] = y.w[3] = 0x7fc07fc0u;
    *reinterpret_cast<uint4*>(kt + kv_key_at(j0 + i, d)) = make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
#pragma unroll
    for (int q = 0; q < 8; ++q)
      vt[kv_value_at(j0 + i, d + q)] = static_cast<uint16_t>(q & 1 ? y.w[q / 2] >> 16 : y.w[q / 2]);
  }
}

struct ValuesArgs {
  KvCache c;
  const int32_t* first;  // [B], or null
  int64_t first_all;
  int64_t tokens;
  float* k;  // [B, tokens, H, D]
  float* v;
};

// One workgroup per (block, head, sequence), a thread for 4 keys x 4 dims: 16 bytes of 4 rows of each output.
__global__ void __launch_bounds__(256) kv8_values_kernel(ValuesArgs a) {
  const KvCache& c = a.c;
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t first = a.first ? a.first[b] : a.first_all;
  const int64_t blk = (first >> 6) + blockIdx.x;
  int start, end;
  kv_range(c, b, INT32_MAX, start, end);
  const int64_t bh = (int64_t)b * c.H + h, at = (bh * c.blocks + blk) * kKvBlock * c.Dp;
  const bool held = blk >= 0 && blk < (end + kKvBlock - 1) / kKvBlock, coded = held && blk < end / kKvBlock;
  const float ks = coded ? c.ks[bh * c.blocks + blk] : 1.0f, vs = coded ? c.vs[bh * c.blocks + blk] : 1.0f;
  const int quads = c.D / 4;
  for (int item = threadIdx.x; item < quads * (kKvBlock / 4); item += 256) {
    const int kg = item / quads, d = (item - kg * quads) * 4, j0 = kg * 4;
    float k[4][4] = {}, v[4][4] = {};
    if (coded) {
      uint32_t kw[4], vw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kw[i] = *reinterpret_cast<const uint32_t*>(c.k + at + kv_key_at(j0 + i, d));
        vw[i] = *reinterpret_cast<const uint32_t*>(c.v + at + kv_value_at(j0, d + i));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          k[i][q] = ks * static_cast<float>(static_cast<int8_t>(kw[i] >> (8 * q)));
          v[i][q] = vs * static_cast<float>(static_cast<int8_t>(vw[q] >> (8 * i)));
        }
    } else if (held) {
      const uint16_t* kt = c.kt + bh * kKvBlock * c.Dp;
      const uint16_t* vt = c.vt + bh * kKvBlock * c.Dp;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint2 x = *reinterpret_cast<const uint2*>(kt + kv_key_at(j0 + i, d));
        const uint2 y = *reinterpret_cast<const uint2*>(vt + kv_value_at(j0, d + i));
        k[i][0] = lo_f(x.x), k[i][1] = hi_f(x.x), k[i][2] = lo_f(x.y), k[i][3] = hi_f(x.y);
        v[0][i] = lo_f(y.x), v[1][i] = hi_f(y.x), v[2][i] = lo_f(y.y), v[3][i] = hi_f(y.y);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t pos = blk * kKvBlock + j0 + i, tok = pos - first;
      if (tok < 0 || tok >= a.tokens) continue;
      const bool in = pos < end;
      const int64_t o = ((b * a.tokens + tok) * c.H + h) * c.D + d;
      typedef float f4 __attribute__((ext_vector_type(4)));
      f4 x = {k[i][0], k[i][1], k[i][2], k[i][3]}, y = {v[i][0], v[i][1], v[i][2], v[i][3]};
      if (!in) x = y = f4{};
      // past the caches, which hold the rows and codes that come next: 145 -> 106 us for 268 MB an output
      __builtin_nontemporal_store(x, reinterpret_cast<f4*>(a.k + o));
      __builtin_nontemporal_store(y, reinterpret_cast<f4*>(a.v + o));
    }
  }
}

}  // namespace

int kv8_cache(const sf_kv8_cache* d, const char* what, KvCache& c) {
  SF_CHECK_ARG(d, "%s: no cache", what);
  SF_CHECK_ARG(d->batch >= 1 && d->batch < 65536 && d->kv_heads >= 1 && d->kv_heads < 65536,
               "%s: batch %lld and kv_heads %lld must lie in 1 .. 65535", what, (long long)d->batch,
               (long long)d->kv_heads);
  SF_CHECK_ARG(d->head_dim >= 8 && d->head_dim <= kKvMaxD && d->head_dim % 8 == 0,
               "%s: head_dim %lld must be a multiple of 8 up to %d", what, (long long)d->head_dim, kKvMaxD);
  SF_CHECK_ARG(d->blocks >= 1 && d->blocks <= (1ll << 24), "%s: %lld blocks", what, (long long)d->blocks);
  SF_CHECK_ARG(d->k_codes && d->v_codes && d->k_scales && d->v_scales && d->k_tail && d->v_tail && d->starts && d->ends,
               "%s: null pointer", what);
  c = KvCache{static_cast<int8_t*>(d->k_codes), static_cast<int8_t*>(d->v_codes), d->k_scales, d->v_scales,
              static_cast<uint16_t*>(d->k_tail), static_cast<uint16_t*>(d->v_tail), d->starts, d->ends, d->blocks,
              static_cast<int>(d->batch), static_cast<int>(d->kv_heads), static_cast<int>(d->head_dim),
              static_cast<int>(kv_pad(d->head_dim))};
  for (const void* p : {d->k_codes, d->v_codes, d->k_tail, d->v_tail})
    SF_CHECK_ARG(reinterpret_cast<uintptr_t>(p) % 16 == 0, "%s: codes and tails must be 16-byte aligned", what);
  return SF_OK;
}

}  // namespace sf

using namespace sf;

extern "C" int sf_kv8_extend(const sf_kv8_cache* cache, int64_t n, const int32_t* counts, void* stream) {
  KvCache c;
  if (int rc = kv8_cache(cache, "sf_kv8_extend", c)) return rc;
  SF_CHECK_ARG(n >= 0 && n <= c.blocks * kKvBlock, "sf_kv8_extend: %lld tokens for a capacity of %lld", (long long)n,
               (long long)(c.blocks * kKvBlock));
  kv8_extend_kernel<<<static_cast<unsigned>(ceil_div(c.B, 256)), 256, 0, static_cast<hipStream_t>(stream)>>>(
      c, static_cast<int>(n), counts);
  return launch_status("sf_kv8_extend");
}

extern "C" int sf_kv8_append(const sf_kv8_cache* cache, const void* k, int64_t k_sb, int64_t k_ss, int64_t k_sh,
                             const void* v, int64_t v_sb, int64_t v_ss, int64_t v_sh, int64_t n, void* stream) {
  AppendArgs a;
  if (int rc = kv8_cache(cache, "sf_kv8_append", a.c)) return rc;
  SF_CHECK_ARG(n >= 0 && n <= a.c.blocks * kKvBlock, "sf_kv8_append: %lld rows for a capacity of %lld", (long long)n,
               (long long)(a.c.blocks * kKvBlock));
  if (n == 0) return SF_OK;
  SF_CHECK_ARG(k && v, "sf_kv8_append: null pointer");
  SF_CHECK_ARG((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 &&
                   (k_sb | k_ss | k_sh | v_sb | v_ss | v_sh) % 8 == 0,
               "sf_kv8_append: rows must be 16-byte aligned");
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.ksb = k_sb, a.kss = k_ss, a.ksh = k_sh, a.vsb = v_sb, a.vss = v_ss, a.vsh = v_sh;
  a.n = static_cast<int>(n);
  // blocks that n rows can touch from any start
  const int64_t touched = (n + kKvBlock - 2) / kKvBlock + 1;
  kv8_append_kernel<<<dim3((unsigned)touched, a.c.H, a.c.B), 2 * a.c.Dp, 0, static_cast<hipStream_t>(stream)>>>(a);
  return launch_status("sf_kv8_append");
}

extern "C" int sf_kv8_values(const sf_kv8_cache* cache, const int32_t* first, int64_t first_all, int64_t tokens,
                             float* k, float* v, void* stream) {
  ValuesArgs a;
  if (int rc = kv8_cache(cache, "sf_kv8_values", a.c)) return rc;
  SF_CHECK_ARG(tokens >= 0 && tokens <= a.c.blocks * kKvBlock, "sf_kv8_values: %lld tokens of a capacity of %lld",
               (long long)tokens, (long long)(a.c.blocks * kKvBlock));
  if (tokens == 0) return SF_OK;
  SF_CHECK_ARG(k && v, "sf_kv8_values: null pointer");
  SF_CHECK_ARG((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0,
               "sf_kv8_values: outputs must be 16-byte aligned");
  a.first = first;
  a.first_all = first_all;
  a.tokens = tokens;
  a.k = k;
  a.v = v;
  const int64_t touched = (tokens + kKvBlock - 2) / kKvBlock + 1;
  kv8_values_kernel<<<dim3((unsigned)touched, a.c.H, a.c.B), 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  return launch_status("sf_kv8_values");
}
