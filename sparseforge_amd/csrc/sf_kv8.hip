// The 8-bit cache of keys and values (layout: sf_kv8.hpp): new rows appended, and what the cache stands for.
//
// A block that the new rows complete is coded: a = max |x| over its 64 x D elements, code = rint(127 x / a) (ties to
// even), scale = a / 127.  127 x is exact in f32 for a bf16 x and the quotient, correctly rounded, lies on a
// half-integer only where the exact one does, so the codes are those of exact arithmetic.  Rows of an incomplete
// block are kept as they come until the block is whole: what the cache holds does not depend on how many rows came
// at a time.  A token whose key or value (of a head) holds a NaN or an infinity is a NaN token: both its rows become
// NaN, and the block it completes has NaN for its scales.
//
// Both are bound by memory: append reads 4 D bytes per token and head and writes 2 D, values reads 2 D and writes
// 8 D.
#include "sf_kv8.hpp"

namespace sf {
namespace {

constexpr int kAppBlock = 256;

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

// One workgroup per (block, head, sequence).  The first block's also keeps the rows of the last, incomplete one, after
// it has read the tail that they replace.
__global__ void __launch_bounds__(kAppBlock) kv8_append_kernel(AppendArgs a) {
  __shared__ uint32_t top[2][kAppBlock / 64];
  __shared__ uint32_t bad[kKvBlock];
  const KvCache& c = a.c;
  const int h = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  int start, end;
  kv_range(c, b, a.n, start, end);
  const int blk = start / kKvBlock + blockIdx.x, last = end / kKvBlock;
  const int64_t bh = (int64_t)b * c.H + h;
  const int chunks = c.Dp / 8;  // of a row
  const uint16_t* kin = a.k + b * a.ksb + h * a.ksh;
  const uint16_t* vin = a.v + b * a.vsb + h * a.vsh;
  uint16_t* kt = c.kt + bh * kKvBlock * c.Dp;
  uint16_t* vt = c.vt + bh * kKvBlock * c.Dp;
  auto new_row = [&](const uint16_t* in, int64_t ss, int row, int d) {
    return d < c.D ? ld16(in + (row - start) * ss + d) : zero16();
  };
  if (start < end && blk < last) {
    constexpr int N = kKvBlock * kKvMaxD / 8 / kAppBlock;  // chunks of a thread at most
    V4 kx[N], vx[N];
    uint32_t mk = 0, mv = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = t + i * kAppBlock;
      if (at >= kKvBlock * chunks) break;
      const int j = at / chunks, d = (at - j * chunks) * 8, row = blk * kKvBlock + j;
      if (row < start) {
        kx[i] = ld16(kt + kv_key_at(j, d));
#pragma unroll
        for (int q = 0; q < 4; ++q)
          vx[i].w[q] = vt[kv_value_at(j, d + 2 * q)] | (uint32_t)vt[kv_value_at(j, d + 2 * q + 1)] << 16;
      } else {
        kx[i] = new_row(kin, a.kss, row, d);
        vx[i] = new_row(vin, a.vss, row, d);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // magnitudes of bf16 order as integers, infinities and NaN at the top
        const uint32_t x = kx[i].w[q] & 0x7fff7fffu, y = vx[i].w[q] & 0x7fff7fffu;
        mk = max(mk, max(x & 0xffffu, x >> 16));
        mv = max(mv, max(y & 0xffffu, y >> 16));
      }
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
#pragma unroll
    for (int w = 0; w < kAppBlock / 64; ++w) {
      mk = max(mk, top[0][w]);
      mv = max(mv, top[1][w]);
    }
    const bool nan = mk >= 0x7f80u || mv >= 0x7f80u;
    const float ak = __uint_as_float(mk << 16), av = __uint_as_float(mv << 16);
    auto code = [&](uint32_t bits, float amax) -> int {
      float x = __uint_as_float(bits), m = amax;
      if (m >= 0x1p64f) {  // keep 127 x below the largest float
        x *= 0x1p-16f;
        m *= 0x1p-16f;
      }
      return m > 0.0f && !nan ? static_cast<int>(rintf(127.0f * x / m)) : 0;
    };
    int8_t* kc = c.k + (bh * c.blocks + blk) * kKvBlock * c.Dp;
    int8_t* vc = c.v + (bh * c.blocks + blk) * kKvBlock * c.Dp;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = t + i * kAppBlock;
      if (at >= kKvBlock * chunks) break;
      const int j = at / chunks, d = (at - j * chunks) * 8;
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint32_t x = q & 1 ? kx[i].w[q / 2] & 0xffff0000u : kx[i].w[q / 2] << 16;
        const uint32_t y = q & 1 ? vx[i].w[q / 2] & 0xffff0000u : vx[i].w[q / 2] << 16;
        w[q / 4] |= (uint32_t)(code(x, ak) & 255) << (8 * (q & 3));
        vc[kv_value_at(j, d + q)] = static_cast<int8_t>(code(y, av));
      }
      *reinterpret_cast<uint2*>(kc + kv_key_at(j, d)) = make_uint2(w[0], w[1]);
    }
    if (t == 0) {
      c.ks[bh * c.blocks + blk] = nan ? __builtin_nanf("") : ak / 127.0f;
      c.vs[bh * c.blocks + blk] = nan ? __builtin_nanf("") : av / 127.0f;
    }
  }
  if (blockIdx.x != 0 || start >= end || end % kKvBlock == 0) return;
  const int from = max(start, last * kKvBlock);
  if (t < kKvBlock) bad[t] = 0;
  __syncthreads();  // also: the tail has been read
  const int rows = end - from, j0 = from % kKvBlock;
  for (int at = t; at < rows * chunks; at += kAppBlock) {
    const int j = at / chunks, d = (at - j * chunks) * 8;
    const V4 kx = new_row(kin, a.kss, from + j, d), vx = new_row(vin, a.vss, from + j, d);
    bool any = false;
#pragma unroll
    for (int q = 0; q < 4; ++q) any |= nonfinite(kx.w[q]) || nonfinite(vx.w[q]);
    if (any) bad[j] = 1;  // every writer writes 1
  }
  __syncthreads();
  for (int at = t; at < rows * chunks; at += kAppBlock) {
    const int j = at / chunks, d = (at - j * chunks) * 8;
    V4 kx = new_row(kin, a.kss, from + j, d), vx = new_row(vin, a.vss, from + j, d);
    if (bad[j]) kx.w[0] = kx.w[1] = kx.w[2] = kx.w[3] = vx.w[0] = vx.w[1] = vx.w[2] = vx.w[3] = 0x7fc07fc0u;
    *reinterpret_cast<uint4*>(kt + kv_key_at(j0 + j, d)) = make_uint4(kx.w[0], kx.w[1], kx.w[2], kx.w[3]);
#pragma unroll
    for (int q = 0; q < 8; ++q)
      vt[kv_value_at(j0 + j, d + q)] = static_cast<uint16_t>(q & 1 ? vx.w[q / 2] >> 16 : vx.w[q / 2]);
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

// A thread takes 4 dims of one token and head.
__global__ void __launch_bounds__(256) kv8_values_kernel(ValuesArgs a) {
  const KvCache& c = a.c;
  const int quads = (c.D + 3) / 4;
  const int64_t per_seq = a.tokens * c.H * quads;
  const int b = blockIdx.y;
  const int64_t at = blockIdx.x * 256ll + threadIdx.x;
  if (at >= per_seq) return;
  const int64_t row = at / quads;  // (token, head)
  const int d = static_cast<int>(at - row * quads) * 4;
  const int64_t tok = row / c.H;
  const int h = static_cast<int>(row - tok * c.H);
  const int64_t pos = (a.first ? a.first[b] : a.first_all) + tok;
  int start, end;
  kv_range(c, b, INT32_MAX, start, end);
  float k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
  if (pos >= 0 && pos < end) {
    const int64_t bh = (int64_t)b * c.H + h;
    const int blk = static_cast<int>(pos / kKvBlock), j = static_cast<int>(pos % kKvBlock);
    if (blk < end / kKvBlock) {
      const int64_t g = bh * c.blocks + blk;
      const float ks = c.ks[g], vs = c.vs[g];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        k[q] = ks * c.k[g * kKvBlock * c.Dp + kv_key_at(j, d + q)];
        v[q] = vs * c.v[g * kKvBlock * c.Dp + kv_value_at(j, d + q)];
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        k[q] = bf16_to_f32(c.kt[bh * kKvBlock * c.Dp + kv_key_at(j, d + q)]);
        v[q] = bf16_to_f32(c.vt[bh * kKvBlock * c.Dp + kv_value_at(j, d + q)]);
      }
    }
  }
  const int64_t o = ((b * a.tokens + tok) * c.H + h) * c.D + d;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (d + q < c.D) {
      a.k[o + q] = k[q];
      a.v[o + q] = v[q];
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
  kv8_append_kernel<<<dim3((unsigned)touched, a.c.H, a.c.B), kAppBlock, 0, static_cast<hipStream_t>(stream)>>>(a);
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
  const int64_t grid = ceil_div(tokens * a.c.H * ((a.c.D + 3) / 4), 256);
  SF_CHECK_ARG(grid < (1ll << 31), "sf_kv8_values: too many tokens");
  kv8_values_kernel<<<dim3((unsigned)grid, a.c.B), 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  return launch_status("sf_kv8_values");
}
