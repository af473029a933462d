// Attention of the newest tokens over the 8-bit cache (layout: sf_kv8.hpp):
//   o_i = softmax_j(scale q_i k_j) v_j over the keys j <= i, and j > i - window where there is a window,
// with i, j positions of a sequence.  A query that sees no key (its sequence has ended) gives 0.
//
// The query heads that share a key-value head are rows of one product with it: row r of (sequence, key-value head) is
// query r / group of head r % group.  A wave takes 16 RT rows over whole blocks of 64 keys.  q codes and p codes are
// products of bf16 operands (codes up to 127 are exact in bf16) with f32 sums; the block's key scale multiplies the
// scores with the softmax's factor, its value scale the probabilities before they round to bf16.
//
// A wave's running maximum is one for all lanes of a row and is raised only when a score passes it by 8 (in log2):
// probabilities up to 2^8 cost nothing in f32 or bf16, and most blocks need no exchange between lanes.
//
// Bound by memory for single tokens: every code is read once, 2 D bytes per key and head.
#include "sf_kv8.hpp"

namespace sf {
namespace {

constexpr int kAtnWaves = 4;
constexpr float kAtnLog2e = 1.4426950408889634f;
constexpr float kAtnLow = -3.0e38f;  // below every score that counts
constexpr float kAtnSlack = 8.0f;
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct AttendArgs {
  KvCache c;
  const uint16_t* q;  // [B, n, heads, D]
  int64_t qsb, qss, qsh;
  uint16_t* out;      // [B, n, heads, D] contiguous
  int n, heads, group;
  int window;         // 0: none
  float scale;        // times log2 e
  int tiles;          // of 16 RT rows
  int splits, chunk;  // key blocks of a workgroup: at least `chunk`
  float* po;          // [B H tiles][splits][16 RT][Dp] unnormalised outputs
  float* pml;         // [B H tiles][splits][2][16 RT] maxima, sums
};

// What a tile of rows sees.
struct TileRange {
  int start, end;          // newest tokens
  int i0, i1;              // queries of the tile, [i0, i1); none if i0 >= i1
  int b0, b1;              // key blocks, [b0, b1)
  int per;                 // blocks of a split
  __device__ __forceinline__ int used() const { return b1 > b0 ? (b1 - b0 + per - 1) / per : 0; }
};
template <int ROWS>
__device__ __forceinline__ TileRange tile_range(const AttendArgs& a, int b, int tile) {
  TileRange r;
  kv_range(a.c, b, a.n, r.start, r.end);
  const int cnt = r.end - r.start;
  r.i0 = tile * ROWS / a.group;
  r.i1 = min(cnt, (tile * ROWS + ROWS - 1) / a.group + 1);
  r.b0 = r.b1 = 0;
  r.per = 1;
  if (r.i0 >= r.i1) return r;
  const int hi = r.start + r.i1;  // keys below
  const int lo = a.window ? max(0, r.start + r.i0 - a.window + 1) : 0;
  r.b0 = lo / kKvBlock;
  r.b1 = (hi + kKvBlock - 1) / kKvBlock;
  r.per = max(a.chunk, (r.b1 - r.b0 + a.splits - 1) / a.splits);
  return r;
}

// 8 codes -> bf16, exact: a code has at most 8 significant bits, so the high half of its float is the bf16.
__device__ __forceinline__ bf16x8_t codes_to_bf16(uint32_t w0, uint32_t w1) {
  uint32_t o[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t w = q < 2 ? w0 : w1;
    const int sh = 16 * (q & 1);
    const float lo = static_cast<float>(static_cast<int8_t>(w >> sh));
    const float hi = static_cast<float>(static_cast<int8_t>(w >> (sh + 8)));
    o[q] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
  }
  return __builtin_bit_cast(bf16x8_t, make_uint4(o[0], o[1], o[2], o[3]));
}

// Operands of a block of codes, loaded whole: chunk (hh, t) of keys, dim tile dt of values.
template <int DB>
struct CodeBlock {
  V4 k[DB * 4], v[DB * 4];
  __device__ __forceinline__ void load(const int8_t* kc, const int8_t* vc) {
    const int lane = threadIdx.x & 63, at = (lane & 15) * 64 + (lane >> 4) * 16;
#pragma unroll
    for (int i = 0; i < DB * 4; ++i) k[i] = ld16(kc + i * 1024 + at);
#pragma unroll
    for (int i = 0; i < DB * 4; ++i) v[i] = ld16(vc + i * 1024 + at);
  }
  __device__ __forceinline__ bf16x8_t key(int hh, int t, int a) const {
    const V4& x = k[hh * 4 + t];
    return codes_to_bf16(x.w[2 * a], x.w[2 * a + 1]);
  }
  __device__ __forceinline__ bf16x8_t value(int dt, int u) const { return codes_to_bf16(v[dt].w[2 * u], v[dt].w[2 * u + 1]); }
};

// The same of an incomplete block: rows past the end and NaN tokens have zeros for their values (a NaN token's key
// makes its probability NaN where it is seen, and where it is not its values must not turn 0 into NaN).
template <int DB>
struct TailBlock {
  const uint16_t* kt;
  const uint16_t* vt;
  int rows;  // of the block
  __device__ __forceinline__ bf16x8_t key(int hh, int t, int a) const {
    const int lane = threadIdx.x & 63;
    const V4 x = ld16(kt + (hh * 64 + t * 16 + (lane & 15)) * 64 + (lane >> 4) * 16 + a * 8);
    return __builtin_bit_cast(bf16x8_t, make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]));
  }
  __device__ __forceinline__ bf16x8_t value(int dt, int u) const {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    V4 x = ld16(vt + (dt * 16 + (lane & 15)) * 64 + g * 16 + u * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int key = 16 * (2 * u + e / 4) + 4 * g + e % 4;
      const uint32_t bits = e & 1 ? x.w[e / 2] >> 16 : x.w[e / 2] & 0xffffu;
      if (key >= rows || (bits & 0x7fffu) > 0x7f80u) x.w[e / 2] &= e & 1 ? 0xffffu : 0xffff0000u;
    }
    return __builtin_bit_cast(bf16x8_t, make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]));
  }
};

// A wave's rows: queries, running softmax and output, transposed (lane: row lane % 16 of each 16).
template <int DB, int RT>
struct RowState {
  bf16x8_t q[RT][DB][2];
  f32x4_t o[RT][DB * 4];
  float m[RT], l[RT];  // l: of the keys this lane's group holds
  int pos[RT];         // position of the row's query, -1: no such row

  template <class Block>
  __device__ __forceinline__ void block(const Block& x, int blk, float ks, float vs, int window, bool masked) {
    const int g = (threadIdx.x & 63) >> 4;
    f32x4_t s[RT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int r = 0; r < RT; ++r) s[r][t] = f32x4_t{};
#pragma unroll
      for (int hh = 0; hh < DB; ++hh)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const bf16x8_t kf = x.key(hh, t, a);
#pragma unroll
          for (int r = 0; r < RT; ++r) s[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[r][hh][a], s[r][t], 0, 0, 0);
        }
    }
    bf16x8_t p[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      uint32_t seen = 0xffffu;  // bit 4 t + e: the row sees key 16 t + 4 g + e
      if (masked) {
        seen = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = blk * kKvBlock + 16 * (i / 4) + 4 * g + i % 4;
          const bool in = key <= pos[r] && (!window || key > pos[r] - window);
          seen |= in ? 1u << i : 0u;
        }
      }
      float mx = kAtnLow;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = s[r][i / 4][i % 4] * ks;
        mx = fmaxf(mx, !masked || (seen >> i & 1) ? x : kAtnLow);
      }
      if (__builtin_amdgcn_ballot_w64(mx > m[r] + kAtnSlack)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m[r], mx), f = __builtin_amdgcn_exp2f(m[r] - mn);
        m[r] = mn;
        l[r] *= f;
#pragma unroll
        for (int dt = 0; dt < DB * 4; ++dt) o[r][dt] *= f;
      }
      float e[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        e[i] = __builtin_amdgcn_exp2f(fmaf(s[r][i / 4][i % 4], ks, -m[r]));
        if (masked && !(seen >> i & 1)) e[i] = 0.0f;
        l[r] += e[i];
        e[i] *= vs;
        if (masked && !(seen >> i & 1)) e[i] = 0.0f;  // vs may be NaN
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
        p[r][u] = __builtin_bit_cast(bf16x8_t, make_uint4(pack2(e[8 * u], e[8 * u + 1]), pack2(e[8 * u + 2], e[8 * u + 3]),
                                                          pack2(e[8 * u + 4], e[8 * u + 5]), pack2(e[8 * u + 6], e[8 * u + 7])));
    }
#pragma unroll
    for (int dt = 0; dt < DB * 4; ++dt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8_t vf = x.value(dt, u);
#pragma unroll
        for (int r = 0; r < RT; ++r) o[r][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, p[r][u], o[r][dt], 0, 0, 0);
      }
  }
};

// One split of one tile of rows: the waves take its blocks in turn and join at the end.
template <int DB, int RT>
__global__ void __launch_bounds__(kAtnWaves * 64, 2) kv8_attend_kernel(AttendArgs a) {
  constexpr int ROWS = 16 * RT, Dp = DB * 64;
  __shared__ float sml[2][kAtnWaves][ROWS];
  __shared__ __align__(16) float so[kAtnWaves][ROWS][Dp + 4];
  const int tile = blockIdx.x % a.tiles, split = blockIdx.y;
  const int64_t bh = blockIdx.x / a.tiles;
  const int b = static_cast<int>(bh / a.c.H), h = static_cast<int>(bh % a.c.H);
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TileRange tr = tile_range<ROWS>(a, b, tile);
  const int used = tr.used();
  if (split >= used && split > 0) return;
  RowState<DB, RT> st;
  int first_pos = INT32_MAX, last_pos = -1;  // of the tile's queries
  if (used) first_pos = tr.start + tr.i0, last_pos = tr.start + tr.i1 - 1;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = tile * ROWS + r * 16 + (lane & 15), i = row / a.group, hq = h * a.group + row % a.group;
    const bool real = i < tr.i1;
    st.pos[r] = real ? tr.start + i : -1;
    const uint16_t* q = a.q + b * a.qsb + i * a.qss + hq * a.qsh;
#pragma unroll
    for (int hh = 0; hh < DB; ++hh)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int d = hh * 64 + g * 16 + x * 8;
        const V4 w = real && d < a.c.D ? ld16(q + d) : zero16();
        st.q[r][hh][x] = __builtin_bit_cast(bf16x8_t, make_uint4(w.w[0], w.w[1], w.w[2], w.w[3]));
      }
#pragma unroll
    for (int dt = 0; dt < DB * 4; ++dt) st.o[r][dt] = f32x4_t{};
    st.m[r] = kAtnLow;
    st.l[r] = 0.0f;
  }
  if (used) {
    const int whole = tr.end / kKvBlock;  // blocks of codes
    const int bs = tr.b0 + split * tr.per, be = min(tr.b1, bs + tr.per);
    const int8_t* kc = a.c.k + bh * a.c.blocks * kKvBlock * Dp;
    const int8_t* vc = a.c.v + bh * a.c.blocks * kKvBlock * Dp;
    const int ce = min(be, whole);
    auto masked = [&](int blk) {
      return blk * kKvBlock + kKvBlock - 1 > first_pos || (a.window && blk * kKvBlock <= last_pos - a.window);
    };
    int blk = bs + wave;
    CodeBlock<DB> cur, next;
    if (blk < ce) cur.load(kc + (int64_t)blk * kKvBlock * Dp, vc + (int64_t)blk * kKvBlock * Dp);
    for (; blk < ce; blk += kAtnWaves) {
      const int nb = blk + kAtnWaves;
      if (nb < ce) next.load(kc + (int64_t)nb * kKvBlock * Dp, vc + (int64_t)nb * kKvBlock * Dp);
      const float ks = a.c.ks[bh * a.c.blocks + blk] * a.scale, vs = a.c.vs[bh * a.c.blocks + blk];
      st.block(cur, blk, ks, vs, a.window, masked(blk));
      cur = next;
    }
    if (blk < be) {  // the incomplete block
      const TailBlock<DB> tail{a.c.kt + bh * kKvBlock * Dp, a.c.vt + bh * kKvBlock * Dp, tr.end - blk * kKvBlock};
      st.block(tail, blk, a.scale, 1.0f, a.window, true);
    }
  }
  // join the waves
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    st.l[r] += __shfl_xor(st.l[r], 16, 64);
    st.l[r] += __shfl_xor(st.l[r], 32, 64);
    const int row = r * 16 + (lane & 15);
    if (g == 0) {
      sml[0][wave][row] = st.m[r];
      sml[1][wave][row] = st.l[r];
    }
#pragma unroll
    for (int dt = 0; dt < DB * 4; ++dt)
      *reinterpret_cast<float4*>(&so[wave][row][dt * 16 + 4 * g]) =
          make_float4(st.o[r][dt][0], st.o[r][dt][1], st.o[r][dt][2], st.o[r][dt][3]);
  }
  __syncthreads();
  for (int at = threadIdx.x; at < ROWS * (Dp / 4); at += kAtnWaves * 64) {
    const int row = at / (Dp / 4), d = (at - row * (Dp / 4)) * 4;
    float m = kAtnLow, l = 0.0f, o[4] = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kAtnWaves; ++w) m = fmaxf(m, sml[0][w][row]);
#pragma unroll
    for (int w = 0; w < kAtnWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sml[0][w][row] - m);
      const float4 x = *reinterpret_cast<const float4*>(&so[w][row][d]);
      l += f * sml[1][w][row];
      o[0] += f * x.x;
      o[1] += f * x.y;
      o[2] += f * x.z;
      o[3] += f * x.w;
    }
    if (a.splits > 1) {
      const int64_t part = (int64_t)blockIdx.x * a.splits + split;
      *reinterpret_cast<float4*>(a.po + (part * ROWS + row) * Dp + d) = make_float4(o[0], o[1], o[2], o[3]);
      if (d == 0) {
        a.pml[(part * 2 + 0) * ROWS + row] = m;
        a.pml[(part * 2 + 1) * ROWS + row] = l;
      }
    } else {
      const int gr = tile * ROWS + row, i = gr / a.group, hq = h * a.group + gr % a.group;
      if (i < a.n && d < a.c.D) {
        const float f = i < tr.i1 ? 1.0f / l : 0.0f;  // a sum of 0 where every score is -inf: NaN, as 0 / 0
        uint2 w = make_uint2(0, 0);
        if (i < tr.i1) w = make_uint2(pack2(o[0] * f, o[1] * f), pack2(o[2] * f, o[3] * f));
        *reinterpret_cast<uint2*>(a.out + (((int64_t)b * a.n + i) * a.heads + hq) * a.c.D + d) = w;
      }
    }
  }
}

// Joins the splits of one tile.
template <int DB, int RT>
__global__ void __launch_bounds__(256) kv8_join_kernel(AttendArgs a) {
  constexpr int ROWS = 16 * RT, Dp = DB * 64;
  const int tile = blockIdx.x % a.tiles;
  const int64_t bh = blockIdx.x / a.tiles;
  const int b = static_cast<int>(bh / a.c.H), h = static_cast<int>(bh % a.c.H);
  const TileRange tr = tile_range<ROWS>(a, b, tile);
  const int used = tr.used();
  const int64_t part0 = (int64_t)blockIdx.x * a.splits;
  for (int at = threadIdx.x; at < ROWS * (Dp / 4); at += 256) {
    const int row = at / (Dp / 4), d = (at - row * (Dp / 4)) * 4;
    const int gr = tile * ROWS + row, i = gr / a.group, hq = h * a.group + gr % a.group;
    if (i >= a.n || d >= a.c.D) continue;
    float m = kAtnLow, l = 0.0f, o[4] = {0, 0, 0, 0};
    if (i < tr.i1) {
      for (int s = 0; s < used; ++s) m = fmaxf(m, a.pml[((part0 + s) * 2) * ROWS + row]);
      for (int s = 0; s < used; ++s) {
        const float f = __builtin_amdgcn_exp2f(a.pml[((part0 + s) * 2) * ROWS + row] - m);
        const float4 x = *reinterpret_cast<const float4*>(a.po + ((part0 + s) * ROWS + row) * Dp + d);
        l += f * a.pml[((part0 + s) * 2 + 1) * ROWS + row];
        o[0] += f * x.x;
        o[1] += f * x.y;
        o[2] += f * x.z;
        o[3] += f * x.w;
      }
    }
    const float f = 1.0f / l;
    uint2 w = make_uint2(0, 0);
    if (i < tr.i1) w = make_uint2(pack2(o[0] * f, o[1] * f), pack2(o[2] * f, o[3] * f));
    *reinterpret_cast<uint2*>(a.out + (((int64_t)b * a.n + i) * a.heads + hq) * a.c.D + d) = w;
  }
}

template <int DB, int RT>
void launch_attend(const AttendArgs& a, hipStream_t st) {
  const unsigned tiles = static_cast<unsigned>((int64_t)a.c.B * a.c.H * a.tiles);
  kv8_attend_kernel<DB, RT><<<dim3(tiles, a.splits), kAtnWaves * 64, 0, st>>>(a);
  if (a.splits > 1) kv8_join_kernel<DB, RT><<<tiles, 256, 0, st>>>(a);
}

// How a call is cut: rows of a tile and key splits.
struct AttendPlan {
  int rt;
  int64_t tiles;  // of one (sequence, head)
  int splits, chunk;
  size_t bytes;
};
AttendPlan attend_plan(int64_t B, int64_t H, int64_t heads, int64_t Dp, int64_t n, int64_t bound) {
  AttendPlan p;
  const int64_t rows = n * (heads / H);
  p.rt = rows <= 16 || Dp > 128 ? 1 : 2;
  p.tiles = ceil_div(rows, 16 * p.rt);
  const int64_t wgs = B * H * p.tiles, blocks = ceil_div(bound, kKvBlock);
  // enough workgroups for two on every CU, none with less than two blocks for each of its waves
  int64_t s = ceil_div(1024, wgs);
  const int64_t most = ceil_div(blocks, 2 * kAtnWaves);
  if (s > most) s = most;
  if (s < 1) s = 1;
  p.splits = static_cast<int>(s);
  p.chunk = static_cast<int>(blocks > 0 ? ceil_div(blocks, s) : 1);
  p.bytes = s > 1 ? static_cast<size_t>(wgs) * s * (16 * p.rt) * (Dp + 2) * 4 : 0;
  return p;
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" size_t sf_kv8_attend_workspace_size(int64_t batch, int64_t kv_heads, int64_t heads, int64_t head_dim,
                                               int64_t n, int64_t bound) {
  if (batch < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads || head_dim < 1 || n < 1 || bound < 0) return 0;
  return attend_plan(batch, kv_heads, heads, kv_pad(head_dim), n, bound).bytes;
}

extern "C" int sf_kv8_attend(const sf_kv8_cache* cache, const void* q, int64_t q_sb, int64_t q_ss, int64_t q_sh,
                             int64_t n, int64_t heads, float scale, int64_t window, int64_t bound, void* out,
                             void* workspace, size_t workspace_bytes, void* stream) {
  AttendArgs a;
  if (int rc = kv8_cache(cache, "sf_kv8_attend", a.c)) return rc;
  const int64_t cap = a.c.blocks * kKvBlock;
  SF_CHECK_ARG(n >= 0 && n <= cap, "sf_kv8_attend: %lld rows for a capacity of %lld", (long long)n, (long long)cap);
  SF_CHECK_ARG(heads >= a.c.H && heads < 65536 && heads % a.c.H == 0,
               "sf_kv8_attend: %lld query heads for %d key-value heads", (long long)heads, a.c.H);
  SF_CHECK_ARG(scale > 0.0f && scale <= 3.0e38f, "sf_kv8_attend: scale %g must be positive and finite", scale);
  SF_CHECK_ARG(window >= 0, "sf_kv8_attend: window %lld", (long long)window);
  SF_CHECK_ARG(bound >= 0 && bound <= cap, "sf_kv8_attend: bound %lld of a capacity of %lld", (long long)bound,
               (long long)cap);
  if (n == 0) return SF_OK;
  SF_CHECK_ARG(q && out, "sf_kv8_attend: null pointer");
  SF_CHECK_ARG((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 == 0 &&
                   (q_sb | q_ss | q_sh) % 8 == 0,
               "sf_kv8_attend: rows must be 16-byte aligned");
  const AttendPlan p = attend_plan(a.c.B, a.c.H, heads, a.c.Dp, n, bound);
  SF_CHECK_ARG(workspace_bytes >= p.bytes && (p.bytes == 0 || workspace), "sf_kv8_attend: workspace of %zu bytes, %zu needed",
               workspace_bytes, p.bytes);
  SF_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "sf_kv8_attend: workspace must be 16-byte aligned");
  const int64_t wgs = (int64_t)a.c.B * a.c.H * p.tiles;
  SF_CHECK_ARG(wgs < (1ll << 31) && n * (heads / a.c.H) < (1ll << 30), "sf_kv8_attend: too many rows");
  a.q = static_cast<const uint16_t*>(q);
  a.qsb = q_sb, a.qss = q_ss, a.qsh = q_sh;
  a.out = static_cast<uint16_t*>(out);
  a.n = static_cast<int>(n);
  a.heads = static_cast<int>(heads);
  a.group = static_cast<int>(heads / a.c.H);
  a.window = static_cast<int>(window < cap ? window : 0);
  a.scale = scale * kAtnLog2e;
  a.tiles = static_cast<int>(p.tiles);
  a.splits = p.splits;
  a.chunk = p.chunk;
  a.po = static_cast<float*>(workspace);
  a.pml = a.po ? a.po + wgs * p.splits * 16 * p.rt * a.c.Dp : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (a.c.Dp / 64 * 10 + p.rt) {
    case 11: launch_attend<1, 1>(a, st); break;
    case 12: launch_attend<1, 2>(a, st); break;
    case 21: launch_attend<2, 1>(a, st); break;
    case 22: launch_attend<2, 2>(a, st); break;
    case 31: launch_attend<3, 1>(a, st); break;
    case 41: launch_attend<4, 1>(a, st); break;
  }
  return launch_status("sf_kv8_attend");
}
