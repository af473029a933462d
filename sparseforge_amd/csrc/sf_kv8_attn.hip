// Attention of the newest tokens over the 8-bit cache (layout: sf_kv8.hpp):
//   o_i = softmax_j(scale q_i k_j) v_j over the keys j <= i, and j > i - window where there is a window,
// with i, j positions of a sequence.  A query that sees no key (its sequence has ended) gives 0.
//
// The query heads that share a key-value head are rows of one product with it: row r of (sequence, key-value head) is
// query r / group of head r % group.  A wave takes 16 RT rows over whole blocks of 64 keys, one pass with a running
// maximum and sum.  Both products are v_mfma_f32_16x16x32_bf16 on codes converted to bf16, which is exact (8 significant
// bits), with f32 scores, sums and outputs.  The key scale multiplies the scores with the softmax's factor; the value
// scale enters the exponent (BlockScale).
//
// The probabilities round to bf16 as operands of the second product, which moves an output by 2^-8 of its terms at most,
// as much as storing it in bf16 does; the sums are of the rounded ones.  f16 would hold three bits more at the same rate,
// but nothing below 2^-39 of the largest (2^-25 whole): an output that only small weights make, because the largest has a
// code of 0 there, would come out wrong by more than its rounding.  Two parts in bf16, 16 bits, take the single-token form
// 10 to 25 % longer; the incomplete block's weights, one block of many, are such.
//
// A row's running maximum is raised only when a score passes it by 8 (in log2): probabilities up to 2^8 cost nothing in
// f32 or bf16, and most blocks need no exchange between lanes.
//
// Two forms:
//   up to 16 rows (32 with heads of at most 128): kv8_attend_kernel.  Bound by reading the codes, 2 D bytes per key and
//     key-value head.  Each wave takes blocks of its own, converted in registers, and the keys are split over workgroups;
//     kv8_join_kernel joins them.  Conversion and softmax, about 500 vector instructions a block and wave, stay under
//     the memory's time.  Measured: 32 sequences of 1024 .. 4096, 32 heads of 128: 112 us, 5.8 TB/s; 2 of 131071, 32
//     heads over 8: 84 us + 5 us for the join, 6.0 TB/s; one of 33 tokens, 32 heads of 64: 5.4 us.
//   more: kv8_chunk_kernel.  Bound by power: the matrix unit is busy in 51 % of its cycles and the vector unit beside it
//     (an exponential, its argument, a maximum and half a conversion to bf16 for each score) in 56 %, and the clock falls
//     to 1.9 .. 2.1 GHz under that load.  Measured: 2048 tokens over 18001, 32 heads of 128 over 8: 495 to 526 us from
//     one card to another in a row of calls, 1083 to 1150 TFLOP/s (554 to 610 us in the first dozen, while the clock
//     settles), where a large library product of bf16 reaches 1130 to 1330; 32 heads of 64 over 18048: 342 us, 835
//     TFLOP/s; from an empty cache, where the tiles are unequal, 32 heads of 128: 64 us, 540 TFLOP/s.
#include "sf_kv8.hpp"

namespace sf {
namespace {

constexpr int kAtnWaves = 4;
constexpr float kAtnLog2e = 1.4426950408889634f;
constexpr float kAtnLow = -3.0e38f;  // below every score that counts
constexpr float kAtnSlack = 8.0f;
constexpr float kAtnHuge = 0x1p40f;
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct AttendArgs {
  KvCache c;
  const uint16_t* q;  // [B, n, heads, D]
  int64_t qsb, qss, qsh;
  uint16_t* out;      // [B, n, heads, D] contiguous
  int n, heads, group;
  int window;         // 0: none
  float scale;        // times log2 e
  int rows, tiles;    // rows of a workgroup, and how many times that a (sequence, head) has
  int splits, chunk;  // key blocks of a workgroup: at least `chunk`
  float* po;          // [B H tiles][splits][rows][Dp] outputs over a split's keys alone
  float* pml;         // [B H tiles][splits][2][rows] maxima, sums
};

// A scale, in a vector register until it is used: as a scalar, which the compiler makes of what all lanes load alike, it
// would be waited for where it is loaded, a block early (10 % of a chunk with heads of 64).
__device__ __forceinline__ float ld_scale(const float* p) {
  int same = 0;
  asm("" : "+v"(same));
  return p[same];
}

// What a tile of rows sees.
struct TileRange {
  int start, end;          // newest tokens
  int i0, i1;              // queries of the tile, [i0, i1); none if i0 >= i1
  int b0, b1;              // key blocks, [b0, b1)
  int per;                 // blocks of a split
  __device__ __forceinline__ int used() const { return b1 > b0 ? (b1 - b0 + per - 1) / per : 0; }
};
__device__ __forceinline__ TileRange tile_range(const AttendArgs& a, int rows, int b, int tile) {
  TileRange r;
  kv_range(a.c, b, a.n, r.start, r.end);
  const int cnt = r.end - r.start;
  r.i0 = tile * rows / a.group;
  r.i1 = min(cnt, (tile * rows + rows - 1) / a.group + 1);
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

// Workgroup -> tile: those of one (sequence, head) on one XCD, whose L2 then holds its codes, longest rows first.
__device__ __forceinline__ void tile_of(const AttendArgs& a, int64_t& bh, int& tile) {
  const int64_t id = blockIdx.x, all = (int64_t)a.c.B * a.c.H;
  if (all % kXcds == 0) {
    const int64_t r = id / kXcds;
    bh = r / a.tiles * kXcds + id % kXcds;
    tile = static_cast<int>(r % a.tiles);
  } else {
    bh = id / a.tiles;
    tile = static_cast<int>(id % a.tiles);
  }
  tile = a.tiles - 1 - tile;
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

// 16 bytes that nothing else of the call reads: past the caches (5.1 -> 5.8 TB/s over whole caches of codes).
__device__ __forceinline__ V4 ld16_once(const void* p) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 x = __builtin_nontemporal_load(static_cast<const u32x4*>(p));
  V4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o.w[i] = x[i];
  return o;
}

// Operands of a block of codes, in registers: chunk (hh, t) of keys, dim tile dt of values.
template <int DB>
struct CodeBlock {
  V4 k[DB * 4], v[DB * 4];
  __device__ __forceinline__ static void load(V4 (&w)[DB * 4], const int8_t* codes) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < DB * 4; ++i) w[i] = ld16_once(codes + i * 1024 + (lane & 15) * 64 + (lane >> 4) * 16);
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

// What a block's scales do to its scores and probabilities.  The value scale, in the wave's terms (RowState::refer), goes
// into the exponent, which costs nothing for each key, and the sum of a row takes it out again.  A scale of 0 has codes
// of 0, for which any other does as well.
struct BlockScale {
  float ks;      // of the scores, with log2 e; positive
  float v;       // of the values, 0 where any does
  float lv, rv;  // log2 of the value scale in the wave's terms, and its reciprocal
  bool far;      // so small that the sum is taken apart
  bool nan;      // a block of NaN: its scores become NaN
  __device__ __forceinline__ BlockScale(float k, float v, float scale)
      : v(v > 0.0f ? v : 0.0f), lv(0.0f), rv(1.0f), far(false) {
    nan = k != k;  // both are
    // neither 0, which makes NaN of a hidden score's -inf, nor infinite, which does of a score of 0
    ks = k > 0.0f ? __builtin_amdgcn_fmed3f(k * scale, 0x1p-149f, 3.0e38f) : 1.0f;
  }
};

// A wave's rows: queries, running softmax and output, transposed (lane: row lane % 16 of each 16).
template <int DB, int RT>
struct RowState {
  bf16x8_t q[RT][DB][2];
  f32x4_t o[RT][DB * 4];
  float m[RT], l[RT];
  int pos[RT];  // position of the row's query, -1: no such row
  bool huge;    // o is in terms of kAtnHuge

  // The queries of rows row0 + 16 r + lane % 16 of key-value head h; rows past the tile's queries are zeros.
  __device__ __forceinline__ void start(const AttendArgs& a, const TileRange& tr, int b, int h, int row0) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = row0 + r * 16 + (lane & 15), i = row / a.group, hq = h * a.group + row % a.group;
      const bool real = i < tr.i1;
      pos[r] = real ? tr.start + i : -1;
      const uint16_t* src = a.q + b * a.qsb + i * a.qss + hq * a.qsh;
#pragma unroll
      for (int hh = 0; hh < DB; ++hh)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int d = hh * 64 + g * 16 + x * 8;
          const V4 w = real && d < a.c.D ? ld16(src + d) : zero16();
          q[r][hh][x] = __builtin_bit_cast(bf16x8_t, make_uint4(w.w[0], w.w[1], w.w[2], w.w[3]));
        }
#pragma unroll
      for (int dt = 0; dt < DB * 4; ++dt) o[r][dt] = f32x4_t{};
      m[r] = kAtnLow;
      l[r] = 0.0f;
    }
    huge = false;
  }

  // The block's value scale in the wave's terms.  A probability (up to 2^8), a code and the number of keys take up to 40
  // powers of two beside it, so from the first scale of 2^80 on o is held in terms of 2^40: the largest values of bf16 stay
  // inside the range of floats in products and sums, as their mean does, and rows that do not see them keep theirs (down
  // to 2^-86).  Probabilities times scales below 2^-64 may leave the floats: their sum is taken without the scale.
  __device__ __forceinline__ void refer(BlockScale& sc) {
    const float v = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(sc.v)));
    if (!(v > 0.0f)) return;
    if (v >= 0x1p80f && !huge) {
      huge = true;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int dt = 0; dt < DB * 4; ++dt) o[r][dt] *= 1.0f / kAtnHuge;
    }
    const float x = huge ? v * (1.0f / kAtnHuge) : v;
    sc.far = x < 0x1p-64f;
    sc.lv = __builtin_amdgcn_logf(x);  // of next to nothing: -inf, and the block adds nothing
    sc.rv = sc.far ? 0.0f : __builtin_amdgcn_rcpf(x);
  }

  // Scores of a block that some row does not see whole, or that is NaN.
  __device__ __forceinline__ void hide(int r, f32x4_t (&s)[4], int blk, bool nan, int window) {
    const int g = (threadIdx.x & 63) >> 4;
    const int hi = pos[r] - blk * kKvBlock - 4 * g, lo = window ? hi - window : -1 - 4 * g;  // seen: lo < key <= hi
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = 16 * (i / 4) + i % 4;
      float x = s[i / 4][i % 4];
      x = nan ? __builtin_nanf("") : x;
      s[i / 4][i % 4] = key <= hi && key > lo ? x : -INFINITY;
    }
  }

  template <class Block>
  __device__ __forceinline__ void scores(const Block& x, f32x4_t (&s)[RT][4]) const {
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
  }

  // What is rare before a block's probabilities: rows that do not see it whole, a maximum that has to rise, a value
  // scale far from 1.
  __device__ __forceinline__ void settle(f32x4_t (&s)[RT][4], int blk, BlockScale& sc, int window, bool masked) {
    refer(sc);
    if (masked || sc.nan) {
#pragma unroll
      for (int r = 0; r < RT; ++r) hide(r, s[r], blk, sc.nan, window);
    }
    float mx[RT];
    bool rise = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      mx[r] = s[r][0][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx[r] = fmaxf(mx[r], s[r][i / 4][i % 4]);
      mx[r] *= sc.ks;
      rise |= mx[r] > m[r] + kAtnSlack;
    }
    if (__builtin_amdgcn_ballot_w64(rise)) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float x = fmaxf(mx[r], __shfl_xor(mx[r], 16, 64));
        x = fmaxf(x, __shfl_xor(x, 32, 64));
        const float mn = fmaxf(m[r], x), f = __builtin_amdgcn_exp2f(m[r] - mn);
        m[r] = mn;
        l[r] *= f;
#pragma unroll
        for (int dt = 0; dt < DB * 4; ++dt) o[r][dt] *= f;
      }
    }
    if (sc.far) {
      f32x4_t e[4];
#pragma unroll
      for (int r = 0; r < RT; ++r) l[r] += sum(s[r], sc, -m[r], e);
    }
  }

  // The exponentials of a row's scores, and their sum.
  __device__ __forceinline__ static float sum(const f32x4_t (&s)[4], const BlockScale& sc, float off, f32x4_t (&e)[4]) {
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) x += e[i / 4][i % 4] = __builtin_amdgcn_exp2f(fmaf(s[i / 4][i % 4], sc.ks, off));
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
  }

  // Probabilities times the value scale, as operands of the second product.
  __device__ __forceinline__ void weights(const f32x4_t (&s)[RT][4], const BlockScale& sc, bf16x8_t (&p)[RT][2]) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float off = sc.lv - m[r];
      float e[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(s[r][i / 4][i % 4], sc.ks, off));
#pragma unroll
      for (int u = 0; u < 2; ++u)
        p[r][u] = __builtin_bit_cast(bf16x8_t, make_uint4(pack2(e[8 * u], e[8 * u + 1]), pack2(e[8 * u + 2], e[8 * u + 3]),
                                                          pack2(e[8 * u + 4], e[8 * u + 5]), pack2(e[8 * u + 6], e[8 * u + 7])));
    }
  }

  // The sums of the rows' probabilities, as a product with ones: the vector unit has more to do than the matrix unit,
  // and the sums are those of the rounded probabilities that the output takes.
  __device__ __forceinline__ void sums(const bf16x8_t (&p)[RT][2], const BlockScale& sc) {
    const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u));
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      f32x4_t t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[r][0], f32x4_t{}, 0, 0, 0);
      t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[r][1], t, 0, 0, 0);
      l[r] = fmaf(t[0], sc.rv, l[r]);
    }
  }

  // Weights in one part or in several.
  template <class Block, class... Parts>
  __device__ __forceinline__ void output(const Block& x, const Parts&... parts) {
#pragma unroll
    for (int dt = 0; dt < DB * 4; ++dt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8_t vf = x.value(dt, u);
#pragma unroll
        for (int r = 0; r < RT; ++r)
          ((o[r][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, parts[r][u], o[r][dt], 0, 0, 0)), ...);
      }
  }

  // The output over the wave's keys: o over its sum, in terms of 1.  Rows that have met no key are 0.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float f = l[r] == 0.0f ? 0.0f : (huge ? kAtnHuge : 1.0f) / l[r];
#pragma unroll
      for (int dt = 0; dt < DB * 4; ++dt) o[r][dt] *= f;
    }
  }

  // The incomplete block, which comes last, and finish(): its values, any bf16 numbers, are products with weights that
  // are final, at most 1, in a high and a low part (16 bits together; one block, so this costs next to nothing).  s: its
  // scores.
  template <class Block>
  __device__ __forceinline__ void last(const Block& x, f32x4_t (&s)[RT][4], int blk, float scale, int window) {
    BlockScale sc(1.0f, 0.0f, scale);
    settle(s, blk, sc, window, true);
#pragma unroll
    for (int r = 0; r < RT; ++r) l[r] += sum(s[r], sc, -m[r], s[r]);
    finish();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float f = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
#pragma unroll
      for (int t = 0; t < 4; ++t) s[r][t] *= f;
    }
    bf16x8_t p[2][RT][2];
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f32x4_t& e = s[r][2 * u + i / 2];
            w[i] = pack2(e[i % 2 * 2], e[i % 2 * 2 + 1]);
            e[i % 2 * 2] -= lo_f(w[i]);
            e[i % 2 * 2 + 1] -= hi_f(w[i]);
          }
          p[part][r][u] = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
        }
    output(x, p[0], p[1]);
  }

  // scores(x, next), weights(s, sc, p), sums(p, sc) and output(x, p) as one stream of instructions: products of the next
  // scores between exponentials, and `rest(i, n)`, i = 0 .. n - 1, between products of the output.  The compiler may
  // reorder four fragments' worth of it at a time (the whole of it: 760 us where this takes 536, single ones 555).  The
  // products of the output, which have little beside them, go before what the other wave of the SIMD has.
  template <class Block, class Rest>
  __device__ __forceinline__ void turn(const Block& x, const f32x4_t (&s)[RT][4], f32x4_t (&next)[RT][4],
                                       const BlockScale& sc, const Rest& rest) {
    constexpr int F = DB * 8;  // fragments of keys, and of values
    float off[RT];
    uint32_t pw[RT][8];
    constexpr int A = 4;  // fragments read ahead
    bf16x8_t f[A + 1];
    auto key = [&](int i) { return x.key(i / 2 % DB, i / (2 * DB), i % 2); };
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      off[r] = sc.lv - m[r];
#pragma unroll
      for (int t = 0; t < 4; ++t) next[r][t] = f32x4_t{};
    }
#pragma unroll
    for (int i = 0; i < A; ++i) f[i] = key(i);
#pragma unroll
    for (int i = 0; i < F; ++i) {
      if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);
      f[(i + A) % (A + 1)] = i + A < F ? key(i + A) : x.value((i + A - F) / 2, (i + A - F) % 2);
#pragma unroll
      for (int r = 0; r < RT; ++r)
        next[r][i / (2 * DB)] =
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[i % (A + 1)], q[r][i / 2 % DB][i % 2], next[r][i / (2 * DB)], 0, 0, 0);
      // pairs of weights: 8 RT of them over F places
#pragma unroll
      for (int j = i * 8 * RT / F; j < (i + 1) * 8 * RT / F; ++j) {
        const int r = j / 8, e = j % 8 * 2;
        const float a = __builtin_amdgcn_exp2f(fmaf(s[r][e / 4][e % 4], sc.ks, off[r]));
        const float b = __builtin_amdgcn_exp2f(fmaf(s[r][e / 4][e % 4 + 1], sc.ks, off[r]));
        pw[r][j % 8] = pack2(a, b);
      }
    }
    bf16x8_t p[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        p[r][u] = __builtin_bit_cast(bf16x8_t, make_uint4(pw[r][4 * u], pw[r][4 * u + 1], pw[r][4 * u + 2], pw[r][4 * u + 3]));
    __builtin_amdgcn_s_setprio(1);
    sums(p, sc);
#pragma unroll
    for (int i = 0; i < F; ++i) {
      if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);
      if (i + A < F) f[(F + i + A) % (A + 1)] = x.value((i + A) / 2, (i + A) % 2);
#pragma unroll
      for (int r = 0; r < RT; ++r)
        o[r][i / 2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[(F + i) % (A + 1)], p[r][i % 2], o[r][i / 2], 0, 0, 0);
      rest(i, F);
    }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
  }
};

// Waves a SIMD that the registers hold without spilling (heads of 256 run 2 waves 20 % slower: they spill).
constexpr int attend_waves(int db, int rt) { return db * rt == 1 ? 4 : db == 2 && rt == 1 ? 3 : db == 4 ? 1 : 2; }

// Few rows: one split of one tile.  The waves take its blocks in turn and join at the end.
template <int DB, int RT>
__global__ void __launch_bounds__(kAtnWaves * 64, attend_waves(DB, RT)) kv8_attend_kernel(AttendArgs a) {
  constexpr int ROWS = 16 * RT, Dp = DB * 64;
  __shared__ float sml[2][kAtnWaves][ROWS];
  __shared__ __align__(16) float so[kAtnWaves][ROWS][Dp + 4];
  const int tile = blockIdx.x % a.tiles, split = blockIdx.y;
  const int64_t bh = blockIdx.x / a.tiles;
  const int b = static_cast<int>(bh / a.c.H), h = static_cast<int>(bh % a.c.H);
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TileRange tr = tile_range(a, ROWS, b, tile);
  const int used = tr.used();
  if (split >= used && split > 0) return;
  RowState<DB, RT> st;
  st.start(a, tr, b, h, tile * ROWS);
  const int first_pos = tr.start + tr.i0, last_pos = tr.start + tr.i1 - 1;  // of the tile's queries
  if (used) {
    const int whole = tr.end / kKvBlock;  // blocks of codes
    const int bs = tr.b0 + split * tr.per, be = min(tr.b1, bs + tr.per);
    const int8_t* kc = a.c.k + bh * a.c.blocks * kKvBlock * Dp;
    const int8_t* vc = a.c.v + bh * a.c.blocks * kKvBlock * Dp;
    const int ce = min(be, whole);
    auto masked = [&](int blk) {
      return blk * kKvBlock + kKvBlock - 1 > first_pos || (a.window && blk * kKvBlock <= last_pos - a.window);
    };
    // A block's keys are replaced by the next's once its scores are there, its values after the output: half a block
    // is always on its way, and the registers of a second block hold another wave instead.
    const float* ks = a.c.ks + bh * a.c.blocks;
    const float* vs = a.c.vs + bh * a.c.blocks;
    int blk = bs + wave;
    CodeBlock<DB> x;
    float k1 = 1.0f, v1 = 1.0f;  // the next block's scales
    if (blk < ce) {
      x.load(x.k, kc + (int64_t)blk * kKvBlock * Dp);
      x.load(x.v, vc + (int64_t)blk * kKvBlock * Dp);
      k1 = ld_scale(ks + blk), v1 = ld_scale(vs + blk);
    }
    for (; blk < ce; blk += kAtnWaves) {
      const int64_t next = blk + kAtnWaves;
      f32x4_t s[RT][4];
      bf16x8_t p[RT][2];
      st.scores(x, s);
      BlockScale sc(k1, v1, a.scale);
      if (next < ce) {
        x.load(x.k, kc + next * kKvBlock * Dp);
        k1 = ld_scale(ks + next), v1 = ld_scale(vs + next);
      }
      st.settle(s, blk, sc, a.window, masked(blk));
      st.weights(s, sc, p);
      st.sums(p, sc);
      st.output(x, p);
      if (next < ce) x.load(x.v, vc + next * kKvBlock * Dp);
    }
    if (blk < be) {  // the incomplete block
      const TailBlock<DB> tail{a.c.kt + bh * kKvBlock * Dp, a.c.vt + bh * kKvBlock * Dp, tr.end - blk * kKvBlock};
      f32x4_t s[RT][4];
      st.scores(tail, s);
      st.last(tail, s, blk, a.scale, a.window);
    } else {
      st.finish();
    }
  }
  // join the waves
#pragma unroll
  for (int r = 0; r < RT; ++r) {
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
    float m = kAtnLow, l = 0.0f, o[4] = {0, 0, 0, 0}, c[kAtnWaves];
#pragma unroll
    for (int w = 0; w < kAtnWaves; ++w) m = fmaxf(m, sml[0][w][row]);
#pragma unroll
    for (int w = 0; w < kAtnWaves; ++w) {
      c[w] = __builtin_amdgcn_exp2f(sml[0][w][row] - m) * sml[1][w][row];
      l += c[w];
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int w = 0; w < kAtnWaves; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(&so[w][row][d]);
      o[0] += c[w] * f * x.x;
      o[1] += c[w] * f * x.y;
      o[2] += c[w] * f * x.z;
      o[3] += c[w] * f * x.w;
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
        const float none = l == 0.0f ? __builtin_nanf("") : 0.0f;  // every score is -inf: NaN, as 0 / 0
        uint2 w = make_uint2(0, 0);
        if (i < tr.i1) w = make_uint2(pack2(o[0] + none, o[1] + none), pack2(o[2] + none, o[3] + none));
        *reinterpret_cast<uint2*>(a.out + (((int64_t)b * a.n + i) * a.heads + hq) * a.c.D + d) = w;
      }
    }
  }
}

// Many rows: the waves of a workgroup share the blocks.  Each converts its part of a block into LDS once, in the
// operands' order (a fragment of 16 bytes a lane, 1 KB, is written and read in a row, without bank conflicts), and
// takes all of it for its own 16 RT rows.  In a turn, the scores of the next block are products on the matrix unit
// while the probabilities of this one are exponentials on the vector unit; a block after, its codes loaded at the
// turn's start, is converted at its end.  Keys are staged one block further than values.
template <int DB, int RT, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, 2) kv8_chunk_kernel(AttendArgs a) {
  constexpr int ROWS = 16 * RT * WAVES, Dp = DB * 64, N = DB * 8 / WAVES;  // chunks of a lane: keys', then values'
  // A barrier every other turn where there is room for it (4 % faster): a turn then stages what is read two turns later,
  // into a slot whose block was read before the last barrier.
  constexpr bool PAIR = WAVES == 8 && DB <= 2;
  constexpr int AHEAD = PAIR ? 3 : 2, SLOTS = PAIR ? 4 : 2;
  __shared__ __align__(16) unsigned char lds[SLOTS][DB * 16][1024];  // fragments (hh, t, a) of keys, (dt, u) of values
  int tile, split = blockIdx.y;
  int64_t bh;
  tile_of(a, bh, tile);
  const int b = static_cast<int>(bh / a.c.H), h = static_cast<int>(bh % a.c.H);
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TileRange tr = tile_range(a, ROWS, b, tile);
  const int used = tr.used();
  if (split >= used && split > 0) return;
  const int row0 = tile * ROWS + wave * 16 * RT;
  RowState<DB, RT> st;
  st.start(a, tr, b, h, row0);
  // positions of the wave's queries
  const int first_pos = tr.start + row0 / a.group;
  const int last_pos = row0 / a.group < tr.i1 ? tr.start + min(tr.i1 - 1, (row0 + 16 * RT - 1) / a.group) : -kKvBlock;
  if (used) {
    const int whole = tr.end / kKvBlock;
    const int bs = tr.b0 + split * tr.per, be = min(tr.b1, bs + tr.per), ce = min(be, whole);
    const int8_t* kc = a.c.k + bh * a.c.blocks * kKvBlock * Dp;
    const int8_t* vc = a.c.v + bh * a.c.blocks * kKvBlock * Dp;
    const float* ks = a.c.ks + bh * a.c.blocks;
    const float* vs = a.c.vs + bh * a.c.blocks;
    const int coded = max(bs, ce - 1);  // the last block of codes here, or any that exists
    const TailBlock<DB> tail{a.c.kt + bh * kKvBlock * Dp, a.c.vt + bh * kKvBlock * Dp, tr.end - whole * kKvBlock};
    V4 w[N];
    // Chunk c of DB * 8 (codes of keys, then of values) of blocks kb and vb; past the codes it is read for nothing.
    auto load = [&](int kb, int vb) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = j * WAVES + wave;
        const int8_t* src = c < DB * 4 ? kc + c * 1024 : vc + (c - DB * 4) * 1024;
        w[j] = ld16(src + (int64_t)min(c < DB * 4 ? kb : vb, coded) * kKvBlock * Dp + (lane & 15) * 64 + g * 16);
      }
    };
    auto stage_half = [&](int j, int x, int kb, int vb) {
      const int c = j * WAVES + wave;
      *reinterpret_cast<bf16x8_t*>(&lds[(c < DB * 4 ? kb : vb) & (SLOTS - 1)][2 * c + x][lane * 16]) =
          codes_to_bf16(w[j].w[2 * x], w[j].w[2 * x + 1]);
    };
    auto stage = [&](int kb, int vb) {
#pragma unroll
      for (int j = 0; j < 2 * N; ++j) stage_half(j / 2, j % 2, kb, vb);
    };
    auto stage_tail = [&](int kb, int vb) {
      if (kb != whole && vb != whole) return;
#pragma unroll 1
      for (int j = 0; j < 2 * N; ++j) {
        const int c = j / 2 * WAVES + wave, x = j % 2;
        if ((c < DB * 4 ? kb : vb) != whole) continue;
        *reinterpret_cast<bf16x8_t*>(&lds[whole & (SLOTS - 1)][2 * c + x][lane * 16]) =
            c < DB * 4 ? tail.key(c / 4, c % 4, x) : tail.value(c - DB * 4, x);
      }
    };
    struct {
      const unsigned char* k;
      const unsigned char* v;
      __device__ __forceinline__ bf16x8_t key(int hh, int t, int x) const {
        return *reinterpret_cast<const bf16x8_t*>(k + ((hh * 4 + t) * 2 + x) * 1024);
      }
      __device__ __forceinline__ bf16x8_t value(int dt, int u) const {
        return *reinterpret_cast<const bf16x8_t*>(v + (DB * 8 + dt * 2 + u) * 1024);
      }
    } frags;
    // blocks that some row of this wave sees
    const int from = a.window ? min(be, max(bs, (first_pos - a.window + 1) / kKvBlock)) : bs;
    const int to = max(from, min(be, last_pos / kKvBlock + 1));
#pragma unroll 1
    for (int i = 0; i < AHEAD - 1; ++i) {
      load(bs + i, bs);
      stage(bs + i, bs);
      stage_tail(bs + i, bs);
    }
    int blk = bs - 1;
    auto meet = [&] {
      if (!PAIR || ((blk ^ bs) & 1)) __syncthreads();
    };
    // Turn blk: the block's own products after the next one's scores.
    auto turn_of_others = [&] {
      meet();
      load(blk + AHEAD, blk + AHEAD - 1);
      stage(blk + AHEAD, blk + AHEAD - 1);
      stage_tail(blk + AHEAD, blk + AHEAD - 1);
    };
    for (; blk < from - 1; ++blk) turn_of_others();
    f32x4_t s[RT][4];
    if (to > from) {
      meet();
      load(blk + AHEAD, blk + AHEAD - 1);
      frags.k = &lds[from & (SLOTS - 1)][0][lane * 16];
      st.scores(frags, s);
      stage(blk + AHEAD, blk + AHEAD - 1);
      stage_tail(blk + AHEAD, blk + AHEAD - 1);
      float k1 = ld_scale(ks + min(from, coded)), v1 = ld_scale(vs + min(from, coded));  // the next block's scales
      for (++blk; blk < min(to, whole); ++blk) {
        meet();  // every wave is done with what this turn overwrites
        load(blk + AHEAD, blk + AHEAD - 1);
        BlockScale sc(k1, v1, a.scale);
        k1 = ld_scale(ks + min(blk + 1, coded)), v1 = ld_scale(vs + min(blk + 1, coded));
        st.settle(s, blk, sc, a.window,
                  blk * kKvBlock + kKvBlock - 1 > first_pos || (a.window && blk * kKvBlock <= last_pos - a.window));
        frags.k = &lds[(blk + 1) & (SLOTS - 1)][0][lane * 16];
        frags.v = &lds[blk & (SLOTS - 1)][0][lane * 16];
        f32x4_t next[RT][4];  // past the last block: of what lies there, unused
        st.turn(frags, s, next, sc, [&](int i, int n) {
#pragma unroll
          for (int j = i * 2 * N / n; j < (i + 1) * 2 * N / n; ++j) stage_half(j / 2, j % 2, blk + AHEAD, blk + AHEAD - 1);
        });
        stage_tail(blk + AHEAD, blk + AHEAD - 1);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int t = 0; t < 4; ++t) s[r][t] = next[r][t];
      }
      if (blk < to) {  // the incomplete block, the last of all: nothing is staged after it
        meet();
        frags.v = &lds[blk & (SLOTS - 1)][0][lane * 16];
        st.last(frags, s, blk, a.scale, a.window);
        ++blk;
      } else {
        st.finish();
      }
    }
    for (; blk < be; ++blk) turn_of_others();
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = row0 + r * 16 + (lane & 15), i = row / a.group, hq = h * a.group + row % a.group;
    if (a.splits > 1) {
      const int64_t part = (bh * a.tiles + tile) * a.splits + split;
      const int tr_row = row - tile * ROWS;
#pragma unroll
      for (int dt = 0; dt < DB * 4; ++dt)
        *reinterpret_cast<float4*>(a.po + (part * ROWS + tr_row) * Dp + dt * 16 + 4 * g) =
            make_float4(st.o[r][dt][0], st.o[r][dt][1], st.o[r][dt][2], st.o[r][dt][3]);
      if (g == 0) {
        a.pml[(part * 2 + 0) * ROWS + tr_row] = st.m[r];
        a.pml[(part * 2 + 1) * ROWS + tr_row] = st.l[r];
      }
    } else if (i < a.n) {
      uint16_t* dst = a.out + (((int64_t)b * a.n + i) * a.heads + hq) * a.c.D;
      const float none = st.l[r] == 0.0f ? __builtin_nanf("") : 0.0f;  // every score is -inf: NaN, as 0 / 0
#pragma unroll
      for (int dt = 0; dt < DB * 4; ++dt) {
        const int d = dt * 16 + 4 * g;
        if (d < a.c.D)
          *reinterpret_cast<uint2*>(dst + d) =
              i < tr.i1 ? make_uint2(pack2(st.o[r][dt][0] + none, st.o[r][dt][1] + none),
                                     pack2(st.o[r][dt][2] + none, st.o[r][dt][3] + none))
                        : make_uint2(0, 0);
      }
    }
  }
}

// Joins the splits of output rows: `teams` groups of Dp / 4 threads take those of one row in turn.
template <int DB>
__global__ void __launch_bounds__(256) kv8_join_kernel(AttendArgs a, int teams) {
  constexpr int L = DB * 16, G = DB == 3 ? 4 : 256 / L, Dp = DB * 64;
  __shared__ __align__(16) float so[G][Dp + 4];
  __shared__ float sml[2][G];
  const int t = threadIdx.x, grp = t / L, team = grp % teams, first = grp - team;
  const int64_t out_row = (int64_t)blockIdx.x * (G / teams) + grp / teams;
  const bool real = grp < G && out_row < (int64_t)a.c.B * a.n * a.heads;
  const int hq = static_cast<int>(out_row % a.heads);
  const int64_t bi = real ? out_row / a.heads : 0;
  const int b = static_cast<int>(bi / a.n), i = static_cast<int>(bi % a.n);
  const int gr = i * a.group + hq % a.group, tile = gr / a.rows, row = gr - tile * a.rows;
  const TileRange tr = tile_range(a, a.rows, b, tile);
  const int used = i < tr.i1 ? tr.used() : 0, d = (t - grp * L) * 4;
  const int64_t part0 = (((int64_t)b * a.c.H + hq / a.group) * a.tiles + tile) * a.splits;
  float m = kAtnLow, l = 0.0f, o[4] = {0, 0, 0, 0};
  if (real) {
#pragma unroll 4
    for (int s = team; s < used; s += teams) {
      const float ms = a.pml[(part0 + s) * 2 * a.rows + row], ls = a.pml[((part0 + s) * 2 + 1) * a.rows + row];
      const float4 x = *reinterpret_cast<const float4*>(a.po + ((part0 + s) * a.rows + row) * Dp + d);
      const float mn = fmaxf(m, ms), c0 = __builtin_amdgcn_exp2f(m - mn) * l, c1 = __builtin_amdgcn_exp2f(ms - mn) * ls;
      m = mn;
      l = c0 + c1;
      const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(l), f0 = c0 * f, f1 = c1 * f;
      o[0] = o[0] * f0 + x.x * f1;
      o[1] = o[1] * f0 + x.y * f1;
      o[2] = o[2] * f0 + x.z * f1;
      o[3] = o[3] * f0 + x.w * f1;
    }
    *reinterpret_cast<float4*>(&so[grp][d]) = make_float4(o[0], o[1], o[2], o[3]);
    if (d == 0) {
      sml[0][grp] = m;
      sml[1][grp] = l;
    }
  }
  __syncthreads();
  if (!real || team != 0 || d >= a.c.D) return;
  m = kAtnLow;
  l = o[0] = o[1] = o[2] = o[3] = 0.0f;
  for (int k = first; k < first + teams; ++k) m = fmaxf(m, sml[0][k]);
  for (int k = first; k < first + teams; ++k) l += __builtin_amdgcn_exp2f(sml[0][k] - m) * sml[1][k];
  const float f = 1.0f / l;  // a sum of 0: every score is -inf, and the row NaN, as 0 / 0
  for (int k = first; k < first + teams; ++k) {
    const float c = __builtin_amdgcn_exp2f(sml[0][k] - m) * sml[1][k] * f;
    const float4 x = *reinterpret_cast<const float4*>(&so[k][d]);
    o[0] += c * x.x;
    o[1] += c * x.y;
    o[2] += c * x.z;
    o[3] += c * x.w;
  }
  *reinterpret_cast<uint2*>(a.out + (bi * a.heads + hq) * a.c.D + d) =
      i < tr.i1 ? make_uint2(pack2(o[0], o[1]), pack2(o[2], o[3])) : make_uint2(0, 0);
}

// How a call is cut: waves of a workgroup that share blocks (0: each takes its own), 16-row pieces of a wave, rows of a
// workgroup, key splits.
struct AttendPlan {
  int waves, rt, rows;
  int64_t tiles;  // of one (sequence, head)
  int splits, chunk;
  size_t bytes;
};
AttendPlan attend_plan(int64_t B, int64_t H, int64_t heads, int64_t Dp, int64_t n, int64_t bound) {
  AttendPlan p;
  const int64_t rows = n * (heads / H), blocks = ceil_div(bound, kKvBlock);
  // Sharing pays from 33 rows on: 8 sequences of 16000, 8 heads of 128, 24 rows 59 us against 74 shared, 48 rows 98
  // against 91.
  p.rt = rows <= 16 || Dp > 128 ? 1 : 2;
  // Eight waves convert a block once where four and four convert it twice; up to 128 rows half of them would have none
  // of their own, and with heads above 128 four leave a SIMD one wave: 8 sequences of 4000, 2048 rows of 128 a head, 267
  // us against 293; 2 of 8000, 150 rows, 52 against 56 and 60 rows, 37 against 34; 60 rows of 256, 31 against 35.
  p.waves = rows <= 16 * p.rt ? 0 : rows <= 128 && Dp <= 128 ? 4 : 8;
  p.rows = 16 * p.rt * (p.waves ? p.waves : 1);
  p.tiles = ceil_div(rows, p.rows);
  const int64_t wgs = B * H * p.tiles;
  // one workgroup of 8 waves or two of 4 on every CU (three or four of the latter fit, but then each has too few blocks
  // to hide its start: 4 sequences of 16000 over 8 heads take 28 us with 512, 36 us with 1024), none with less than two
  // blocks for each of its waves
  int64_t s = ceil_div(p.waves == 8 ? 256 : 512, wgs);
  const int64_t most = ceil_div(blocks, 2 * kAtnWaves);
  if (s > most) s = most;
  // four blocks for each wave cost less than joining splits: 1000 tokens over 8 heads of 128 take 11.5 us, 16 us in two
  if (!p.waves && blocks <= 4 * kAtnWaves) s = 1;
  if (s < 1) s = 1;
  p.splits = static_cast<int>(s);
  p.chunk = static_cast<int>(blocks > 0 ? ceil_div(blocks, s) : 1);
  p.bytes = s > 1 ? static_cast<size_t>(wgs) * s * p.rows * (Dp + 2) * 4 : 0;
  return p;
}

template <int DB>
void launch_attend(const AttendArgs& a, const AttendPlan& p, hipStream_t st) {
  constexpr int RT = DB <= 2 ? 2 : 1;  // of the shared form: what the registers hold twice a SIMD
  const dim3 grid(static_cast<unsigned>((int64_t)a.c.B * a.c.H * a.tiles), a.splits);
  if (p.waves == 8) {
    kv8_chunk_kernel<DB, RT, 8><<<grid, 512, 0, st>>>(a);
  } else if (p.waves == 4) {
    if constexpr (DB <= 2) kv8_chunk_kernel<DB, RT, 4><<<grid, 256, 0, st>>>(a);  // the plan's only such heads
  } else if (p.rt == RT) {
    kv8_attend_kernel<DB, RT><<<grid, kAtnWaves * 64, 0, st>>>(a);
  } else {
    kv8_attend_kernel<DB, 1><<<grid, kAtnWaves * 64, 0, st>>>(a);
  }
  if (a.splits > 1) {
    constexpr int G = DB == 3 ? 4 : 16 / DB;  // groups of a workgroup: as many on a row as it has splits, else more rows
    int teams = 1;
    while (teams < G && teams < a.splits) teams *= 2;
    const int64_t rows = (int64_t)a.c.B * a.n * a.heads;
    kv8_join_kernel<DB><<<static_cast<unsigned>(ceil_div(rows, G / teams)), 256, 0, st>>>(a, teams);
  }
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
  SF_CHECK_ARG(a.c.B * n * heads < (1ll << 31) && wgs < (1ll << 23), "sf_kv8_attend: too many rows");
  a.q = static_cast<const uint16_t*>(q);
  a.qsb = q_sb, a.qss = q_ss, a.qsh = q_sh;
  a.out = static_cast<uint16_t*>(out);
  a.n = static_cast<int>(n);
  a.heads = static_cast<int>(heads);
  a.group = static_cast<int>(heads / a.c.H);
  a.window = static_cast<int>(window < cap ? window : 0);
  a.scale = scale < 2.0e38f ? scale * kAtnLog2e : 3.0e38f;
  a.rows = p.rows;
  a.tiles = static_cast<int>(p.tiles);
  a.splits = p.splits;
  a.chunk = p.chunk;
  a.po = static_cast<float*>(workspace);
  a.pml = a.po ? a.po + wgs * p.splits * p.rows * a.c.Dp : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (a.c.Dp / 64) {
    case 1: launch_attend<1>(a, p, st); break;
    case 2: launch_attend<2>(a, p, st); break;
    case 3: launch_attend<3>(a, p, st); break;
    case 4: launch_attend<4>(a, p, st); break;
  }
  return launch_status("sf_kv8_attend");
}
