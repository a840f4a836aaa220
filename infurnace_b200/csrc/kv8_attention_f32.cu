// Causal attention over pages of keys and values held in 8 bits (kv8.cu has the format), float32 queries and output, compiled for
// one head size (-DHEAD_DIM=<multiple of 16, at most 256>).
//
// All products are products of whole numbers on the tensor cores (mma.sync, 8-bit operands, exact 32-bit sums): the codes as
// they lie in the pages, queries and softmax weights as fixed-point numbers of three bytes, a product for each byte.  A query row
// is in units of its largest number over 2^23; a weight, times its page's step, in units of the largest of its row among 32 keys
// over 2^24, so that a long row of small weights beside one large one keeps all bits.  A page's step is a factor of its keys'
// scores; half a step beside each code is half the sum of the row's queries or weights.  Queries and weights are rounded once
// each; everything outside of the products is float32.
// Errors against 64 bits 4 to 6e-7 of the output, below those of plain float32 sums (6e-7 to 1.4e-6); with queries and weights of two
// half-precision terms each, in the same time, 1.4 to 2.4e-6 (the running sums of half-precision products are cut off, not
// rounded).  For bfloat16 the two are not of the same time: eight requests of 3,967 to 8,095 keys 31 us here, 26.5
// as in kv8_attention.cu.
#define KV8_F32 1
#include "kv8_attention.cuh"

// d += a b of whole numbers: a 16 x 32 (rows by k) codes, b 32 x 8, with or without a sign.
template <bool SIGNED> __device__ __forceinline__ void mma_k32(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (SIGNED)
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same for k = 16.
template <bool SIGNED> __device__ __forceinline__ void mma_k16(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  if (SIGNED)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};\n"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(b0));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};\n"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(b0));
}
// The weights of 32 keys as a product's operand: for each byte (the highest first) of row tile n the two words of four keys.
template <int NT> struct Weights { uint32_t b[3][NT][2]; };
// A sum below 2^22 in size that began as this is a float, 1.5 2^23 and the sum: no conversion.
constexpr int MAGIC = 0x4b400000;
__device__ __forceinline__ float magic_sum(int x) { return __int_as_float(x) - 12582912.f; }

// The values of two groups of 16 keys as a lane holds them: keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 (c = lane % 4) of each.  Blocks follow
// one another.
template <int LEFT> struct Values {
  static constexpr int W = LEFT >= 128 ? 128 : LEFT >= 64 ? 64 : LEFT >= 32 ? 32 : 16;
  Piece<W> v[2][4];
  Values<LEFT - W> rest;
  __device__ __forceinline__ void load(int group, const int8_t* p, int lane) {       // p: the first of the group's keys at this block, and the lane's offset
    v[group][0].load(p); v[group][1].load(p + D); v[group][2].load(p + 8 * D); v[group][3].load(p + 9 * D);
    rest.load(group, p + next_block<LEFT>(lane), lane);
  }
  // o += v^T p^T times the rows' factors.  The k index of a product: 4 c + j is key 2 c + 8 j, 16 + 4 c + j key 2 c + 1 + 8 j, so that a
  // word of an operand has the same byte of four keys that the lane holds.  M tile i of a block has dimension chunk + 2 i in its row
  // lane / 4 and chunk + 2 i + 1 in row lane / 4 + 8.
  template <int NT>
  __device__ __forceinline__ void multiply(float (*o)[NT][4], const Weights<NT>& p, const float (&factor)[NT][2]) const {
#pragma unroll
    for (int i = 0; i < (W + 31) / 32; ++i) {                           // words of four dimensions (two of the last kind)
      uint32_t d[2][4];                                                 // [keys 2 c.., 2 c + 1..][dimension], a byte for each key
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t k0 = v[0][s].word(i), k1 = v[0][s + 2].word(i), k2 = v[1][s].word(i), k3 = v[1][s + 2].word(i);
        const uint32_t t0 = __byte_perm(k0, k1, 0x5140), u0 = __byte_perm(k2, k3, 0x5140);
        d[s][0] = __byte_perm(t0, u0, 0x5410);
        d[s][1] = __byte_perm(t0, u0, 0x7632);
        if (W > 16) {
          const uint32_t t1 = __byte_perm(k0, k1, 0x7362), u1 = __byte_perm(k2, k3, 0x7362);
          d[s][2] = __byte_perm(t1, u1, 0x5410);
          d[s][3] = __byte_perm(t1, u1, 0x7632);
        }
      }
#pragma unroll
      for (int m = 0; m < (W > 16 ? 2 : 1); ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float (&to)[4] = o[2 * i + m][n];
          int x[4] = {0, 0, 0, 0}, y[4] = {MAGIC, MAGIC, MAGIC, MAGIC};
          mma_k32<false>(x, d[0][2 * m], d[0][2 * m + 1], d[1][2 * m], d[1][2 * m + 1], p.b[0][n][0], p.b[0][n][1]);
          mma_k32<false>(y, d[0][2 * m], d[0][2 * m + 1], d[1][2 * m], d[1][2 * m + 1], p.b[2][n][0], p.b[2][n][1]);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] *= 256;
          mma_k32<false>(x, d[0][2 * m], d[0][2 * m + 1], d[1][2 * m], d[1][2 * m + 1], p.b[1][n][0], p.b[1][n][1]);
#pragma unroll
          for (int j = 0; j < 4; ++j) to[j] = fmaf(fmaf((float)x[j], 256.f, magic_sum(y[j])), factor[n][j & 1], to[j]);
        }
    }
    rest.template multiply<NT>(o + W / 16, p, factor);
  }
};
template <> struct Values<0> {
  __device__ __forceinline__ void load(int, const int8_t*, int) {}
  template <int NT> __device__ __forceinline__ void multiply(float (*)[NT][4], const Weights<NT>&, const float (&)[NT][2]) const {}
};

// One warp over tiles of 32 keys for up to 8 NT score rows of one key head.  In the layout of the results a lane has rows
// 8 n + 2 (lane % 4) + {0, 1} of row tile n.
template <int NT>
struct Stream {
  static constexpr int ROW_TILES = NT, TILE = 32;                        // keys of a step
  static constexpr int CTAS = NT == 1 ? (D <= 128 ? 3 : 2) : D <= 128 ? 2 : 1;      // on an SM, that the registers are cut for
  uint32_t qb[3][NT][KS];                // bytes of the rows' numbers, the highest (with the sign) first; four dimensions a word
  float qscale[NT][2], qoff[NT][2];      // what turns a product into a number of real units: times qscale, and qoff
  int last[NT][2];                       // position of the row's query (NO_ROW: no such row)
  // m: reference of the row's scores; l: this lane's part of the sum of the weights 2^(score - m)
  // r: log2 of the unit of o and wsum, 2^m apart; wsum: this lane's part of the sum of weights times steps, whose half o lacks
  float m[NT][2], l[NT][2], r[NT][2], wsum[NT][2];
  float o[KS][NT][4];
  // log2 of the largest weight as a whole number, 24 - 2^-12: differences to `top`, a number of up to 2^8 and more, are exact (23.9999 is
  // rounded to 2^-17 there, and all weights with it, 5e-6 beside their sum)
  static constexpr float TOP = 23.999755859375f;

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) { m[n][e] = r[n][e] = -INFINITY; l[n][e] = wsum[n][e] = 0.f; }
#pragma unroll
      for (int i = 0; i < KS; ++i) { o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f; }
    }
  }
  // pos0: position of the request's first query.
  __device__ __forceinline__ void queries(const Queries<NT>& raw, int row0, int rows, int pos0, int G, int lane) {
    auto number = [&](int n, int ks, int j) { return __uint_as_float(raw.w[n][ks][j]); };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t amax = 0;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = max(amax, __float_as_uint(number(n, ks, j)) & 0x7fffffffu);
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // the row's largest number becomes one of [2^22, 2^23], by a power of two that a float holds either way round
      constexpr int UP = 127 + 22;
      const int f = min(max((int)(amax >> 23), UP - 126), 250);
      const float to = __uint_as_float((uint32_t)(127 + UP - f) << 23), back = __uint_as_float((uint32_t)(127 - UP + f) << 23);
      int sum = 0;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = (uint32_t)min(__float2int_rn(number(n, ks, j) * to), (1 << 23) - 1);      // (a number next to a power of two rounds up to it)
          sum += (int)x[j];
        }
        const uint32_t t = __byte_perm(x[0], x[1], 0x5140), u = __byte_perm(x[2], x[3], 0x5140);       // their lowest two bytes
        qb[2][n][ks] = __byte_perm(t, u, 0x5410);
        qb[1][n][ks] = __byte_perm(t, u, 0x7632);
        qb[0][n][ks] = __byte_perm(__byte_perm(x[0], x[1], 0x0062), __byte_perm(x[2], x[3], 0x0062), 0x5410);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      // a row with an infinity or a NaN has NaN for its scores
      const float half = (amax >> 23) == 255u ? __uint_as_float(0x7fffffffu) : 0.5f * (float)sum * back;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int from = ((lane & 3) * 2 + e) * 4;
        qscale[n][e] = __shfl_sync(0xffffffffu, back, from);
        qoff[n][e] = __shfl_sync(0xffffffffu, half, from);
        const int r = row0 + n * 8 + (lane & 3) * 2 + e;
        last[n][e] = r < rows ? pos0 + r / G : NO_ROW;
      }
    }
  }

  template <bool SIGNED>
  __device__ __forceinline__ void product(const Keys& k, int (&x)[4], const uint32_t (&q)[KS]) const {
#pragma unroll
    for (int ks = 0; ks < 4 * K64; ks += 2) mma_k32<SIGNED>(x, k.word(0, ks), k.word(1, ks), k.word(0, ks + 1), k.word(1, ks + 1), q[ks], q[ks + 1]);
#pragma unroll
    for (int ks = 4 * K64; ks < KS; ++ks) mma_k16<SIGNED>(x, k.word(0, ks), k.word(1, ks), q[ks]);
  }
  // Scores of 16 keys from `key0` on.  step: of the keys, times the softmax's factor.
  template <bool MASK>
  __device__ __forceinline__ void scores(const Keys& k, float step, int key0, int window, float (&s)[NT][4], int lane) const {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      int x[4] = {0, 0, 0, 0};
      product<true>(k, x, qb[0][n]);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] *= 256;
      product<false>(k, x, qb[1][n]);
      int y[4] = {0, 0, 0, 0};
      product<false>(k, y, qb[2][n]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = fmaf((float)x[j], 256.f, (float)y[j]);           // (of up to 256 numbers: y may pass 2^22)
        const float z = fmaf(p, qscale[n][j & 1], qoff[n][j & 1]) * step;
        bool seen = true;
        if (MASK) {
          const int key = key0 + (lane >> 2) + (j >> 1) * 8, q = last[n][j & 1];
          seen = key <= q && (window == 0 || key > q - window);
        }
        s[n][j] = seen ? z : -INFINITY;
      }
    }
  }

  // Weights of 32 keys, and o += p v.  vf: the exponent fields of the groups' values; 0 also for a page of NaN, whose scores are NaN
  // where they are seen.
  __device__ __forceinline__ void weigh(const float (&s)[2][NT][4], const Values<D>& v, int vf0, int vf1) {
    // The references are floats' and move only when sums would leave the range.
    bool up = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        up |= fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e])) > m[n][e] + 60.f;
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e]));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = fmaxf(x, m[n][e]);
          if (x != m[n][e]) {
            l[n][e] *= kv8_exp2(m[n][e] - x);
            r[n][e] += m[n][e] == -INFINITY ? 0.f : m[n][e] - x;        // (o stays what it is, in a unit that is named anew)
            m[n][e] = x;
          }
        }
    }
    // From here on scores are differences to m, small numbers (a score of thousands plus an exponent would lose its last bits).
    // log2 of the values' steps (an exponent field is 133 more); a page of zeros has no weight.
    const float step[2] = {vf0 ? (float)vf0 : -INFINITY, vf1 ? (float)vf1 : -INFINITY};
    float d[2][NT][4], top[NT][2];                                      // top: of each row the largest weight times step, log2
    up = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float less = m[n][e] == -INFINITY ? 0.f : m[n][e];
#pragma unroll
        for (int g = 0; g < 2; ++g) { d[g][n][e] = s[g][n][e] - less; d[g][n][2 + e] = s[g][n][2 + e] - less; }
        float x = fmaxf(fmaxf(d[0][n][e], d[0][n][2 + e]) + step[0], fmaxf(d[1][n][e], d[1][n][2 + e]) + step[1]);
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        top[n][e] = x;
        up |= x > r[n][e] + 60.f;
      }
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = fmaxf(top[n][e], r[n][e]);
          f[e] = x == r[n][e] ? 1.f : kv8_exp2(r[n][e] - x);
          r[n][e] = x;
          wsum[n][e] *= f[e];
        }
#pragma unroll
        for (int i = 0; i < KS; ++i) { o[i][n][0] *= f[0]; o[i][n][1] *= f[1]; o[i][n][2] *= f[0]; o[i][n][3] *= f[1]; }
      }
    }
    Weights<NT> p;
    float factor[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t byte[3][2];                                              // [byte][row]: of four keys, lane / 4 + 8 j
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[n][e] += (kv8_exp2(d[0][n][e]) + kv8_exp2(d[0][n][2 + e])) + (kv8_exp2(d[1][n][e]) + kv8_exp2(d[1][n][2 + e]));
        const bool none = top[n][e] == -INFINITY;
        const float shift = none ? 0.f : TOP - top[n][e];
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = kv8_exp2(d[j >> 1][n][(j & 1) * 2 + e] + (step[j >> 1] + shift));
        // what a unit of these weights is of the sums'
        factor[n][e] = none ? 0.f : kv8_exp2(top[n][e] - r[n][e] - TOP);
        wsum[n][e] = fmaf((x[0] + x[1]) + (x[2] + x[3]), factor[n][e], wsum[n][e]);
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __float2uint_rn(x[j]);
        const uint32_t t = __byte_perm(w[0], w[1], 0x5140), u = __byte_perm(w[2], w[3], 0x5140);       // their lowest two bytes
        byte[2][e] = __byte_perm(t, u, 0x5410);
        byte[1][e] = __byte_perm(t, u, 0x7632);
        byte[0][e] = __byte_perm(__byte_perm(w[0], w[1], 0x0062), __byte_perm(w[2], w[3], 0x0062), 0x5410);
      }
      // from (keys of lane / 4, two rows) to (row lane / 4, keys of 2 c and of 2 c + 1)
#pragma unroll
      for (int b = 0; b < 3; ++b) {
        const uint32_t lo = transpose8(__byte_perm(byte[b][0], byte[b][1], 0x5410)), hi = transpose8(__byte_perm(byte[b][0], byte[b][1], 0x7632));
        p.b[b][n][0] = __byte_perm(lo, hi, 0x5410);
        p.b[b][n][1] = __byte_perm(lo, hi, 0x7632);
      }
    }
    v.template multiply<NT>(o, p, factor);
  }

  // Tiles from `first` to `end` (exclusive), every `step`-th, of the groups of 16 from `low` up to `high` (exclusive), in two parts: the
  // constructor requests the first of them, `run` works through all.  A tile's group outside is another name for its other group:
  // every row's rule hides its keys.
  struct Walk : Kv8Pages {
    int first, end, step, low, high, next_page[2], kf[2], vf[2];
    Keys k[2];
    Values<D> v;
    __device__ __forceinline__ int group(int t, int g) const { return min(max(2 * t + g, low), high - 1); }
    __device__ __forceinline__ Walk(const Kv8Args& a, const int* table_, int kv_head, int low_, int high_, int first_, int end_, int step_, int lane)
        : Kv8Pages(a, table_, kv8_uniform(kv_head), lane) {
      low = low_; high = high_; first = kv8_uniform(first_); end = kv8_uniform(end_); step = step_;
      if (first >= end) return;
      int page[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        page[g] = page_of(group(first, g));
        next_page[g] = first + step < end ? page_of(group(first + step, g)) : 0;
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const size_t from = at(group(first, g), page[g]);
        read_fields(page[g], kf[g], vf[g]);
        k[g].load(k_base + from, lane);
        v.load(g, v_base + from, lane);
      }
    }
  };
  // full_from, full_to: keys from and up to here are seen by every row that exists.
  __device__ __forceinline__ void run(const Kv8Args& a, Walk& w, int full_from, int full_to, int lane) {
    const float scale64 = a.scale * 0.015625f;
    for (int t = w.first; t < w.end; t += w.step) {
      const bool more = t + w.step < w.end;
      float s[2][NT][4];
      const bool whole = t * TILE >= full_from && t * TILE + TILE - 1 <= full_to;
      int vf[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float ks = kv8_score_step(w.kf[g], w.vf[g], scale64);
        vf[g] = kv8_value_field(w.vf[g]);
        if (whole) scores<false>(w.k[g], ks, t * TILE + g * 16, a.window, s[g], lane);
        else scores<true>(w.k[g], ks, t * TILE + g * 16, a.window, s[g], lane);
      }
      size_t next[2] = {0, 0};
      if (more) {                                                       // the next keys while these values are multiplied
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          next[g] = w.at(w.group(t + w.step, g), w.next_page[g]);
          w.read_fields(w.next_page[g], w.kf[g], w.vf[g]);
          w.k[g].load(w.k_base + next[g], lane);
        }
        if (t + 2 * w.step < w.end) {
#pragma unroll
          for (int g = 0; g < 2; ++g) w.next_page[g] = w.page_of(w.group(t + 2 * w.step, g));
        }
      }
      weigh(s, w.v, vf[0], vf[1]);
      if (more) {                                                       // and the next values while the next scores are formed
#pragma unroll
        for (int g = 0; g < 2; ++g) w.v.load(g, w.v_base + next[g], lane);
      }
    }
  }
  // Sums over the lanes that share a row, and the weighted values in real units (times the weights' common factor 2^-m).
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float unit[2], rest[2];                                           // 2^(r - 133) in two factors: of its own it may be no float
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
          wsum[n][e] += __shfl_xor_sync(0xffffffffu, wsum[n][e], x);
        }
        const int by = kv8_excess(l[n][e], wsum[n][e], r[n][e]);
        const float to = r[n][e] == -INFINITY ? -1000.f : r[n][e] - 133.f - (float)by;
        unit[e] = kv8_exp2(fmaxf(to, -100.f));
        rest[e] = kv8_exp2(fminf(to + 100.f, 0.f));
        l[n][e] *= __uint_as_float((uint32_t)(127 - by) << 23);
        m[n][e] += (float)by;
      }
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][n][j] = fmaf(0.5f, wsum[n][j & 1], o[i][n][j]) * unit[j & 1] * rest[j & 1];
    }
  }
};


KV8_ENTRIES(Stream<1>, Stream<TILES>)
