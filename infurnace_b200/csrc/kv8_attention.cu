// Causal attention over pages of keys and values held in 8 bits (kv8.cu has the format), bfloat16 queries and output, compiled for
// one head size (-DHEAD_DIM=<multiple of 16, at most 256>).
//
// The products run on the tensor cores (mma.sync, float32 accumulation) over the codes as whole numbers, which half precision
// holds exactly; a page's step enters as a factor of its scores (keys) and of its weights (values), so no number is rounded
// for having been 8 bits.  A query row times a power of two is half precision too (exact down to 2^-24 of its largest), and so
// is a softmax weight, the one thing that is rounded (11 bits).
//
// From bits to half-precision numbers: u = code + 128 in the low byte of a half is the subnormal number u 2^-24, exactly; two
// integer instructions make two of them.  Keys stay so (q . (u - 127.5) = q . u - 127.5 sum(q), the second known per row);
// for values 128 is taken off again: a sum over thousands of keys would lose what the offset swamps.
//
// Softmax: weights are 2^(score - m + 8) with a reference m per row that moves (and then rescales the sums) only when a weight, times its
// page's step over the largest step that the warp has met, exceeds it by 6 in the exponent, so that most tiles need no maximum
// over lanes.  That product is what enters the second product: 2^14 is the largest, and half-precision numbers down to 2^-32 of it
// still count, for steps up to 2^80 apart.  (A reference of the scores alone: rows that do not see a page of values 2^24 larger than
// their own, but whose warp does, lose bits, and from 2^33 on are zero.)  Sums are float32.
//
// What bounds it: no one unit.  Over a whole call the integer pipe (for the bytes of keys and values) and the issue slots are half busy, and a third of
// the warps' time is waiting for memory, with the four CTAs on an SM that 128 registers allow: what does not have to stay in one over the
// loop is named anew or uniform (46.1 to 42.2 us in the third figure).  A call has some
// 8 us beside the loop: the look at the lengths, the first trip, the joins.  Eight requests of 3,967 to 8,095 keys (32 heads on 8)
// 26.5 us, 3.7 TB/s; 64 of 129 to 383 (16 on 8) 14.5; 64 of 1,500 (32 on 8) 42.2, 4.7 TB/s.  Slower were: copies to shared memory some tiles
// ahead, requests to the second level of cache two tiles ahead, values requested with the keys, three CTAs with more registers (59 us).
#define KV8_F32 0
#include "kv8_attention.cuh"
#include <cuda_fp16.h>

// d += a b: a 16 x 16 (rows by k), b 16 x 8.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Bytes 0 and 2 (and 1 and 3) of a word of codes as half-precision numbers (code + 128) 2^-24.
__device__ __forceinline__ uint32_t even_bytes(uint32_t w) { return (w & 0x00ff00ffu) ^ 0x00800080u; }
__device__ __forceinline__ uint32_t odd_bytes(uint32_t w) { return ((w >> 8) & 0x00ff00ffu) ^ 0x00800080u; }
__device__ __forceinline__ uint32_t centred(uint32_t x) {               // code 2^-24
  const uint32_t off = 0x80808080u;                                     // -(128 2^-24) twice: sign, subnormal 0x0080
  const __half2 y = __hadd2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<const uint32_t*>(&y);
}

// The values of 16 keys as a lane holds them: keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 (c = lane % 4).  Blocks follow one another.
template <int LEFT> struct Values {
  static constexpr int W = LEFT >= 128 ? 128 : LEFT >= 64 ? 64 : LEFT >= 32 ? 32 : 16;
  Piece<W> v[4];
  Values<LEFT - W> rest;
  __device__ __forceinline__ void load(const int8_t* p, int lane) {       // p: the first of the 16 keys at this block, and the lane's offset
    v[0].load(p); v[1].load(p + D); v[2].load(p + 8 * D); v[3].load(p + 9 * D);
    rest.load(p + next_block<LEFT>(lane), lane);
  }
  // o^T += v^T p^T; m tile i of a block has dimension chunk + 2 i in its row lane / 4 and chunk + 2 i + 1 in row lane / 4 + 8
  template <int NT>
  __device__ __forceinline__ void multiply(float (*o)[NT][4], const uint32_t (&p)[NT][2]) const {
#pragma unroll
    for (int i = 0; i < W / 16; ++i) {
      const uint32_t sel = i & 1 ? 0x7632u : 0x5410u;
      const uint32_t x = __byte_perm(v[0].word(i >> 1), v[1].word(i >> 1), sel), y = __byte_perm(v[2].word(i >> 1), v[3].word(i >> 1), sel);
      const uint32_t a0 = centred(even_bytes(x)), a1 = centred(odd_bytes(x)), a2 = centred(even_bytes(y)), a3 = centred(odd_bytes(y));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(o[i][n], a0, a1, a2, a3, p[n][0], p[n][1]);
    }
    rest.template multiply<NT>(o + W / 16, p);
  }
};
template <> struct Values<0> {
  __device__ __forceinline__ void load(const int8_t*, int) {}
  template <int NT> __device__ __forceinline__ void multiply(float (*)[NT][4], const uint32_t (&)[NT][2]) const {}
};

// One warp over tiles of 16 keys for up to 8 NT score rows of one key head.  In the layout of the results a lane has rows
// 8 n + 2 (lane % 4) + {0, 1} of row tile n.
template <int NT>
struct Stream {
  static constexpr int ROW_TILES = NT, TILE = 16;                        // keys of a step
  static constexpr int CTAS = NT == 1 ? (D <= 128 ? 4 : 2) : D <= 128 ? 2 : 1;      // on an SM, that the registers are cut for
  uint32_t qf[NT][KS][2];
  float qscale[NT][2], qoff[NT][2];      // what turns a product into a number of real units: times qscale, and qoff
  int last[NT][2];                       // position of the row's query (NO_ROW: no such row)
  // m: reference of the row's scores, finite (`weigh`; a weight is 2^(score + (8 - m))); l, wsum: this lane's part of the sums of the weights,
  // and of weights times steps
  float m[NT][2], l[NT][2], wsum[NT][2];
  float o[KS][NT][4];
  int v_ref;                             // exponent field that the sums of weighted values are in units of
  static constexpr int SPREAD = 80;      // what a row's reference lies below its largest score at most, in log2, beside the 6

  __device__ __forceinline__ void reset() {
    v_ref = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) { m[n][e] = NO_SCORE; l[n][e] = 0.f; wsum[n][e] = 0.f; }
#pragma unroll
      for (int i = 0; i < KS; ++i) { o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f; }
    }
  }
  // pos0: position of the request's first query.
  __device__ __forceinline__ void queries(const Queries<NT>& raw, int row0, int rows, int pos0, int G, int lane) {
    auto number = [&](int n, int ks, int j) { const uint32_t w = raw.w[n][ks][j >> 1]; return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16); };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t amax = 0;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = max(amax, __float_as_uint(number(n, ks, j)) & 0x7fffffffu);
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // the row's largest number becomes one of [2^10, 2^11): a power of two that a float holds either way round
      const int f = min(max((int)(amax >> 23), 11), 250);
      const float to = __uint_as_float((uint32_t)(127 + 137 - f) << 23);      // 2^(10 - (f - 127))
      const float back = __uint_as_float((uint32_t)(127 - 137 + f) << 23);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = number(n, ks, j) * to;
        qf[n][ks][0] = pack_half(x[0], x[2]);                        // beside the even and the odd bytes of a word of codes
        qf[n][ks][1] = pack_half(x[1], x[3]);
      }
      // sums of the rounded rows, in the layout of the scores, by a product with ones
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) mma_f16(s, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, qf[n][ks][0], qf[n][ks][1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float b = __shfl_sync(0xffffffffu, back, ((lane & 3) * 2 + e) * 4);
        qscale[n][e] = b * 16777216.f;
        qoff[n][e] = -127.5f * s[e] * b;
        const int r = row0 + n * 8 + (lane & 3) * 2 + e;
        last[n][e] = r < rows ? pos0 + r / G : NO_ROW;
      }
    }
  }

  // Scores of 16 keys from `key0` on, weights, and o += p v.  step: of the keys, times the softmax's factor; vf: the values' field.
  template <bool MASK>
  __device__ __forceinline__ void scores(const Keys& k, float step, int key0, int window, float (&s)[NT][4], int lane) const {
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint32_t a0 = even_bytes(k.word(0, ks)), a1 = even_bytes(k.word(1, ks)), a2 = odd_bytes(k.word(0, ks)), a3 = odd_bytes(k.word(1, ks));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(s[n], a0, a1, a2, a3, qf[n][ks][0], qf[n][ks][1]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = fmaf(s[n][j], qscale[n][j & 1], qoff[n][j & 1]) * step;
        bool seen = true;
        if (MASK) {
          const int key = key0 + (lane >> 2) + (j >> 1) * 8, p = last[n][j & 1];
          seen = key <= p && (window == 0 || key > p - window);
        }
        s[n][j] = seen ? x : -INFINITY;
      }
  }
  // vf: the exponent field of the values; 0 also for a page of NaN, whose scores are NaN where they are seen.
  // A row's reference is that of its weights times their steps, in units of 2^v_ref: a score may exceed it by what its page's step lies below
  // v_ref (by SPREAD at most), and when a page raises v_ref, the reference falls as much.  So a row keeps the bits of its products
  // whatever steps the warp has met that the row does not see or gives no weight.
  __device__ __forceinline__ void weigh(float (&s)[NT][4], const Values<D>& v, int vf) {
    const bool larger = vf > v_ref;                                     // uniform
    const int below = min(max(v_ref - vf, 0), SPREAD);
    const float lag = __int_as_float(0x4b400000 + below) - 12582906.f;  // below + 6
    bool up = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) up |= fmaxf(s[n][e], s[n][2 + e]) > m[n][e] + lag;
    if (__any_sync(0xffffffffu, up) || larger) {
      const int raise = larger ? min(vf - v_ref, SPREAD) : 0;
      float fv = 1.f;
      if (larger) {
        fv = v_ref ? __uint_as_float((uint32_t)max(0, 127 + v_ref - vf) << 23) : 0.f;
        v_ref = vf;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(s[n][e], s[n][2 + e]), sum = l[n][e];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            sum += __shfl_xor_sync(0xffffffffu, sum, x);
          }
          const int room = max(0, min(raise, 214 - (int)(__float_as_uint(sum) >> 23)));      // the row's sum stays below 2^88
          mx = fmaxf(mx - (lag - 6.f), m[n][e] - (float)room);
          f[e] = kv8_exp2(m[n][e] - mx);
          m[n][e] = mx;
          l[n][e] *= f[e];
          f[e] *= fv;
          wsum[n][e] *= f[e];
        }
#pragma unroll
        for (int i = 0; i < KS; ++i) { o[i][n][0] *= f[0]; o[i][n][1] *= f[1]; o[i][n][2] *= f[0]; o[i][n][3] *= f[1]; }
      }
    }
    // the step of this page's values over the reference
    const float fw = vf == 0 ? 0.f : __uint_as_float((uint32_t)max(0, 127 + vf - v_ref) << 23);
    uint32_t p[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = kv8_exp2(s[n][j] + (8.f - m[n][j & 1]));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float both = w[e] + w[2 + e];
        l[n][e] += both;
        wsum[n][e] = fmaf(both, fw, wsum[n][e]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] *= fw;
      p[n][0] = transpose8(pack_half(w[0], w[1]));
      p[n][1] = transpose8(pack_half(w[2], w[3]));
    }
    v.template multiply<NT>(o, p);
  }

  // Tiles first, first + step, ... up to `end` (exclusive) of 16 keys, in two parts: `begin` requests the first of them, `run` works
  // through all.  full_from, full_to: keys from and up to here are seen by every row that exists.
  struct Walk : Kv8Pages {
    int first, end, step, next_page, kf, vf;
    Keys k;
    Values<D> v;
    __device__ __forceinline__ Walk(const Kv8Args& a, const int* table_, int kv_head, int, int, int first_, int end_, int step_, int lane)
        : Kv8Pages(a, table_, kv8_uniform(kv_head), lane) {
      first = kv8_uniform(first_); end = kv8_uniform(end_); step = step_; next_page = 0;
      if (first >= end) return;
      const int page = page_of(first);
      if (first + step < end) next_page = page_of(first + step);
      const size_t from = at(first, page);
      read_fields(page, kf, vf);
      k.load(k_base + from, lane);
      v.load(v_base + from, lane);
    }
  };
  __device__ __forceinline__ void run(const Kv8Args& a, Walk& w, int full_from, int full_to, int lane) {
    const float scale64 = a.scale * 0.015625f;
    for (int t = w.first; t < w.end; t += w.step) {
      const bool more = t + w.step < w.end;
      float s[NT][4];
      const bool whole = t * 16 >= full_from && t * 16 + 15 <= full_to;
      const float ks = kv8_score_step(w.kf, w.vf, scale64);
      const int vf = kv8_value_field(w.vf);
      if (whole) scores<false>(w.k, ks, t * 16, a.window, s, lane);
      else scores<true>(w.k, ks, t * 16, a.window, s, lane);
      size_t next = 0;
      if (more) {                                                       // the next keys while these values are multiplied
        next = w.at(t + w.step, w.next_page);
        w.read_fields(w.next_page, w.kf, w.vf);
        w.k.load(w.k_base + next, lane);
        if (t + 2 * w.step < w.end) w.next_page = w.page_of(t + 2 * w.step);
      }
      weigh(s, w.v, vf);
      if (more) w.v.load(w.v_base + next, lane);                         // and the next values while the next scores are formed
    }
  }
  // Sums over the lanes that share a row, and the weighted values in real units (times the weights' common factor).
  __device__ __forceinline__ void finish() {
    const float unit = kv8_step((uint32_t)v_ref);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float less[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
          wsum[n][e] += __shfl_xor_sync(0xffffffffu, wsum[n][e], x);
        }
        const int by = kv8_excess(l[n][e], wsum[n][e], (float)v_ref);
        less[e] = __uint_as_float((uint32_t)(127 - by) << 23);
        l[n][e] *= less[e];
        m[n][e] += (float)by;
      }
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][n][j] = fmaf(o[i][n][j], 16777216.f, 0.5f * wsum[n][j & 1]) * less[j & 1] * unit;
    }
  }
};


KV8_ENTRIES(Stream<1>, Stream<TILES>)
