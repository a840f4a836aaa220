// What the two kernels of attention over 8-bit pages share: the pages' data as lanes take it, the split of the work, and the
// calls.  kv8_attention.cu (bfloat16 queries and output) and kv8_attention_f32.cu define KV8_F32 and include this, define a
// `Stream` each, one warp's walk over keys for some score rows, and end with KV8_ENTRIES.
//
// The products are transposed: S^T = K Q^T and O^T = V^T P^T, so that keys (and head dimensions) fill the 16 rows of an
// instruction and up to eight score rows (query token x query head of a key head) its 8 columns; decoding with eight query
// heads per key head wastes nothing.  A warp takes groups of 16 keys, which lie in one page each: their codes come from global
// memory to registers in 16-byte pieces, keys each already where its product wants it (any order of the dimensions serves the
// sums over them, so the order is the loads').  There is no shared memory, no barrier and no wait between warps in the loop; the
// other warps of the SM and the order of the requests (the next keys while the values are multiplied, the next values while the
// scores are formed) keep the memory busy.  (Copies to shared memory, four tiles ahead, took the same time.)
//
// Split form: the keys of a key head for one tile of score rows are cut into pieces of nearly one length for all requests,
// whatever their lengths, as many as CTAs fit on the device; a piece leaves its sums in scratch memory, and the CTA that arrives
// last at an item adds them in the order of the pieces.  Whole form (prompts): a warp owns its score rows over all their keys.
// Keys that no row of a tile sees are not read; block-table entries outside are not followed.  A row that sees no key is zero.
#pragma once
#include "common.cuh"
#include <math.h>

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size>"
#endif
#if HEAD_DIM % 16 != 0 || HEAD_DIM < 16 || HEAD_DIM > 256
#error "HEAD_DIM must be a multiple of 16 between 16 and 256"
#endif

typedef __nv_bfloat16 bf16;
#if KV8_F32
typedef float qtype;
#else
typedef bf16 qtype;
#endif
constexpr int D = HEAD_DIM;
constexpr int KS = D / 16;               // words of a key that a lane has; m tiles of an output product
constexpr int WARPS = 4;
constexpr int K64 = D / 64;              // pieces of 64 dimensions of a key that a quad of lanes takes 16 bytes a lane at a time
constexpr int TILES = D <= 128 ? 2 : 1;  // tiles of 8 score rows that a warp has at most (wider heads leave no registers for a second)
constexpr int NO_ROW = -1000000000;
constexpr float NO_SCORE = -3.402823466e38f;      // the lowest float

struct Kv8Args {
  const qtype* q;
  long long q_row;                       // elements between tokens
  const int8_t* codes;
  const uint8_t* exponents;
  const int* tables;
  int table_stride;
  const int* cu_q;
  const int* seq_lens;
  qtype* out;                            // [tokens][heads][D]
  float* parts;                          // split form: [CTA][rows of a tile][D + 2]
  int* counters;                         // split form: one per item, 0 between launches
  int requests, heads, kv_heads, page_size, window;
  float scale;                           // of the scores, times log2(e)
  int min_rows, max_rows;                // requests with fewer or more score rows than this are another kernel's
  int tiles;                             // split form: tiles of score rows that any request has at most
  int most;                              // split form: CTAs that run on the device at a time
};

// A number that all lanes of a warp have, so that it may live in a uniform register: those of the loops over keys are scarce.
__device__ __forceinline__ int kv8_uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ float kv8_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float kv8_step(uint32_t f) {                 // 2^(f - 133), 0, NaN
  if (f == 0u) return 0.f;
  if (f == 255u) return __uint_as_float(0x7fffffffu);
  return f > 6u ? __uint_as_float((f - 6u) << 23) : __uint_as_float(1u << (f + 16u));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {            // of an 8 x 8 matrix of 16-bit numbers over the warp
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

// ---- what a lane holds of values: blocks of 128, 64, 32 and 16 dimensions, an eighth of a block (16, 8, 4, 2 bytes) --------------
template <int W> struct Piece;
template <> struct Piece<128> { uint4 r; __device__ __forceinline__ void load(const int8_t* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; } };
template <> struct Piece<64> { uint2 r; __device__ __forceinline__ void load(const int8_t* p) { r = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? r.x : r.y; } };
template <> struct Piece<32> { uint32_t r; __device__ __forceinline__ void load(const int8_t* p) { r = *reinterpret_cast<const uint32_t*>(p); }
  __device__ __forceinline__ uint32_t word(int) const { return r; } };
template <> struct Piece<16> { uint32_t r; __device__ __forceinline__ void load(const int8_t* p) { r = *reinterpret_cast<const uint16_t*>(p); }
  __device__ __forceinline__ uint32_t word(int) const { return r; } };

// Where a lane's piece of a block of W dimensions of values begins: key 2 (lane % 4).
template <int LEFT> struct ValueBlock { static constexpr int W = LEFT >= 128 ? 128 : LEFT >= 64 ? 64 : LEFT >= 32 ? 32 : LEFT >= 16 ? 16 : 0; };
__device__ __forceinline__ int value_offset(int lane) { return (lane & 3) * 2 * D + (lane >> 2) * (ValueBlock<D>::W / 8); }
// From a block's piece to the next block's.
template <int LEFT> __device__ __forceinline__ int next_block(int lane) {
  constexpr int W = ValueBlock<LEFT>::W, NEXT = ValueBlock<LEFT - W>::W;
  return W + (lane >> 2) * ((NEXT - W) / 8);
}

// The dimension of element e (0, 1) of m tile i of an output product over values of LEFT dimensions, in blocks that follow one another.
template <int LEFT> __device__ __forceinline__ int value_dim(int i, int lane, int e) {
  if constexpr (LEFT == 0) {
    return 0;
  } else {
    constexpr int W = LEFT >= 128 ? 128 : LEFT >= 64 ? 64 : LEFT >= 32 ? 32 : 16;
    if (i < W / 16) return (lane >> 2) * (W / 8) + 2 * i + e;
    return W + value_dim<LEFT - W>(i - W / 16, lane, e);
  }
}

// The keys of a group of 16 as a lane holds them: keys lane / 4 and lane / 4 + 8.
struct Keys {
  uint4 w[2][K64 ? K64 : 1];
  uint32_t tail[2][KS - 4 * K64 ? KS - 4 * K64 : 1];
  static __device__ __forceinline__ int offset(int lane) { return (lane >> 2) * D + (lane & 3) * (K64 ? 16 : 4); }
  __device__ __forceinline__ void load(const int8_t* keys, int lane) {       // keys: the first of the group's, and the lane's offset
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int h = 0; h < K64; ++h) w[e][h] = *reinterpret_cast<const uint4*>(keys + e * 8 * D + h * 64);
#pragma unroll
      for (int s = 0; s < KS - 4 * K64; ++s)
        tail[e][s] = *reinterpret_cast<const uint32_t*>(keys + e * 8 * D + K64 * 64 + s * 16 - (K64 ? (lane & 3) * 12 : 0));
    }
  }
  __device__ __forceinline__ uint32_t word(int e, int ks) const {
    if (ks >= 4 * K64) return tail[e][ks - 4 * K64];
    const uint4& x = w[e][ks >> 2];
    return (ks & 3) == 0 ? x.x : (ks & 3) == 1 ? x.y : (ks & 3) == 2 ? x.z : x.w;
  }
};
// Where the four dimensions of a lane's word ks begin.
__device__ __forceinline__ int key_dim(int ks, int lane) {
  return ks < 4 * K64 ? (ks >> 2) * 64 + (lane & 3) * 16 + (ks & 3) * 4 : K64 * 64 + (ks - 4 * K64) * 16 + (lane & 3) * 4;
}


// The queries of 8 NT score rows as they come: those of row 8 n + lane / 4, four dimensions a word (or two) of a key.
template <int NT> struct Queries { uint32_t w[NT][KS][sizeof(qtype) == 2 ? 2 : 4]; };
// row0: the first of the rows; rows: how many the request has; G: query heads per key head.
template <int NT>
__device__ __forceinline__ void request_queries(Queries<NT>& raw, const Kv8Args& a, int first_token, int row0, int rows, int kv_head, int G, int lane) {
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = row0 + n * 8 + (lane >> 2);
    const bool in = row < rows;
    const int token = in ? row / G : 0, head = in ? row - token * G : 0;
    const qtype* src = a.q + (size_t)(first_token + token) * a.q_row + (size_t)(kv_head * G + head) * D;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = key_dim(ks, lane);
#if KV8_F32
      const uint4 x = in ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
      raw.w[n][ks][0] = x.x; raw.w[n][ks][1] = x.y; raw.w[n][ks][2] = x.z; raw.w[n][ks][3] = x.w;
#else
      const uint2 x = in ? *reinterpret_cast<const uint2*>(src + d) : make_uint2(0, 0);
      raw.w[n][ks][0] = x.x; raw.w[n][ks][1] = x.y;
#endif
    }
  }
}

// The pages of a request as a lane of a stream's walk reads them: few instructions a group, the lane's offsets are in the bases.
struct Kv8Pages {
  const int* table;
  const int8_t *k_base, *v_base;
  const uint8_t* fields;
  uint32_t page_bytes, page_fields, per_page, inverse;
  __device__ __forceinline__ Kv8Pages(const Kv8Args& a, const int* table_, int kv_head, int lane) {
    table = table_;
    page_bytes = 2u * (uint32_t)a.kv_heads * (uint32_t)a.page_size * D;
    k_base = a.codes + (size_t)kv_head * a.page_size * D + Keys::offset(lane);
    v_base = a.codes + (size_t)(a.kv_heads + kv_head) * a.page_size * D + value_offset(lane);
    fields = a.exponents + kv_head;
    page_fields = 2u * (uint32_t)a.kv_heads;
    per_page = (uint32_t)a.page_size / 16;
    inverse = per_page > 1 ? 0xffffffffu / per_page + 1 : 0;
  }
  // The page of a group of 16 keys (its number over groups per page, by a product with the next whole number above 2^32 / per_page:
  // exact for groups below 2^32 / per_page), where its keys begin from a base (and its values from theirs), and its exponent fields.
  __device__ __forceinline__ int place(int group) const { return per_page > 1 ? (int)__umulhi((uint32_t)group, inverse) : group; }
  __device__ __forceinline__ int page_of(int group) const { return table[place(group)]; }
  __device__ __forceinline__ size_t at(int group, int page) const {
    return (size_t)(uint32_t)page * page_bytes + (uint32_t)(group - place(group) * (int)per_page) * (16 * D);
  }
  __device__ __forceinline__ void read_fields(int page, int& kf, int& vf) const {
    const uint8_t* at = fields + (size_t)(uint32_t)page * page_fields;
    kf = at[0];
    vf = at[page_fields >> 1];
  }
};
// The factor of a page's scores: its keys' step times `scale64`, the scores' scale over 64 (a step is 2^-6 of what its field says as a float's).  A page
// whose values are NaN makes the scores NaN that see it, and with them the row; as values its block is then one of zeros.
__device__ __forceinline__ float kv8_score_step(int kf, int vf, float scale64) {
  return max(kf, vf) == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float((uint32_t)kf << 23) * scale64;
}
__device__ __forceinline__ int kv8_value_field(int vf) { return vf == 255 ? 0 : vf; }

__device__ __forceinline__ void kv8_store_pair(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void kv8_store_pair(bf16* p, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b); }
// What a row's reference is raised by at the end (0: as it is).  Sums of weighted values are 127.5 wsum 2^(unit - 133) at most: from 2^118 on the
// weights' sum l is brought to [2^-10, 2^-9), which leaves the joins room.  (Raised always, a reference with a fraction would be
// rounded once more.)
__device__ __forceinline__ int kv8_excess(float l, float wsum, float unit) {
  const int at = (int)(__float_as_uint(wsum) >> 23) - 127;
  return (float)at + unit >= 244.f ? min((int)(__float_as_uint(l) >> 23), 243) - 117 : 0;
}
__device__ __forceinline__ float kv8_ratio(float o, float l) { return l == 0.f ? 0.f : o / l; }

// --------------------------------------------------------------------------------------------
// Whole form: grid (blocks of 32 NT rows, key heads, requests); a warp has 8 NT rows over all their keys.
// --------------------------------------------------------------------------------------------
template <typename S>
__global__ void __launch_bounds__(32 * WARPS)
kv8_attention_whole_kernel(Kv8Args a) {
  constexpr int NT = S::ROW_TILES, TILE = S::TILE;
  ifb_pdl_wait();
  ifb_pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.z, kv_head = blockIdx.y, G = a.heads / a.kv_heads;
  const int q0 = a.cu_q[r], q_len = a.cu_q[r + 1] - q0, L = a.seq_lens[r], rows = q_len * G;
  if (q_len <= 0 || rows < a.min_rows || rows > a.max_rows) return;
  // the rows with the most keys first
  const int row0 = ((int)(gridDim.x - 1 - blockIdx.x) * WARPS + warp) * 8 * NT;
  if (row0 >= rows) return;
  const int pos0 = L - q_len, p_first = pos0 + row0 / G, p_last = pos0 + min(row0 + 8 * NT - 1, rows - 1) / G;
  const int lo = a.window > 0 ? max(0, p_first - a.window + 1) : 0;
  Queries<NT> raw;
  request_queries<NT>(raw, a, q0, row0, rows, kv_head, G, lane);
  typename S::Walk walk(a, a.tables + (size_t)r * a.table_stride, kv_head, lo / 16, p_last / 16 + 1, lo / TILE, p_last >= 0 ? p_last / TILE + 1 : 0, 1, lane);
  S st;
  st.reset();
  st.queries(raw, row0, rows, pos0, G, lane);
  st.run(a, walk, a.window > 0 ? p_last - a.window + 1 : 0, p_first, lane);
  st.finish();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = row0 + n * 8 + (lane & 3) * 2 + e;
      if (row >= rows) continue;
      qtype* to = a.out + ((size_t)(q0 + row / G) * a.heads + kv_head * G + row % G) * D;
#pragma unroll
      for (int i = 0; i < KS; ++i)
        kv8_store_pair(to + value_dim<D>(i, lane, 0), kv8_ratio(st.o[i][n][e], st.l[n][e]), kv8_ratio(st.o[i][n][2 + e], st.l[n][e]));
    }
}

// --------------------------------------------------------------------------------------------
// Split form.  Items are (request, tile of 8 NT rows, key head), in that order; an item has the units of its request (those of
// the request's last row: earlier tiles leave a few empty), one at least, so that a row without keys is written.  A CTA has one
// piece of one item.  With `most` CTAs on the device at once and fewer items, pieces have total / (most - items) units or a little
// less, for which the pieces of all items are no more than `most`; else every item is one piece.  (Equal shares of the units, with
// CTAs that have the end of one item and the beginning of the next, are a tenth shorter and cost a second start and a second join.)
// --------------------------------------------------------------------------------------------
constexpr int MAX_PARTS = 64;            // pieces of an item
constexpr int PITCH = D + 8;             // of a row of sums in shared memory (the rows of a quad of lanes fall on two halves of the banks)
// Where a warp's sums lie in a row: m tile by m tile, the lanes' pairs side by side.
__device__ __forceinline__ int kv8_place(int i, int lane) { return i * 16 + (lane >> 2) * 2; }
__device__ __forceinline__ int kv8_place_dim(int place) { return value_dim<D>(place >> 4, ((place & 15) >> 1) << 2, 0); }

// What a lane knows of a request: where its queries lie, the units of an item and its items (0: not this kernel's).
struct Kv8Look { int q0, q_len, L, units, items; };
__device__ __forceinline__ Kv8Look kv8_ask(const Kv8Args& a, int r) {       // (the last request's numbers beyond it)
  const int at = min(r, a.requests - 1);
  Kv8Look k = {a.cu_q[at], a.cu_q[at + 1], a.seq_lens[at], 0, 0};
  return k;
}
template <int ROWS, int UNIT>
__device__ __forceinline__ Kv8Look kv8_look(const Kv8Args& a, int G, int r, Kv8Look k) {
  k.q_len -= k.q0;
  const int rows = k.q_len * G;
  if (r < a.requests && k.q_len > 0 && rows >= a.min_rows && rows <= a.max_rows) {
    k.items = (rows + ROWS - 1) / ROWS * a.kv_heads;
    const int lo = a.window > 0 ? max(0, k.L - k.q_len - a.window + 1) : 0;
    k.units = k.L > 0 ? max(1, (k.L - 1) / UNIT - lo / UNIT + 1) : 1;
  }
  return k;
}

// ceil(x / y) of whole numbers from 1 on, x below 2^20 (units of a request: 2^26 keys or more): the quotient's error is below the half that
// is taken off.
__device__ __forceinline__ int kv8_parts(int x, float inverse) { return (int)(((float)x - 0.5f) * inverse) + 1; }

// How long pieces are, and whose piece this CTA's is: request r (-1: there are more CTAs than pieces), number `at` of its items' pieces.
struct Kv8Plan { int r, at, units, pieces, q0, q_len, L; };
template <int ROWS, int UNIT>
__device__ __forceinline__ Kv8Plan kv8_plan(const Kv8Args& a, int G, int lane) {
  const Kv8Look asked = kv8_ask(a, lane), asked2 = kv8_ask(a, lane + 32);
  const Kv8Look known = kv8_look<ROWS, UNIT>(a, G, lane, asked), known2 = kv8_look<ROWS, UNIT>(a, G, lane + 32, asked2);
  int total = known.units * known.items + known2.units * known2.items, items = known.items + known2.items, longest = max(known.units, known2.units);
  for (int r = 64 + lane; r < a.requests; r += 32) {
    const Kv8Look k = kv8_look<ROWS, UNIT>(a, G, r, kv8_ask(a, r));
    total += k.units * k.items;
    items += k.items;
    longest = max(longest, k.units);
  }
  total = __reduce_add_sync(0xffffffffu, total);
  items = __reduce_add_sync(0xffffffffu, items);
  longest = __reduce_max_sync(0xffffffffu, longest);
  // A unit takes some sixteen times what a piece adds to the join: no more than 4 sqrt(units) pieces.  (A request of 4,000 keys, 63 and 32 pieces:
  // on 8 key heads 13.5 and 12.3 us, on 2 18.1 and 13.9.  64 and not 32 pieces at the most: 32,000 keys 31.9 and 24.8.)
  const int spare = a.most - items, least = max((longest + MAX_PARTS - 1) / MAX_PARTS, (int)ceilf(sqrtf((float)longest) * 0.25f));
  int per = max(spare > 0 ? (int)((uint32_t)(total + spare - 1) / (uint32_t)spare) : longest, least);
  if (spare > 0 && a.requests <= 64) {
    // pieces up to four units shorter, as long as there are CTAs for them (the bound above counts an unfinished piece for every item)
    int shorter = 0;
#pragma unroll
    for (int i = 1; i <= 4; ++i) {
      const float inverse = 1.f / (float)max(per - i, 1);
      const int all = __reduce_add_sync(0xffffffffu, (known.items ? kv8_parts(known.units, inverse) : 0) * known.items +
                                                     (known2.items ? kv8_parts(known2.units, inverse) : 0) * known2.items);
      if (per - i >= least && all <= a.most) shorter = i;
    }
    per -= shorter;
  }
  const float per_inverse = 1.f / (float)per;
  // the first request whose pieces, with all before it, exceed this CTA's number: 64 of them at a time
  int r = -1, q0 = 0, q_len = 0, L = 0, units = 0, pieces = 0, at = blockIdx.x;
  for (int r0 = 0; r0 < a.requests; r0 += 64) {
    const Kv8Look k = r0 == 0 ? known : kv8_look<ROWS, UNIT>(a, G, r0 + lane, kv8_ask(a, r0 + lane));
    const Kv8Look k2 = r0 == 0 ? known2 : kv8_look<ROWS, UNIT>(a, G, r0 + lane + 32, kv8_ask(a, r0 + lane + 32));
    const int mine = k.items ? kv8_parts(k.units, per_inverse) : 0, mine2 = k2.items ? kv8_parts(k2.units, per_inverse) : 0;
    const int own = mine * k.items, own2 = mine2 * k2.items;
    int upto = own, upto2 = own2;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, d), y2 = __shfl_up_sync(0xffffffffu, upto2, d);
      if (lane >= d) { upto += y; upto2 += y2; }
    }
    upto2 += __shfl_sync(0xffffffffu, upto, 31);
    const uint32_t hit = __ballot_sync(0xffffffffu, at < upto), hit2 = __ballot_sync(0xffffffffu, at < upto2);
    if (hit | hit2) {
      const bool second = hit == 0;
      const int src = __ffs(second ? hit2 : hit) - 1;
      r = r0 + src + (second ? 32 : 0);
      at -= __shfl_sync(0xffffffffu, second ? upto2 - own2 : upto - own, src);
      units = __shfl_sync(0xffffffffu, second ? k2.units : k.units, src);
      pieces = __shfl_sync(0xffffffffu, second ? mine2 : mine, src);
      q0 = __shfl_sync(0xffffffffu, second ? k2.q0 : k.q0, src);
      q_len = __shfl_sync(0xffffffffu, second ? k2.q_len : k.q_len, src);
      L = __shfl_sync(0xffffffffu, second ? k2.L : k.L, src);
      break;
    }
    at -= __shfl_sync(0xffffffffu, upto2, 31);
  }
  return {r, at, units, pieces, q0, q_len, L};
}

__device__ __forceinline__ void kv8_add(float4& o, const float4& x, float f) {
  o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w);
}
// Four numbers side by side (two neighbouring lanes' pairs) of score row `row`; out: the request's first token at the key head's first query head.
__device__ __forceinline__ void kv8_finish(qtype* out, int row, int G, int heads, int place, const float4& o, float l) {
  qtype* to = out + ((size_t)(row / G) * heads + row % G) * D;
  kv8_store_pair(to + kv8_place_dim(place), kv8_ratio(o.x, l), kv8_ratio(o.y, l));
  kv8_store_pair(to + kv8_place_dim(place + 2), kv8_ratio(o.z, l), kv8_ratio(o.w, l));
}
// The sums of an item's pieces, in their order, by the CTA that arrived last (`first`: of piece 0).  A group's sums are on their way while it looks
// at the maxima of all, and while the group before is added.  A call, so that the loop over the keys does not share its registers.
template <int ROWS>
__device__ __noinline__ void kv8_join(const float* first, float* room, int pieces, int here, int row0, int G, int heads, qtype* out) {
  float (*const part_m)[ROWS] = reinterpret_cast<float (*)[ROWS]>(room), (*const part_l)[ROWS] = part_m + MAX_PARTS;      // in shared memory
  constexpr int GROUP = 8;
  struct Group { float4 x[GROUP]; };
  const int tid = threadIdx.x;
  auto request = [&](Group& g, int i, int c0) {                         // number i of a piece's sums, of the pieces from c0 on
    const float* from = first + (size_t)c0 * ROWS * (D + 2) + i * 4;
#pragma unroll
    for (int c = 0; c < GROUP; ++c)
      if (c0 + c < pieces) g.x[c] = __ldcg(reinterpret_cast<const float4*>(from + (size_t)c * ROWS * (D + 2)));
  };
  Group now, next;
  if (tid < here * (D / 4)) request(now, tid, 0);
  for (int i = tid; i < here * pieces; i += 32 * WARPS) {
    const int c = i / here, row = i - c * here;
    const float* from = first + (size_t)c * ROWS * (D + 2) + ROWS * D + row;
    part_m[c][row] = __ldcg(from);
    part_l[c][row] = __ldcg(from + ROWS);
  }
  __syncthreads();
  for (int i = tid; i < here * (D / 4); i += 32 * WARPS) {
    const int row = i / (D / 4);
    float M = -INFINITY, l = 0.f;
    if (i != tid) request(now, i, 0);
    for (int c = 0; c < pieces; ++c) M = fmaxf(M, part_m[c][row]);
    const float U = M == -INFINITY ? 0.f : M;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = 0; c0 < pieces; c0 += GROUP) {
      if (c0 + GROUP < pieces) request(next, i, c0 + GROUP);
#pragma unroll
      for (int c = 0; c < GROUP; ++c)
        if (c0 + c < pieces) {
          const float f = kv8_exp2(part_m[c0 + c][row] - U);
          kv8_add(o, now.x[c], f);
          l = fmaf(part_l[c0 + c][row], f, l);
        }
      now = next;
    }
    kv8_finish(out, row0 + row, G, heads, (i - row * (D / 4)) * 4, o, l);
  }
}

template <typename S>
__global__ void __launch_bounds__(32 * WARPS, S::CTAS)
kv8_attention_split_kernel(Kv8Args a) {
  constexpr int NT = S::ROW_TILES, ROWS = 8 * NT, TILE = S::TILE, UNIT = TILE * WARPS;
  extern __shared__ __align__(16) float sums[];        // [WARPS][ROWS][PITCH], then maxima and sums [WARPS][ROWS] each; in the join the pieces'
  __shared__ int arrived;
  ifb_pdl_wait();
  ifb_pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.heads / a.kv_heads;
  float* const sm_m = sums + WARPS * ROWS * PITCH;
  float* const sm_l = sm_m + WARPS * ROWS;
  const Kv8Plan plan = kv8_plan<ROWS, UNIT>(a, G, lane);                // every warp for itself
  const int r = plan.r, q0 = plan.q0, q_len = plan.q_len, L = plan.L, units = plan.units, pieces = plan.pieces, at = plan.at;
  if (r < 0) return;                                                    // more CTAs than pieces
  const int item = (uint32_t)at / (uint32_t)pieces, piece = at - item * pieces, tile = (uint32_t)item / (uint32_t)a.kv_heads, kv_head = item - tile * a.kv_heads;
  const int rows = q_len * G, row0 = tile * ROWS, here = min(ROWS, rows - row0);
  const int pos0 = L - q_len, p_first = pos0 + row0 / G, p_last = pos0 + (row0 + here - 1) / G;
  const int lo_request = a.window > 0 ? max(0, pos0 - a.window + 1) : 0, lo = a.window > 0 ? max(0, p_first - a.window + 1) : 0;
  const int each = (units + pieces - 1) / pieces;                       // units of a piece
  const int key0 = (lo_request / UNIT + piece * each) * UNIT, key_end = min(p_last + 1, key0 + each * UNIT);
  Queries<NT> raw;
  request_queries<NT>(raw, a, q0, row0, rows, kv_head, G, lane);
  typename S::Walk walk(a, a.tables + (size_t)r * a.table_stride, kv_head, lo / 16, p_last / 16 + 1, max(key0, lo) / TILE + warp,
                                 key_end > 0 ? (key_end + TILE - 1) / TILE : 0, WARPS, lane);
  S st;
  st.reset();
  st.queries(raw, row0, rows, pos0, G, lane);
  st.run(a, walk, a.window > 0 ? p_last - a.window + 1 : 0, p_first, lane);
  st.finish();
  // the warps' sums side by side
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = n * 8 + (lane & 3) * 2 + e;
      if (row < here) {
        float* to = sums + (warp * ROWS + row) * PITCH;
#pragma unroll
        for (int i = 0; i < KS; ++i) *reinterpret_cast<float2*>(to + kv8_place(i, lane)) = make_float2(st.o[i][n][e], st.o[i][n][2 + e]);
        if (lane < 4) { sm_m[warp * ROWS + row] = st.m[n][e]; sm_l[warp * ROWS + row] = st.l[n][e]; }
      }
    }
  __syncthreads();
  float* const mine = a.parts + (size_t)blockIdx.x * ROWS * (D + 2);
  for (int i = tid; i < here * (D / 4); i += 32 * WARPS) {
    const int row = i / (D / 4), place = (i - row * (D / 4)) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm_m[w * ROWS + row]);
    const float U = M == -INFINITY ? 0.f : M;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = kv8_exp2(sm_m[w * ROWS + row] - U);
      kv8_add(o, *reinterpret_cast<const float4*>(sums + (w * ROWS + row) * PITCH + place), f);
      l = fmaf(sm_l[w * ROWS + row], f, l);
    }
    if (pieces == 1) {
      kv8_finish(a.out + ((size_t)q0 * a.heads + kv_head * G) * D, row0 + row, G, a.heads, place, o, l);
    } else {
      *reinterpret_cast<float4*>(mine + row * D + place) = o;
      if (place == 0) { mine[ROWS * D + row] = M; mine[ROWS * (D + 1) + row] = l; }
    }
  }
  if (pieces == 1) return;
  __syncthreads();
  int* const counter = a.counters + ((size_t)r * a.tiles + tile) * a.kv_heads + kv_head;
  if (tid == 0) {                                                       // its fence covers what the barrier ordered before it
    __threadfence();
    arrived = atomicAdd(counter, 1);
    __threadfence();
  }
  __syncthreads();
  if (arrived != pieces - 1) return;
  kv8_join<ROWS>(mine - (size_t)piece * ROWS * (D + 2), sums, pieces, here, row0, G, a.heads, a.out + ((size_t)q0 * a.heads + kv_head * G) * D);
  if (tid == 0) *counter = 0;
}

template <typename S> static size_t kv8_split_smem() {
  constexpr int per_row = WARPS * (PITCH + 2) > 2 * MAX_PARTS ? WARPS * (PITCH + 2) : 2 * MAX_PARTS;
  return (size_t)8 * S::ROW_TILES * per_row * sizeof(float);
}
template <typename S> static int kv8_split_ctas(int* ctas) {                // that fit on the device at once
  static int known[IFB_MAX_DEVICES] = {};
  int dev = 0, per = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= IFB_MAX_DEVICES) return IFB_ERR_ARG;
  if (!known[dev]) {
    IFB_ALLOW_SMEM(kv8_attention_split_kernel<S>, kv8_split_smem<S>());
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kv8_attention_split_kernel<S>, 32 * WARPS, kv8_split_smem<S>());
    if (e != cudaSuccess) return -(int)e;
    known[dev] = (per < 1 ? 1 : per) * ifb_sm_count();
  }
  *ctas = known[dev];
  return IFB_OK;
}

// Floats of scratch memory that the split form of `nt` row tiles (1 to ifb_kv8_attention_tiles) wants, or a negative error.
template <typename S1, typename S2> static long long kv8_scratch(int nt) {
  int ctas = 0;
  const int bad = nt == 1 ? kv8_split_ctas<S1>(&ctas) : kv8_split_ctas<S2>(&ctas);
  return bad ? (bad > 0 ? -bad : bad) : (long long)ctas * 8 * nt * (D + 2);
}

template <typename S> static int kv8_launch_whole(const Kv8Args& a, int max_q, cudaStream_t stream) {
  const int rows = max_q * (a.heads / a.kv_heads);
  const dim3 grid((rows + 8 * S::ROW_TILES * WARPS - 1) / (8 * S::ROW_TILES * WARPS), a.kv_heads, a.requests);
  return ifb_launch(kv8_attention_whole_kernel<S>, grid, dim3(32 * WARPS), 0, stream, a);
}
template <typename S> static int kv8_launch_split(const Kv8Args& a, long long items, cudaStream_t stream) {
  int ctas = 0;
  const int bad = kv8_split_ctas<S>(&ctas);
  if (bad) return bad;
  // (with more items than CTAs at a time each is one piece, and needs no scratch memory)
  if (items > 0x7fffffffLL) return IFB_ERR_SIZE;
  Kv8Args b = a;
  b.most = ctas;
  return ifb_launch(kv8_attention_split_kernel<S>, dim3(items > ctas ? (unsigned)items : (unsigned)ctas), dim3(32 * WARPS), kv8_split_smem<S>(), stream, b);
}

// nt: tiles of 8 score rows per warp (split form).  whole: the whole form, of TILES such tiles.  Requests of min_rows .. max_rows score rows are worked on.  Split form:
// `tiles` tiles of a request at most, `items` (tiles x key heads) of all requests.
// One argument, since a call's price on the host is that of its arguments.
struct Kv8Call {
  const void* q;
  long long dtype, q_row;
  const void *codes, *exponents, *tables;
  long long table_stride;
  const void *cu_q, *seq_lens;
  void *out, *parts, *counters;
  long long requests, heads, kv_heads, page_size, dim, window, max_q, min_rows, max_rows, tiles, nt, whole, items;
  void* stream;
  double scale;
};
template <typename S1, typename S2> static int kv8_call(const Kv8Call* c) {
  const bool whole = c->whole != 0;
  if (c->dtype != (KV8_F32 ? IFB_F32 : IFB_BF16)) return IFB_ERR_DTYPE;
  if (c->dim != D || c->heads < 1 || c->kv_heads < 1 || c->heads % c->kv_heads || c->page_size < 16 || c->page_size % 16 || c->requests < 1 ||
      c->max_q < 1 || c->window < 0 || c->nt < 1 || c->nt > TILES || c->kv_heads > 65535 || c->requests > 65535 || c->max_q > 0x7fffffff ||
      c->window > 0x7fffffff || c->heads > 0x7fffffff || 2 * c->kv_heads * c->page_size * D > 0xffffffffLL)
    return IFB_ERR_SIZE;
  if (!whole && (!c->parts || !c->counters || c->tiles < 1)) return IFB_ERR_ARG;
  if ((((uintptr_t)c->q) | ((uintptr_t)c->codes) | ((uintptr_t)c->out) | (uintptr_t)(c->q_row * sizeof(qtype))) & 15) return IFB_ERR_ALIGN;
  const Kv8Args a = {(const qtype*)c->q, c->q_row, (const int8_t*)c->codes, (const uint8_t*)c->exponents, (const int*)c->tables, (int)c->table_stride,
                     (const int*)c->cu_q, (const int*)c->seq_lens, (qtype*)c->out, (float*)c->parts, (int*)c->counters, (int)c->requests, (int)c->heads,
                     (int)c->kv_heads, (int)c->page_size, (int)c->window, (float)c->scale * 1.4426950408889634f, (int)c->min_rows, (int)c->max_rows,
                     (int)c->tiles, 0};
  cudaStream_t stream = (cudaStream_t)c->stream;
  if (whole) return kv8_launch_whole<S2>(a, (int)c->max_q, stream);
  return c->nt == 1 ? kv8_launch_split<S1>(a, c->items, stream) : kv8_launch_split<S2>(a, c->items, stream);
}

// The library's calls over the file's streams of one and of TILES row tiles.
#define KV8_ENTRIES(S1, S2)                                                                     \
  IFB_EXPORT int ifb_kv8_attention_tiles() { return TILES; }                                    \
  IFB_EXPORT long long ifb_kv8_attention_scratch(int nt) { return kv8_scratch<S1, S2>(nt); }    \
  IFB_EXPORT int ifb_kv8_attention(const Kv8Call* c) { return kv8_call<S1, S2>(c); }
