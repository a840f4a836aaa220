// Keys and values held in 8 bits with a scale for each page, kind (keys or values) and head: the store, and the values that
// the bits stand for.
//
// The definition.  A block is what a page holds of one head's keys or values; f is the exponent field of its largest magnitude
// as a float32 number, step = 2^(f - 133), a code is floor(x / step), which lies in [-128, 127], and stands for (code + 1/2)
// step.  Floors nest: floor(floor(x / s) / 2^d) = floor(x / (s 2^d)), so when a token with a larger number joins a page, a
// shift of the older codes to the right makes them what they would be had all been stored at once, and how the same numbers
// are cut over calls leaves no trace in a page's bits.  (With rounding to nearest in place of floor, the second rounding would.)  f = 0 (all
// numbers zero or subnormal): the values are 0; f = 255 (an infinity or NaN): they are NaN.
//
// Layout: codes int8 [pages][2][heads][page_size][dim], exponents uint8 [pages][2][heads].
#include "common.cuh"

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ float kv8_step(uint32_t f) {                 // 2^(f - 133), 0, NaN
  if (f == 0u) return 0.f;
  if (f == 255u) return __uint_as_float(0x7fffffffu);
  return f > 6u ? __uint_as_float((f - 6u) << 23) : __uint_as_float(1u << (f + 16u));
}
// Codes of numbers whose block has the exponent field f: floor(x / step) is the lowest byte of x / step + 1.5 2^23, rounded downwards
// once (a tiny negative number thus stays below zero).  1 / step = 2^(133 - f) is no float for the smallest f, whose numbers are
// multiplied by 2^64 first; f = 0: any negative number is -1.
struct Kv8Rounding { float before, factor; };
__device__ __forceinline__ Kv8Rounding kv8_rounding(uint32_t f) {
  if (f > 6u) return {1.f, __uint_as_float((260u - min(f, 254u)) << 23)};
  return {__uint_as_float(191u << 23), f ? __uint_as_float((196u - f) << 23) : 1.f};
}
__device__ __forceinline__ uint32_t kv8_codes4(const float* x, const Kv8Rounding& r) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = __float_as_uint(__fmaf_rd(x[i] * r.before, r.factor, 12582912.f));
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}

// A warp per (place, kind, head).  A run is the adjacent rows whose slots follow one another in one page; the warp of place p has the runs that
// begin in rows p, p + 257, p + 514 ..: up to 257 decoding rows have a place each, and since 257 is 1 more than a multiple of a usual
// page, the runs of a prompt fall on all places alike.  (A page's rows must be one run: the caller's contract.)  A warp's time is a
// run's way through memory and back: places and not windows of 16 rows, 2,048 rows of 8 heads of 128: a prompt 6.1 us and 5.7 (bytes alone
// 1.9), beside 48 single tokens 6.8 and 21.5, all single tokens 25.8 and 32.1; a place for every row 11.0, 11.4 and 23.2.
// A lane keeps HELD pieces of eight numbers in registers between the search for the largest and the rounding (a page of 16 tokens of heads
// of 128 in bfloat16 whole); of longer runs the rest is read again, from the first level of cache.
template <typename T> struct Piece8;
template <> struct Piece8<bf16> {
  uint4 w;
  __device__ __forceinline__ void load(const bf16* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void clear() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ uint32_t amax_bits() const {
    const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
    return max(m << 16, m & 0xffff0000u);
  }
  __device__ __forceinline__ void numbers(float (&v)[8]) const {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(x[i] << 16);
      v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
    }
  }
};
template <> struct Piece8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
  __device__ __forceinline__ void clear() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ uint32_t amax_bits() const {
    float x[8];
    numbers(x);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ void numbers(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};
template <typename T>
__device__ __forceinline__ void kv8_store_run(const T* k, const T* v, long long k_row, long long v_row, const int* slots, int8_t* codes,
                                              uint8_t* exponents, int rows, int heads, int page_size, int dim, int row0, int slot, int block, int lane) {
  const int page = slot / page_size, first = slot - page * page_size;
  int n = 1;                                                            // rows of the run
  for (int at = 1; at < page_size - first; at += 32) {
    const int i = at + lane;
    const bool in = i < page_size - first && row0 + i < rows && slots[row0 + i] == slot + i;
    const uint32_t miss = ~__ballot_sync(0xffffffffu, in);
    n = at + (miss ? __ffs(miss) - 1 : 32);
    if (miss) break;
  }
  const int kind = block / heads, head = block - kind * heads;
  const T* src = (kind ? v : k) + (size_t)row0 * (kind ? v_row : k_row) + (size_t)head * dim;
  const long long pitch = kind ? v_row : k_row;
  uint8_t* const exponent = exponents + ((size_t)page * 2 + kind) * heads + head;
  const uint32_t old = first ? *exponent : 0u;
  const int pieces = dim / 8, total = n * pieces;
  constexpr int HELD = sizeof(T) == 2 ? 8 : 4;
  auto at = [&](int i) { const int r = i / pieces; return src + r * pitch + (i - r * pieces) * 8; };
  Piece8<T> held[HELD];
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    if (lane + 32 * j < total) held[j].load(at(lane + 32 * j));
    else held[j].clear();
  }
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < HELD; ++j) m = max(m, held[j].amax_bits());
#pragma unroll 4
  for (int i = lane + 32 * HELD; i < total; i += 32) {
    Piece8<T> p;
    p.load(at(i));
    m = max(m, p.amax_bits());
  }
  m = __reduce_max_sync(0xffffffffu, m);
  const uint32_t f = max(old, m >> 23);
  int8_t* const to = codes + (((size_t)page * 2 + kind) * heads + head) * page_size * dim;
  if (first && f != old) {
    if (lane == 0) *exponent = (uint8_t)f;
    if (f != 255u) {
      // the page's other rows take the larger step
      const int shift = min((int)(f - old), 7);
      const int per = page_size * pieces;
      for (int i = lane; i < per; i += 32) {
        const int r = i / pieces;
        if (r >= first && r < first + n) continue;
        uint2* p = reinterpret_cast<uint2*>(to + (size_t)i * 8);
        uint2 c = *p;
        uint32_t* w = &c.x;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t q = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) q |= ((uint32_t)((int)(int8_t)(w[j] >> (8 * b)) >> shift) & 255u) << (8 * b);
          w[j] = q;
        }
        *p = c;
      }
    }
  }
  if (!first && lane == 0) *exponent = (uint8_t)f;
  const Kv8Rounding rounding = kv8_rounding(f);
  auto round = [&](int i, const Piece8<T>& p) {
    float x[8];
    p.numbers(x);
    *reinterpret_cast<uint2*>(to + (size_t)first * dim + (size_t)i * 8) = make_uint2(kv8_codes4(x, rounding), kv8_codes4(x + 4, rounding));
  };
#pragma unroll
  for (int j = 0; j < HELD; ++j)
    if (lane + 32 * j < total) round(lane + 32 * j, held[j]);
#pragma unroll 4
  for (int i = lane + 32 * HELD; i < total; i += 32) {
    Piece8<T> p;
    p.load(at(i));
    round(i, p);
  }
}

constexpr int KV8_PLACES = 257;
template <typename T>
__global__ void __launch_bounds__(256)
kv8_store_kernel(const T* k, const T* v, long long k_row, long long v_row, const int* slots, int8_t* codes, uint8_t* exponents, int rows,
                 int heads, int page_size, int dim) {
  ifb_pdl_wait();
  ifb_pdl_trigger();
  const int lane = threadIdx.x & 31, block = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (block >= 2 * heads) return;
  for (long long base = blockIdx.x; base < rows; base += 32LL * gridDim.x) {
    const long long row = base + (long long)lane * gridDim.x;
    int slot = -1, before = -1;
    if (row < rows) {
      slot = slots[row];
      if (row) before = slots[row - 1];
    }
    // a row begins a run if it is stored and does not follow the row before it in one page
    uint32_t begins = __ballot_sync(0xffffffffu, slot >= 0 && !(slot % page_size && before == slot - 1));
    while (begins) {
      const int src = __ffs(begins) - 1;
      begins &= begins - 1;
      kv8_store_run<T>(k, v, k_row, v_row, slots, codes, exponents, rows, heads, page_size, dim, (int)(base + (long long)src * gridDim.x),
                       __shfl_sync(0xffffffffu, slot, src), block, lane);
    }
  }
}

__device__ __forceinline__ float4 kv8_numbers4(uint32_t w, float step) {
  return make_float4(((float)(int8_t)(w) + 0.5f) * step, ((float)(int8_t)(w >> 8) + 0.5f) * step, ((float)(int8_t)(w >> 16) + 0.5f) * step,
                     ((float)(int8_t)(w >> 24) + 0.5f) * step);
}
// What 16 codes stand for, as bfloat16 (which, as float32, holds (code + 1/2) step exactly).
__device__ __forceinline__ void kv8_write16(bf16* to, const uint4& c, float step) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t y[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 v = kv8_numbers4(w[i], step);
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
    y[2 * i] = *reinterpret_cast<const uint32_t*>(&lo);
    y[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&hi);
  }
  *reinterpret_cast<uint4*>(to) = make_uint4(y[0], y[1], y[2], y[3]);
  *reinterpret_cast<uint4*>(to + 8) = make_uint4(y[4], y[5], y[6], y[7]);
}
// Bound by the bytes written.  A lane takes 16 codes; as float32 four of each of its warp's four rows of 128, so that a store fills whole
// lines.  8,000 pages of 16 tokens of 8 heads of 128: 121 us
// (6.5 TB/s), as float32 205 (6.4; 291 with a lane's 16 side by side).
template <typename T>
__global__ void __launch_bounds__(256)
kv8_values_kernel(const int8_t* codes, const uint8_t* exponents, T* out, long long pieces, int per_block) {
  ifb_pdl_wait();
  ifb_pdl_trigger();
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (long long)gridDim.x * 256) {
    if constexpr (sizeof(T) == 2) {
      kv8_write16(out + i * 16, *reinterpret_cast<const uint4*>(codes + i * 16), kv8_step(exponents[i / per_block]));
    } else {
      const int lane = threadIdx.x & 31;                                // (pieces are a multiple of 32: whole warps have one)
      const long long first = (i - lane) * 4 + lane;                    // in words of four codes
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = reinterpret_cast<const uint32_t*>(codes)[first + j * 32];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        reinterpret_cast<float4*>(out)[first + j * 32] = kv8_numbers4(w[j], kv8_step(exponents[(first + j * 32) / (4 * per_block)]));
    }
  }
}

// The pages of the requests with more than `above` score rows as bfloat16 pages, for a kernel that reads those: the pages that a
// request's queries see, one after the other over all such requests, and a table of them.  Exact, but for a block of NaN:
// either kind's makes the page's keys NaN and its values 0, so that rows that do not see the page keep their numbers (a weight
// of 0 times NaN would not be 0) and rows that see it are NaN.  Grid (pages of a request, 2 kinds, requests).  Bound by memory: a byte read and
// two written for each number: 2,000 pages of 16 tokens of 8 heads of 128 35 us, 5.6 TB/s.
__device__ __forceinline__ int kv8_first_page(int L, int q_len, int window, int page_size) {
  return window > 0 ? max(0, L - q_len - window + 1) / page_size : 0;
}
__global__ void __launch_bounds__(256)
kv8_expand_kernel(const int8_t* codes, const uint8_t* exponents, const int* tables, int table_stride, const int* cu_q, const int* seq_lens, bf16* out,
                  int* out_tables, int out_pages, int heads, int group, int page_size, int dim, int window, int above) {
  __shared__ int first_sum;
  ifb_pdl_wait();
  ifb_pdl_trigger();
  const int r = blockIdx.z, kind = blockIdx.y, p = blockIdx.x;
  const int q_len = cu_q[r + 1] - cu_q[r], L = seq_lens[r], first = kv8_first_page(L, q_len, window, page_size);
  if (q_len * group <= above || p * page_size >= L || p < first) return;
  if (threadIdx.x < 32) {
    int sum = 0;
    for (int i = threadIdx.x; i < r; i += 32) {
      const int n = cu_q[i + 1] - cu_q[i], l = max(0, seq_lens[i]);
      if (n * group > above) sum += (l + page_size - 1) / page_size - kv8_first_page(l, n, window, page_size);
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (threadIdx.x == 0) first_sum = sum;
  }
  __syncthreads();
  const int to = first_sum + p - first;
  if (to >= out_pages) return;                                          // (more keys than the caller said)
  const int page = tables[(size_t)r * table_stride + p];
  if (kind == 0 && threadIdx.x == 0) out_tables[(size_t)r * gridDim.x + p] = to;
  const uint8_t* fields = exponents + (size_t)page * 2 * heads;
  const int per_head = page_size * dim / 16, total = heads * per_head;
  const int8_t* src = codes + ((size_t)page * 2 + kind) * heads * page_size * dim;
  bf16* dst = out + ((size_t)to * 2 + kind) * heads * page_size * dim;
  for (int i = threadIdx.x; i < total; i += 256) {
    const int h = i / per_head;
    const bool nan = fields[h] == 255 || fields[heads + h] == 255;
    const float step = nan ? (kind ? 0.f : __uint_as_float(0x7fffffffu)) : kv8_step(fields[kind * heads + h]);
    kv8_write16(dst + (size_t)i * 16, *reinterpret_cast<const uint4*>(src + (size_t)i * 16), step);
  }
}

static int kv8_sizes(int heads, int page_size, int dim) {
  if (heads < 1 || heads > 32767 || page_size < 16 || page_size % 16 || page_size > 4096 || dim < 16 || dim % 16 || dim > 256) return IFB_ERR_SIZE;
  return IFB_OK;
}

IFB_EXPORT int ifb_kv8_store(const void* k, const void* v, int dtype, long long k_row, long long v_row, const void* slots, void* codes,
                             void* exponents, int rows, int heads, int page_size, int dim, void* stream) {
  const int bad = kv8_sizes(heads, page_size, dim);
  if (bad) return bad;
  if (rows < 1) return IFB_ERR_SIZE;
  if (dtype != IFB_F32 && dtype != IFB_BF16) return IFB_ERR_DTYPE;
  const int esize = dtype == IFB_F32 ? 4 : 2;
  if ((((uintptr_t)k) | ((uintptr_t)v) | (uintptr_t)(k_row * esize) | (uintptr_t)(v_row * esize) | ((uintptr_t)codes)) & 15) return IFB_ERR_ALIGN;
  const int warps = 2 * heads < 8 ? 2 * heads : 8;
  const dim3 grid(rows < KV8_PLACES ? rows : KV8_PLACES, (2 * heads + warps - 1) / warps);
  if (dtype == IFB_F32)
    return ifb_launch(kv8_store_kernel<float>, grid, dim3(32 * warps), 0, (cudaStream_t)stream, (const float*)k, (const float*)v, k_row, v_row,
                      (const int*)slots, (int8_t*)codes, (uint8_t*)exponents, rows, heads, page_size, dim);
  return ifb_launch(kv8_store_kernel<bf16>, grid, dim3(32 * warps), 0, (cudaStream_t)stream, (const bf16*)k, (const bf16*)v, k_row, v_row,
                    (const int*)slots, (int8_t*)codes, (uint8_t*)exponents, rows, heads, page_size, dim);
}

IFB_EXPORT int ifb_kv8_values(const void* codes, const void* exponents, void* out, int dtype, int pages, int heads, int page_size, int dim,
                              void* stream) {
  const int bad = kv8_sizes(heads, page_size, dim);
  if (bad) return bad;
  if (pages < 1) return IFB_ERR_SIZE;
  if (dtype != IFB_F32 && dtype != IFB_BF16) return IFB_ERR_DTYPE;
  if ((((uintptr_t)codes) | ((uintptr_t)out)) & 15) return IFB_ERR_ALIGN;
  const int per_block = page_size * dim / 16;
  const long long pieces = (long long)pages * 2 * heads * per_block;
  const long long blocks = (pieces + 255) / 256, most = (long long)ifb_sm_count() * 64;
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  if (dtype == IFB_F32)
    return ifb_launch(kv8_values_kernel<float>, grid, dim3(256), 0, (cudaStream_t)stream, (const int8_t*)codes, (const uint8_t*)exponents,
                      (float*)out, pieces, per_block);
  return ifb_launch(kv8_values_kernel<bf16>, grid, dim3(256), 0, (cudaStream_t)stream, (const int8_t*)codes, (const uint8_t*)exponents,
                    (bf16*)out, pieces, per_block);
}

// out: bfloat16 [out_pages][2][heads][page_size][dim], out_tables: int32 [requests][max_pages].
IFB_EXPORT int ifb_kv8_expand(const void* codes, const void* exponents, const void* tables, int table_stride, const void* cu_q, const void* seq_lens,
                              void* out, void* out_tables, int out_pages, int requests, int max_pages, int heads, int group, int page_size, int dim,
                              int window, int above, void* stream) {
  const int bad = kv8_sizes(heads, page_size, dim);
  if (bad) return bad;
  if (requests < 1 || requests > 65535 || max_pages < 1 || out_pages < 1 || group < 1) return IFB_ERR_SIZE;
  if ((((uintptr_t)codes) | ((uintptr_t)out)) & 15) return IFB_ERR_ALIGN;
  return ifb_launch(kv8_expand_kernel, dim3(max_pages, 2, requests), dim3(256), 0, (cudaStream_t)stream, (const int8_t*)codes, (const uint8_t*)exponents,
                    (const int*)tables, table_stride, (const int*)cu_q, (const int*)seq_lens, (bf16*)out, (int*)out_tables, out_pages, heads, group,
                    page_size, dim, window, above);
}
