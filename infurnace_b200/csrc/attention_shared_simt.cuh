// Attention over shared pages in 32-bit arithmetic, for any head size up to 256, any page size and float32 or bfloat16 storage: what
// attention_shared.cuh cuts into pieces, worked on by plain multiply-adds.
//
// A tile is up to 64 score rows (query tokens times the heads of a key head), a unit 32 keys, which the 256 threads of a CTA bring to shared memory as float32,
// by asynchronous copies a unit ahead (heads over 128: there is room for one unit, which is brought when the one before has been read); where a key
// lies is looked up two units ahead.  Thread (y, x) has score rows 2y and 2y + 1: of the scores keys x, x + 8, x + 16 and x + 24, of the sums the columns
// 4 x + 32 j .. + 3.  Rows of keys are padded by four numbers, so that eight lanes that read eight keys 16 bytes at a time meet no bank twice.
//
// What bounds it is a chain of units of 2 to 3 us each (a warp's 2,000 multiply-adds and what they read from shared memory, two warps to a scheduler), behind 4 us of
// plan and first keys; before copies ran ahead and columns came four at a time a unit took 15 to 20 us (nine answers to 1,296 keys 32.3 us, now 19.4; 32
// requests' tokens to 320 shared keys and up to 200 of their own, 12 on 4 heads of 96, 72 to 29; four portions of 121 queries, 8 on 2 heads of 256, 118 to 52).
#pragma once
#include "attention_shared.cuh"
#include <type_traits>

using namespace shared_attention;

constexpr int SH_ROWS = 64, SH_UNIT = 32, SH_THREADS = 256;
static_assert(SH_UNIT == 1 << 5, "unit_log");
__host__ __device__ constexpr int sh_stages(int nj) { return nj <= 4 ? 2 : 1; }

// Four numbers to shared memory, zeros where there are none; float32 without waiting for them.
template <typename T> __device__ __forceinline__ void sh_row4(float* dst, const T* src, bool valid) {
  if constexpr (sizeof(T) == 4) {
    const int size = valid ? 16 : 0;      // 0: src is not read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(size) : "memory");
  } else {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (valid) {
      const uint2 u = *reinterpret_cast<const uint2*>(src);
      v = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
    }
    *reinterpret_cast<float4*>(dst) = v;
  }
}
__device__ __forceinline__ void sh_store4(float* dst, float4 v) { *reinterpret_cast<float4*>(dst) = v; }
__device__ __forceinline__ void sh_store4(__nv_bfloat16* dst, float4 v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// NJ: 32 columns each, as many as the head has.
template <typename T, int NJ>
__global__ void __launch_bounds__(SH_THREADS) shared_simt_kernel(const __grid_constant__ Call c, const T* q, long long q_row, const T* pages, int dim) {
  constexpr int STAGES = sh_stages(NJ);
  extern __shared__ __align__(16) unsigned char sh_smem[];
  __shared__ long long places[2][SH_UNIT];      // of the keys of two units: the first element in the pool, or -1
  const Plan plan = plan_at(sh_smem, c.n_groups + c.n_req);
  const int pitch = dim + 4;
  float* Q = reinterpret_cast<float*>(sh_smem + plan_bytes(c.n_groups + c.n_req));      // [64][pitch]
  float* KV = Q + SH_ROWS * pitch;                                                      // [STAGES][2][32][pitch]
  float* P = KV + STAGES * 2 * SH_UNIT * pitch;                                         // [64][33]
  ifb_pdl_wait();
  ifb_pdl_trigger();
  make_plan(c, c, plan);
  Walk walk;
  walk.begin(c, plan, blockIdx.x, c.workers);
  write_parts(c, c, plan);
  const int tid = threadIdx.x, x = tid & 7, y = tid >> 3, quads = dim / 4;
  const int group = c.heads / c.kv_heads;
  const long long values = (long long)c.kv_heads * c.page_size * dim;      // from a page's keys to its values
  Piece p;
  while (walk.next(c, plan, p)) {
    const int rows = p.tokens * group, units = (p.last - p.first + SH_UNIT - 1) / SH_UNIT;
    auto place = [&](int u) {      // of the unit's key tid
      const int key = p.first + u * SH_UNIT + tid;
      long long at = -1;
      if (key >= p.lo && key < p.last) {
        at = page_at(c, p.w.table(key), key / c.page_size);
        if (at < 0) atomicExch(c.err, IFB_DEV_ERR_SHARED_PAGE);
        else at += ((long long)p.kv_head * c.page_size + key % c.page_size) * dim;
      }
      return at;
    };
    auto bring = [&](int u) {
      float* to = KV + u % STAGES * (2 * SH_UNIT * pitch);
#pragma unroll 4
      for (int i = tid; i < SH_UNIT * quads; i += SH_THREADS) {
        const int key = i / quads, col = i % quads * 4;
        const long long at = places[u & 1][key];
        const T* src = pages + (at < 0 ? 0 : at + col);
        sh_row4(to + key * pitch + col, src, at >= 0);
        sh_row4(to + (SH_UNIT + key) * pitch + col, src + (at < 0 ? 0 : values), at >= 0);
      }
      asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    __syncthreads();      // the piece before has read its tiles
    if (tid < SH_UNIT) {
      const long long a = place(0), b = units > 1 ? place(1) : -1;
      places[0][tid] = a; places[1][tid] = b;
    }
    for (int i = tid; i < SH_ROWS * quads; i += SH_THREADS) {
      const int row = i / quads, col = i % quads * 4;
      sh_row4(Q + row * pitch + col, q + (row < rows ? (p.row0 + row / group) * q_row + (long long)(p.kv_head * group + row % group) * dim + col : 0), row < rows);
    }
    int hi[2], lo[2];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float4 o[2][NJ];
    int all_lo = 0, all_hi = 0x7fffffff;      // what all rows of the warp that exist see
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = 2 * y + e;
      const int pos = row < rows ? row_position(c, plan, p.w, p.row0 + row / group) : NO_POSITION;
      hi[e] = min(pos + 1, p.last);      // the row sees lo .. hi - 1 of the piece
      lo[e] = max(p.lo, c.window > 0 ? pos - c.window + 1 : 0);
      if (row < rows) { all_lo = max(all_lo, lo[e]); all_hi = min(all_hi, hi[e]); }
#pragma unroll
      for (int j = 0; j < NJ; ++j) o[e][j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    all_lo = __reduce_max_sync(0xffffffffu, all_lo);
    all_hi = __reduce_min_sync(0xffffffffu, all_hi);
    const bool work = (2 * y & ~7) < rows;      // some row of the warp's eight exists
    __syncthreads();
    bring(0);
    for (int u = 0; u < units; ++u) {
      const int key0 = p.first + u * SH_UNIT;
      long long ahead = -1;
      if (tid < SH_UNIT && u + 2 < units) ahead = place(u + 2);
      if (STAGES == 2 && u + 1 < units) {
        bring(u + 1);
        asm volatile("cp.async.wait_group 1;\n" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");
      }
      __syncthreads();
      const float *Ks = KV + u % STAGES * (2 * SH_UNIT * pitch), *Vs = Ks + SH_UNIT * pitch;
      if (work) {
        float s[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[e][k] = 0.f;
#pragma unroll 2
        for (int d = 0; d < dim; d += 4) {
          float4 a[2], b[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) a[e] = *reinterpret_cast<const float4*>(Q + (2 * y + e) * pitch + d);
#pragma unroll
          for (int k = 0; k < 4; ++k) b[k] = *reinterpret_cast<const float4*>(Ks + (x + 8 * k) * pitch + d);
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              s[e][k] = fmaf(a[e].x, b[k].x, s[e][k]);
              s[e][k] = fmaf(a[e].y, b[k].y, s[e][k]);
              s[e][k] = fmaf(a[e].z, b[k].z, s[e][k]);
              s[e][k] = fmaf(a[e].w, b[k].w, s[e][k]);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = -INFINITY;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int key = key0 + x + 8 * k;
            s[e][k] = key >= lo[e] && key < hi[e] ? s[e][k] * c.scale_log2 : -INFINITY;
            top = fmaxf(top, s[e][k]);
          }
#pragma unroll
          for (int d = 1; d < 8; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          const float next = fmaxf(m[e], top), ref = next == -INFINITY ? 0.f : next;
          const float f = exp2f(m[e] - ref);
          m[e] = next;
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int key = key0 + x + 8 * k;
            const float w = key >= lo[e] && key < hi[e] ? exp2f(s[e][k] - ref) : 0.f;
            sum += w;
            P[(2 * y + e) * 33 + x + 8 * k] = w;
          }
          l[e] = fmaf(l[e], f, sum);
#pragma unroll
          for (int j = 0; j < NJ; ++j) { o[e][j].x *= f; o[e][j].y *= f; o[e][j].z *= f; o[e][j].w *= f; }
        }
        __syncwarp();      // (a warp's rows of P are its own)
        auto add = [&](auto masked) {
#pragma unroll 4
          for (int k = 0; k < SH_UNIT; ++k) {
            const float w0 = P[(2 * y) * 33 + k], w1 = P[(2 * y + 1) * 33 + k];
            const bool s0 = !decltype(masked)::value || (key0 + k >= lo[0] && key0 + k < hi[0]), s1 = !decltype(masked)::value || (key0 + k >= lo[1] && key0 + k < hi[1]);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {      // (columns beyond the head are what lies behind the row, and go nowhere)
              const float4 v = *reinterpret_cast<const float4*>(Vs + k * pitch + 4 * x + 32 * j);
              if (s0) { o[0][j].x = fmaf(w0, v.x, o[0][j].x); o[0][j].y = fmaf(w0, v.y, o[0][j].y); o[0][j].z = fmaf(w0, v.z, o[0][j].z); o[0][j].w = fmaf(w0, v.w, o[0][j].w); }
              if (s1) { o[1][j].x = fmaf(w1, v.x, o[1][j].x); o[1][j].y = fmaf(w1, v.y, o[1][j].y); o[1][j].z = fmaf(w1, v.z, o[1][j].z); o[1][j].w = fmaf(w1, v.w, o[1][j].w); }
            }
          }
        };
        if (key0 >= all_lo && key0 + SH_UNIT <= all_hi) add(std::false_type());
        else add(std::true_type());      // what a row does not see may be infinite or NaN
      }
      if (tid < SH_UNIT) places[u & 1][tid] = ahead;      // (this unit's were used a barrier ago)
      __syncthreads();
      if (STAGES == 1 && u + 1 < units) bring(u + 1);
    }
    const int2 workers = walk.item_workers(c, p, blockIdx.x);
    const bool sole = is_sole(p, workers);
    const long long slot = (long long)(p.item + blockIdx.x) * c.rows;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = 2 * y + e;
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
      if (row >= rows) continue;
      const float inv = !sole ? 1.f : l[e] > 0.f ? 1.f / l[e] : l[e] == 0.f ? 0.f : l[e];      // (NaN stays)
      T* dst = reinterpret_cast<T*>(c.out) + ((long long)(p.row0 + row / group) * c.heads + p.kv_head * group + row % group) * dim;
      if (!sole && x == 0) c.part_ml[slot + row] = make_float2(m[e], l[e]);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int col = 4 * x + 32 * j;
        if (col >= dim) continue;
        if (sole) sh_store4(dst + col, make_float4(o[e][j].x * inv, o[e][j].y * inv, o[e][j].z * inv, o[e][j].w * inv));
        else sh_store4(c.part_o + (slot + row) * dim + col, o[e][j]);
      }
    }
    if (tid == 0) c.pieces[p.item] = workers;
  }
}

static inline Call sh_call(int n_tokens, int n_req, int n_groups, int kv_heads, int group, int ctas) {      // (ctas: of an SM)
  Call c = {};
  c.which = EVERY;
  c.n_tokens = n_tokens; c.n_req = n_req; c.n_groups = n_groups;
  c.kv_heads = kv_heads; c.heads = kv_heads * group;
  c.tokens = SH_ROWS / group; c.rows = SH_ROWS; c.unit_log = 5; c.align_log = 0;
  c.workers = ifb_sm_count() * ctas;
  c.extra = 1;
  return c;
}
// (one function for each kernel: what IFB_ALLOW_SMEM remembers is a kernel's)
template <typename T, int NJ>
static int sh_main(const Call& c, const T* q, long long q_row, const T* pages, int dim, cudaStream_t stream) {
  const size_t smem = plan_bytes(c.n_req + c.n_groups) + (size_t)((SH_ROWS + sh_stages(NJ) * 2 * SH_UNIT) * (dim + 4) + SH_ROWS * 33) * 4;
  if (smem > MOST_SMEM) return IFB_ERR_SIZE;
  IFB_ALLOW_SMEM((shared_simt_kernel<T, NJ>), smem);
  return ifb_launch(shared_simt_kernel<T, NJ>, dim3(c.workers), dim3(SH_THREADS), smem, stream, c, q, q_row, pages, dim);
}
