// Attention over shared pages in 32-bit arithmetic, for any head size up to 256, any page size and float32 or bfloat16 storage: what
// attention_shared.cuh cuts into pieces, worked on by plain multiply-adds.
//
// A tile is up to 64 score rows (query tokens times the heads of a key head), a unit 32 keys.  The 256 threads of a CTA bring a unit's keys and values to
// shared memory as float32; thread (y, x) has score rows 2y and 2y + 1: of the scores keys x, x + 8, x + 16 and x + 24, of the sums columns
// x + 8 j.  Rows of keys are padded by four numbers, so that eight lanes that read eight keys 16 bytes at a time meet no bank twice.
#pragma once
#include "attention_shared.cuh"

using namespace shared_attention;

constexpr int SH_ROWS = 64, SH_UNIT = 32, SH_THREADS = 256;
static_assert(SH_UNIT == 1 << 5, "unit_log");

template <typename T>
__device__ __forceinline__ void sh_row4(float* dst, const T* src, bool valid) {      // four numbers
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (valid) {
    if constexpr (sizeof(T) == 4) v = *reinterpret_cast<const float4*>(src);
    else {
      const uint2 u = *reinterpret_cast<const uint2*>(src);
      v = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
    }
  }
  *reinterpret_cast<float4*>(dst) = v;
}

// parts: whether this kernel writes where the rows' pieces are.  DC: columns of a thread, the head size over eight rounded up to 8, 16 or 32.
template <typename T, int DC>
__global__ void __launch_bounds__(SH_THREADS) shared_simt_kernel(const __grid_constant__ Call c, const __grid_constant__ Call other, const T* q, long long q_row, const T* pages, int dim, int parts) {
  extern __shared__ __align__(16) unsigned char sh_smem[];
  const Plan plan = plan_at(sh_smem, c.n_groups + c.n_req);
  const int pitch = dim + 4;
  float* Q = reinterpret_cast<float*>(sh_smem + plan_bytes(c.n_groups + c.n_req));      // [64][pitch]
  float* Ks = Q + SH_ROWS * pitch;                                                      // [32][pitch]
  float* Vs = Ks + SH_UNIT * pitch;
  float* P = Vs + SH_UNIT * pitch;                                                      // [64][33]
  ifb_pdl_wait();
  ifb_pdl_trigger();
  make_plan(c, other, plan);
  Walk walk;
  const int ctas = c.which == EVERY ? c.workers : wide_sms(c.workers, plan.starts[c.n_groups + c.n_req] * c.cost, plan.sums[63] * other.cost);
  walk.begin(c, plan, blockIdx.x, ctas);
  if (parts) write_parts(c, other, plan);
  const int tid = threadIdx.x, x = tid & 7, y = tid >> 3, quads = dim / 4;
  const int group = c.heads / c.kv_heads;
  const long long values = (long long)c.kv_heads * c.page_size * dim;      // from a page's keys to its values
  Piece p;
  while (walk.next(c, plan, p)) {
    const int rows = p.tokens * group;
    __syncthreads();      // the piece before has read its tiles
    for (int i = tid; i < SH_ROWS * quads; i += SH_THREADS) {
      const int row = i / quads, col = i % quads * 4;
      sh_row4(Q + row * pitch + col, q + (p.row0 + row / group) * q_row + (long long)(p.kv_head * group + row % group) * dim + col, row < rows);
    }
    int hi[2], lo[2];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2][DC];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = 2 * y + e;
      const int pos = row < rows ? row_position(c, plan, p.w, p.row0 + row / group) : NO_POSITION;
      hi[e] = min(pos + 1, p.last);      // the row sees lo .. hi - 1 of the piece
      lo[e] = max(p.lo, c.window > 0 ? pos - c.window + 1 : 0);
#pragma unroll
      for (int j = 0; j < DC; ++j) o[e][j] = 0.f;
    }
    const bool work = (2 * y & ~7) < rows;      // some row of the warp's eight exists
    for (int key0 = p.first; key0 < p.last; key0 += SH_UNIT) {
      __syncthreads();      // the unit before has been read
      for (int i = tid; i < SH_UNIT * quads; i += SH_THREADS) {
        const int key = key0 + i / quads, col = i % quads * 4;
        const bool in = key >= p.lo && key < p.last;
        long long at = 0;
        bool valid = in;
        if (in) {
          at = page_at(c, p.w.table(key), key / c.page_size);
          valid = at >= 0;
          if (!valid) atomicExch(c.err, IFB_DEV_ERR_SHARED_PAGE);
          at += ((long long)p.kv_head * c.page_size + key % c.page_size) * dim + col;
        }
        sh_row4(Ks + i / quads * pitch + col, pages + at, valid);
        sh_row4(Vs + i / quads * pitch + col, pages + at + values, valid);
      }
      __syncthreads();
      if (!work) continue;
      float s[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[e][k] = 0.f;
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
        for (int j = 0; j < DC; ++j) o[e][j] *= f;
      }
      __syncwarp();      // (a warp's rows of P are its own)
      for (int k = 0; k < SH_UNIT; ++k) {
        const float w0 = P[(2 * y) * 33 + k], w1 = P[(2 * y + 1) * 33 + k];
        const bool s0 = key0 + k >= lo[0] && key0 + k < hi[0], s1 = key0 + k >= lo[1] && key0 + k < hi[1];
#pragma unroll
        for (int j = 0; j < DC; ++j) {
          if (x + 8 * j < dim) {
            const float v = Vs[k * pitch + x + 8 * j];
            if (s0) o[0][j] = fmaf(w0, v, o[0][j]);      // what a row does not see may be infinite or NaN
            if (s1) o[1][j] = fmaf(w1, v, o[1][j]);
          }
        }
      }
      __syncwarp();
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
      if (sole) {
        const float inv = l[e] > 0.f ? 1.f / l[e] : l[e] == 0.f ? 0.f : l[e];      // (NaN stays)
        T* dst = reinterpret_cast<T*>(c.out) + ((long long)(p.row0 + row / group) * c.heads + p.kv_head * group + row % group) * dim;
#pragma unroll
        for (int j = 0; j < DC; ++j)
          if (x + 8 * j < dim) dst[x + 8 * j] = from_f32<T>(o[e][j] * inv);
        continue;
      }
      if (x == 0) c.part_ml[slot + row] = make_float2(m[e], l[e]);
#pragma unroll
      for (int j = 0; j < DC; ++j)
        if (x + 8 * j < dim) c.part_o[(slot + row) * dim + x + 8 * j] = o[e][j];
    }
    if (tid == 0) c.pieces[p.item] = workers;
  }
}

static inline Call sh_call(int n_tokens, int n_req, int n_groups, int kv_heads, int group, int dim, Class which) {
  Call c = {};
  c.which = which;
  c.n_tokens = n_tokens; c.n_req = n_req; c.n_groups = n_groups;
  c.kv_heads = kv_heads; c.heads = kv_heads * group;
  c.tokens = SH_ROWS / group; c.rows = SH_ROWS; c.unit_log = 5; c.align_log = 0;
  c.workers = ifb_sm_count() * (which == EVERY && dim <= 128 ? 2 : 1);      // (registers: two CTAs on an SM; beside narrow owners one)
  c.cost = 16;
  c.extra = 1;
  return c;
}
// (one function for each kernel: what IFB_ALLOW_SMEM remembers is a kernel's)
template <typename T, int DC>
static int sh_main(const Call& c, const Call& other, const T* q, long long q_row, const T* pages, int dim, bool parts, cudaStream_t stream) {
  const size_t smem = plan_bytes(c.n_req + c.n_groups) + (size_t)((SH_ROWS + 2 * SH_UNIT) * (dim + 4) + SH_ROWS * 33) * 4;
  if (smem > MOST_SMEM) return IFB_ERR_SIZE;
  IFB_ALLOW_SMEM((shared_simt_kernel<T, DC>), smem);
  return ifb_launch(shared_simt_kernel<T, DC>, dim3(c.workers), dim3(SH_THREADS), smem, stream, c, other, q, q_row, pages, dim, parts ? 1 : 0);
}
