// Attention over shared pages for narrow owners (at most 16 score rows) of bfloat16 heads of HEAD_DIM: a request's decoded token over its own keys, and
// a few requests' over the keys they share.  attention_shared.cuh says how the work is cut and joined.
//
// The work is the reading of keys and values.  Every warp is a worker of its own: it walks over its pieces in chunks of 16 keys, which it brings to its part
// of shared memory by asynchronous copies of 16 bytes (any page size), two chunks ahead and across the ends of pieces, so that no warp waits for
// another and 2 x 4 warps of an SM have 130 KB on their way.  Products are mma.sync of bfloat16 with the keys, and then the columns of the values, on the
// side of 16 and the score rows on the side of eight, one or two times: S^T = K Q^T, O^T += V^T P^T.  (With the rows on the side of 16 a chunk of four rows
// took 48 products in place of 24, and their issue, some 16 cycles each, was the longest part of it.)  In both a thread has rows 2 (lane mod 4) and
// the next, so that the factors of a row's maximum need no exchange; weights cross over from accumulator to operand by movmatrix.  A row's weights
// are formed in float32 against its running maximum and enter the second product as two bfloat16 terms (16 bits of a weight); sums are float32.
#pragma once
#include "attention_shared.cuh"

using namespace shared_attention;

namespace narrow {

typedef __nv_bfloat16 bf16;
constexpr int WARPS = 4;
constexpr int CHUNK = 16, UNIT = 32;
constexpr int STAGES = 3;
constexpr int PITCH = D + 8;                          // rows in shared memory: 16 bytes more keep ldmatrix free of conflicts
constexpr int KB = D / 16;
constexpr int STAGE_ELEMENTS = 2 * CHUNK * PITCH;     // keys, then values
constexpr int WARP_BYTES = STAGES * STAGE_ELEMENTS * 2;
constexpr int CTAS_PER_SM = WARPS * WARP_BYTES <= 108 * 1024 ? 2 : 1;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(void* dst, const void* src, bool valid) {
  const int size = valid ? 16 : 0;      // 0: zeros, src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(size) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// An 8 x 8 matrix of 16-bit numbers, a row in four lanes, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
// A pair of weights as bfloat16: rounded, and the rounding of what that left out.
__device__ __forceinline__ void terms(float a, float b, uint32_t& first, uint32_t& second) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
  const float2 f = __bfloat1622float2(r);
  const __nv_bfloat162 s = __floats2bfloat162_rn(a - f.x, b - f.y);
  first = *reinterpret_cast<const uint32_t*>(&r);
  second = *reinterpret_cast<const uint32_t*>(&s);
}

// `beside`: the wide owners' kernel is the one before this in the stream; all its CTAs have waited for their own predecessor before this begins, and
// nothing that it writes is read here.  So this kernel waits for it at its end instead of at its start: who waits for this one has waited for both.
__global__ void __launch_bounds__(WARPS * 32, CTAS_PER_SM)
shared_narrow_kernel(const __grid_constant__ Call c, const __grid_constant__ Call other, const bf16* q, long long q_row, const bf16* pages, int sms, int beside) {
  extern __shared__ __align__(16) unsigned char narrow_smem[];
  if (!beside) ifb_pdl_wait();
  ifb_pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Plan plan = plan_at(narrow_smem, c.n_groups + c.n_req);
  bf16* stages = reinterpret_cast<bf16*>(narrow_smem + plan_bytes(c.n_groups + c.n_req) + (size_t)warp * WARP_BYTES);
  make_plan(c, other, plan);
  const int G = c.heads / c.kv_heads;
  // the SMs that the wide owners' kernel leaves
  const int mine = sms - wide_sms(sms, plan.sums[63] * other.cost, plan.starts[c.n_groups + c.n_req] * c.cost);
  const int worker = blockIdx.x * WARPS + warp, limit = min(c.workers, mine * CTAS_PER_SM * WARPS);
  const long long values = (long long)c.kv_heads * c.page_size * D;

  // ---- the copies' walk, ahead of the products'
  Walk ahead;
  ahead.begin(c, plan, worker, limit);
  Walk walk = ahead;      // the products'
  Piece ap;
  int akey = 0;
  bool more = ahead.next(c, plan, ap);
  if (more) akey = ap.first;
  int put = 0, page0 = 0, id = 0;      // the piece's pages page0 .. page0 + 31, one a lane
  bool fresh = true;
  auto request = [&]() {      // the next chunk of 16 keys, if there is one; a group of copies in any case
    if (more) {
      bf16* st = stages + put * STAGE_ELEMENTS;
      put = put + 1 == STAGES ? 0 : put + 1;
      // lanes 0 .. 15 (16 .. 31 likewise) find the places of the chunk's keys; the table is asked once for 32 pages
      const int key = akey + (lane & 15), page = key / c.page_size;
      if (fresh || __shfl_sync(0xffffffffu, page, 15) >= page0 + 32) {
        page0 = __shfl_sync(0xffffffffu, page, 0);
        const int first = (page0 + lane) * c.page_size;      // of the lane's page
        id = first < ap.last ? c.block_tables[ap.w.table(first) * c.bt_stride + page0 + lane] : -1;
        fresh = false;
      }
      const int mine = __shfl_sync(0xffffffffu, id, page - page0 & 31);
      long long at = -1;
      if (key >= ap.lo && key < ap.last) {
        if (mine < 0 || mine >= c.num_pages) atomicExch(c.err, IFB_DEV_ERR_SHARED_PAGE);
        else at = mine * c.page_stride + ((long long)ap.kv_head * c.page_size + key - page * c.page_size) * D;
      }
      constexpr int PARTS = D / 8;      // 16-byte parts of a row
#pragma unroll
      for (int i = 0; i < (CHUNK * PARTS + 31) / 32; ++i) {
        const int e = i * 32 + lane, row = e / PARTS, col = e % PARTS * 8;
        const long long from = __shfl_sync(0xffffffffu, at, row & 15);
        if (e < CHUNK * PARTS) {
          const bf16* src = pages + (from < 0 ? 0 : from + col);
          copy16(st + row * PITCH + col, src, from >= 0);
          copy16(st + (CHUNK + row) * PITCH + col, src + (from < 0 ? 0 : values), from >= 0);
        }
      }
      akey += CHUNK;
      if (akey >= ap.last) {
        more = ahead.next(c, plan, ap);
        if (more) akey = ap.first;
        fresh = true;
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) request();
  write_parts(other, c, plan);

  // ---- products
  Piece p;
  int get = 0;
  const int pair = (lane & 3) << 1;      // the thread's rows of a tile of eight: pair, pair + 1
  while (walk.next(c, plan, p)) {
    const int rows = p.tokens * G;
    const bool two = rows > 8;           // tiles of eight rows
    uint32_t qf[2][KB][2];               // rows lane / 4 and lane / 4 + 8
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int row = (lane >> 2) + 8 * t;
      const bool in = row < rows;
      const bf16* src = q + (p.row0 + (in ? row / G : 0)) * q_row + (long long)(p.kv_head * G + (in ? row % G : 0)) * D + pair;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        qf[t][k][0] = in ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
        qf[t][k][1] = in ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
      }
    }
    int lo[2][2], hi[2][2];
    float m[2][2], l[2][2], o[2][KB][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 8 * t + pair + e;
        const int pos = row < rows ? row_position(c, plan, p.w, p.row0 + row / G) : NO_POSITION;
        lo[t][e] = max(p.lo, c.window > 0 ? pos - c.window + 1 : 0);
        hi[t][e] = min(p.last, pos + 1);
        m[t][e] = -INFINITY; l[t][e] = 0.f;
      }
#pragma unroll
      for (int n = 0; n < KB; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.f;
    }
    for (int key0 = p.first; key0 < p.last; key0 += CHUNK) {
      asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory");
      __syncwarp();                    // the chunk is there for all lanes, and all are done with the one before
      request();                       // over that one
      const bf16 *Ks = stages + get * STAGE_ELEMENTS, *Vs = Ks + CHUNK * PITCH;
      get = get + 1 == STAGES ? 0 : get + 1;
      float s[2][2][4];                // of even and of odd steps along the head: two chains of products in place of one
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][0][e] = s[t][1][e] = 0.f;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        uint32_t a[4];
        ldmatrix_x4(a, Ks + (lane & 15) * PITCH + k * 16 + ((lane >> 4) << 3));
        mma(s[0][k & 1], a, qf[0][k][0], qf[0][k][1]);
        if (two) mma(s[1][k & 1], a, qf[1][k][0], qf[1][k][1]);
      }
      uint32_t b1[2][2], b2[2][2];     // weights as operands: [tile][keys 0 .. 7, 8 .. 15]
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (t && !two) break;
        // z[e + 2 h]: key key0 + 8 h + lane / 4, row pair + e
        float z[4], top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 8 * (e >> 1) + (lane >> 2);
          const bool sees = key >= lo[t][e & 1] && key < hi[t][e & 1];
          z[e] = sees ? (s[t][0][e] + s[t][1][e]) * c.scale_log2 : -INFINITY;
          top[e & 1] = fmaxf(top[e & 1], z[e]);
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
#pragma unroll
          for (int e = 0; e < 2; ++e) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], d));
        if (__any_sync(0xffffffffu, top[0] > m[t][0] || top[1] > m[t][1])) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float next = fmaxf(m[t][e], top[e]);
            f[e] = next == m[t][e] ? 1.f : fast_exp2(m[t][e] - next);
            m[t][e] = next;
            l[t][e] *= f[e];
          }
#pragma unroll
          for (int n = 0; n < KB; ++n) { o[t][n][0] *= f[0]; o[t][n][1] *= f[1]; o[t][n][2] *= f[0]; o[t][n][3] *= f[1]; }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 8 * (e >> 1) + (lane >> 2);
          const float ref = m[t][e & 1] == -INFINITY ? 0.f : m[t][e & 1];
          z[e] = key >= lo[t][e & 1] && key < hi[t][e & 1] ? fast_exp2(z[e] - ref) : 0.f;
          l[t][e & 1] += z[e];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t first, second;
          terms(z[2 * h], z[2 * h + 1], first, second);
          b1[t][h] = transposed(first);
          b2[t][h] = transposed(second);
        }
      }
#pragma unroll
      for (int n = 0; n < KB; ++n) {
        uint32_t a[4];      // columns 16 n .. 16 n + 15 by 16 keys
        ldmatrix_x4_trans(a, Vs + ((lane & 7) + ((lane >> 4) << 3)) * PITCH + n * 16 + (((lane >> 3) & 1) << 3));
        mma(o[0][n], a, b1[0][0], b1[0][1]);
        if (two) mma(o[1][n], a, b1[1][0], b1[1][1]);
        mma(o[0][n], a, b2[0][0], b2[0][1]);
        if (two) mma(o[1][n], a, b2[1][0], b2[1][1]);
      }
    }
    const int2 workers = walk.item_workers(c, p, worker);
    const bool sole = is_sole(p, workers);
    const long long slot = (long long)(p.item + worker) * c.rows;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], d);
        const int row = 8 * t + pair + e;
        if (row >= rows) continue;
        // columns 16 n + lane / 4 and the one eight on: eight lanes write 32 bytes (16 of bfloat16) together
        if (sole) {
          const float inv = l[t][e] > 0.f ? 1.f / l[t][e] : l[t][e] == 0.f ? 0.f : l[t][e];      // (NaN stays)
          bf16* dst = reinterpret_cast<bf16*>(c.out) + ((long long)(p.row0 + row / G) * c.heads + p.kv_head * G + row % G) * D + (lane >> 2);
#pragma unroll
          for (int n = 0; n < KB; ++n) {
            dst[n * 16] = __float2bfloat16_rn(o[t][n][e] * inv);
            dst[n * 16 + 8] = __float2bfloat16_rn(o[t][n][2 + e] * inv);
          }
        } else {
          if (lane < 4) c.part_ml[slot + row] = make_float2(m[t][e], l[t][e]);
          float* dst = c.part_o + (slot + row) * D + (lane >> 2);
#pragma unroll
          for (int n = 0; n < KB; ++n) { dst[n * 16] = o[t][n][e]; dst[n * 16 + 8] = o[t][n][2 + e]; }
        }
      }
    }
    if (lane == 0) c.pieces[p.item] = workers;
  }
  asm volatile("cp.async.wait_all;\n" ::: "memory");
  if (beside && (blockIdx.x == 0 || (int)blockIdx.x * WARPS < limit)) ifb_pdl_wait();      // (one CTA that waits is enough for the grid)
}

static inline Call call(int n_tokens, int n_req, int n_groups, int kv_heads, int group) {
  Call c = {};
  c.which = NARROW;
  c.n_tokens = n_tokens; c.n_req = n_req; c.n_groups = n_groups;
  c.kv_heads = kv_heads; c.heads = kv_heads * group;
  c.tokens = group <= NARROW_ROWS ? NARROW_ROWS / group : 1; c.unit = UNIT; c.rows = NARROW_ROWS; c.align = 1;
  c.workers = ifb_sm_count() * CTAS_PER_SM * WARPS;
  c.cost = 1;
  c.extra = 1;
  return c;
}
static int run(const Call& c, const Call& other, const bf16* q, long long q_row, const bf16* pages, bool beside, cudaStream_t stream) {
  const size_t smem = plan_bytes(c.n_req + c.n_groups) + WARPS * WARP_BYTES;
  IFB_ALLOW_SMEM(shared_narrow_kernel, smem);
  return ifb_launch(shared_narrow_kernel, dim3(c.workers / WARPS), dim3(WARPS * 32), smem, stream, c, other, q, q_row, pages, ifb_sm_count(), beside ? 1 : 0);
}

}  // namespace narrow
