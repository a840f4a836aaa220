// Attention over shared pages for narrow owners (at most 16 score rows) of bfloat16 heads of HEAD_DIM: a request's decoded token over its own keys, and
// a few requests' over the keys they share.  attention_shared.cuh says how the work is cut and joined.
//
// The work is the reading of keys and values.  Every warp is a worker of its own: it walks over its pieces in chunks of 16 keys, which it brings to its part
// of shared memory by asynchronous copies of 16 bytes (any page size), two chunks ahead and across the ends of pieces, so that no warp waits for
// another and 2 x 4 warps of an SM have 130 KB on their way.  The 16 score rows meet 16 keys in mma.sync products of bfloat16; a row's weights
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
  const int mine = sms - wide_sms(sms, plan.sums[31] * other.cost, plan.starts[c.n_groups + c.n_req] * c.cost);
  const int worker = blockIdx.x * WARPS + warp, limit = min(c.workers, mine * CTAS_PER_SM * WARPS);
  const long long values = (long long)c.kv_heads * c.page_size * D;

  // ---- the copies' walk, ahead of the products'
  Walk ahead;
  ahead.begin(c, plan, worker, limit);
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
  Walk walk;
  walk.begin(c, plan, worker, limit);
  Piece p;
  int get = 0;
  const int rowA = lane >> 2, rowB = rowA + 8;
  while (walk.next(c, plan, p)) {
    const int rows = p.tokens * G;
    uint32_t qf[KB][4];
    {
      const bool a = rowA < rows, b = rowB < rows;
      const bf16* qa = q + (p.row0 + (a ? rowA / G : 0)) * q_row + (long long)(p.kv_head * G + (a ? rowA % G : 0)) * D + (lane & 3) * 2;
      const bf16* qb = q + (p.row0 + (b ? rowB / G : 0)) * q_row + (long long)(p.kv_head * G + (b ? rowB % G : 0)) * D + (lane & 3) * 2;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        qf[k][0] = a ? *reinterpret_cast<const uint32_t*>(qa + k * 16) : 0u;
        qf[k][1] = b ? *reinterpret_cast<const uint32_t*>(qb + k * 16) : 0u;
        qf[k][2] = a ? *reinterpret_cast<const uint32_t*>(qa + k * 16 + 8) : 0u;
        qf[k][3] = b ? *reinterpret_cast<const uint32_t*>(qb + k * 16 + 8) : 0u;
      }
    }
    int lo[2], hi[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = e ? rowB : rowA;
      const int pos = row < rows ? row_position(c, plan, p.w, p.row0 + row / G) : NO_POSITION;
      lo[e] = max(p.lo, c.window > 0 ? pos - c.window + 1 : 0);
      hi[e] = min(p.last, pos + 1);
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    for (int key0 = p.first; key0 < p.last; key0 += CHUNK) {
      asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory");
      __syncwarp();                    // the chunk is there for all lanes, and all are done with the one before
      request();                       // over that one
      const bf16 *Ks = stages + get * STAGE_ELEMENTS, *Vs = Ks + CHUNK * PITCH;
      get = get + 1 == STAGES ? 0 : get + 1;
      float s[2][4], odd[2][4];      // of even and of odd steps along the head: two chains of products in place of one
#pragma unroll
      for (int n = 0; n < 2; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = odd[n][0] = odd[n][1] = odd[n][2] = odd[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        uint32_t b[4];
        ldmatrix_x4(b, Ks + ((lane & 7) + ((lane >> 4) << 3)) * PITCH + k * 16 + (((lane >> 3) & 1) << 3));
        mma(k & 1 ? odd[0] : s[0], qf[k], b[0], b[1]);
        mma(k & 1 ? odd[1] : s[1], qf[k], b[2], b[3]);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] += odd[n][e];
      // rows A and B of the scores, keys key0 + 8 n + 2 (lane & 3) + j
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 8 * n + ((lane & 3) << 1) + (e & 1), r = e >> 1;
          const bool sees = key >= lo[r] && key < hi[r];
          s[n][e] = sees ? s[n][e] * c.scale_log2 : -INFINITY;
          top[r] = fmaxf(top[r], s[n][e]);
        }
      float ref[2];
      bool grew = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
        grew |= top[r] > m[r];
      }
      if (__any_sync(0xffffffffu, grew)) {
        float f[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float next = fmaxf(m[r], top[r]);
          f[r] = next == m[r] ? 1.f : fast_exp2(m[r] - next);
          m[r] = next;
          l[r] *= f[r];
        }
#pragma unroll
        for (int n = 0; n < D / 8; ++n) { o[n][0] *= f[0]; o[n][1] *= f[0]; o[n][2] *= f[1]; o[n][3] *= f[1]; }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) ref[r] = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 8 * n + ((lane & 3) << 1) + (e & 1), r = e >> 1;
          s[n][e] = key >= lo[r] && key < hi[r] ? fast_exp2(s[n][e] - ref[r]) : 0.f;
          l[r] += s[n][e];
        }
      uint32_t a1[4], a2[4];
      terms(s[0][0], s[0][1], a1[0], a2[0]);
      terms(s[0][2], s[0][3], a1[1], a2[1]);
      terms(s[1][0], s[1][1], a1[2], a2[2]);
      terms(s[1][2], s[1][3], a1[3], a2[3]);
#pragma unroll
      for (int n = 0; n < KB; ++n) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, Vs + ((lane & 7) + (((lane >> 3) & 1) << 3)) * PITCH + n * 16 + ((lane >> 4) << 3));
        mma(o[2 * n], a1, b[0], b[1]);
        mma(o[2 * n + 1], a1, b[2], b[3]);
        mma(o[2 * n], a2, b[0], b[1]);
        mma(o[2 * n + 1], a2, b[2], b[3]);
      }
    }
    const int2 workers = walk.item_workers(c, p);
    const bool sole = is_sole(p, workers);
    const long long slot = (long long)(p.item + worker) * c.rows;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      const int row = r ? rowB : rowA;
      if (row < rows && sole) {
        const float inv = l[r] > 0.f ? 1.f / l[r] : l[r] == 0.f ? 0.f : l[r];      // (NaN stays)
        bf16* dst = reinterpret_cast<bf16*>(c.out) + ((long long)(p.row0 + row / G) * c.heads + p.kv_head * G + row % G) * D + ((lane & 3) << 1);
#pragma unroll
        for (int n = 0; n < D / 8; ++n) *reinterpret_cast<__nv_bfloat162*>(dst + n * 8) = __floats2bfloat162_rn(o[n][2 * r] * inv, o[n][2 * r + 1] * inv);
      } else if (row < rows) {
        if ((lane & 3) == 0) c.part_ml[slot + row] = make_float2(m[r], l[r]);
        float* dst = c.part_o + (slot + row) * D + ((lane & 3) << 1);
#pragma unroll
        for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
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
