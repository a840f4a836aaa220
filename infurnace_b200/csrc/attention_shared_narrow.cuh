// Attention over shared pages for narrow owners (at most 16 score rows) of bfloat16 heads of HEAD_DIM: a request's decoded token over its own keys, and
// a few requests' over the keys they share.  attention_shared.cuh says how the work is cut and joined.
//
// The work is the reading of keys and values.  Every warp is a worker of its own: it walks over its pieces in chunks of 16 keys, which it has brought to its
// part of shared memory two chunks ahead and across the ends of pieces, so that no warp waits for another and the 2 x 4 warps of an SM have 130 KB
// on their way.  By TMA where heads are whole rows of 64 columns and pages whole chunks (a box of 64 columns by 16 keys in the 128-byte swizzle, a barrier
// for each stage); else by asynchronous copies of 16 bytes into padded rows.  (The copies' 160 instructions a chunk were a quarter of what bound the
// kernel when it had no other form: a chunk took a warp 630 instructions and 1.6 us.)
//
// Products are mma.sync of bfloat16 with the keys, and then the columns of the values, on the side of 16 and the score rows on the side of eight, one or two
// times: S^T = K Q^T, O^T += V^T P^T.  (With the rows on the side of 16 a chunk of four rows takes 48 products in place of 24.)  In both a thread
// has rows 2 (lane mod 4) and the next, so that the factors of a row's maximum need no exchange; weights cross over from accumulator to operand by movmatrix.
// A row's weights are formed in float32 against its running maximum and enter the second product as two bfloat16 terms (16 bits of a weight); sums
// are float32.  Values of a chunk that lie outside of the piece's keys are made zeros before they meet weights of zero; rows that come out infinite or NaN by values
// which only others of the piece see are worked out anew by the join.
#pragma once
#include "attention_shared.cuh"
#include "tc_ops.cuh"
#include <type_traits>

using namespace shared_attention;

namespace narrow {

typedef __nv_bfloat16 bf16;
constexpr int WARPS = 4;
constexpr int CHUNK = 16, UNIT = 32;
static_assert(UNIT == 1 << 5 && CHUNK == 1 << 4, "unit_log, align_log");
constexpr int STAGES = 3;
constexpr int KB = D / 16;
constexpr bool TMA_HEADS = D % 64 == 0;               // whole rows of 64 columns
constexpr int HALVES = TMA_HEADS ? D / 64 : 1;
constexpr int PITCH = D + 8;                          // padded rows: 16 bytes more keep ldmatrix free of conflicts
constexpr int RING = 4;                               // pieces that the copies are ahead of the products, at most STAGES
template <bool TMA> struct Room {
  static constexpr int KEYS = TMA ? CHUNK * D * 2 : CHUNK * PITCH * 2;      // bytes of a chunk's keys
  static constexpr int STAGE = 2 * KEYS, WARP = STAGES * STAGE;
  static constexpr int CTAS = WARPS * WARP <= 108 * 1024 ? 2 : 1;           // of an SM
};
// A piece as the copies' walk leaves it to the products.
struct Entry {
  Owner w;
  int row0, tokens, kv_head, item, first, last, lo;
  int2 workers;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(void* dst, const void* src, bool valid) {
  const int size = valid ? 16 : 0;      // 0: zeros, src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(size) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
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

// A thread's part of two tiles of eight rows.
struct Rows {
  uint32_t q[2][KB][2];      // rows lane / 4 (+ 8)
  int lo[2][2], hi[2][2];    // the keys that its rows see
  float m[2][2], l[2][2], o[2][KB][4];
};

// `beside`: the wide owners' kernel is the one before this in the stream; all its CTAs have waited for their own predecessor before this begins, and
// nothing that it writes is read here.  So this kernel waits for it at its end instead of at its start: who waits for this one has waited for both.
template <bool TMA>
__global__ void __launch_bounds__(WARPS * 32, Room<TMA>::CTAS)
shared_narrow_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, PageRows mrows, const __grid_constant__ Call c,
                     const __grid_constant__ Call other, const bf16* q, long long q_row, const bf16* pages, int sms, int beside) {
  extern __shared__ __align__(1024) unsigned char narrow_smem[];
  __shared__ Entry ring[WARPS][RING];
  __shared__ uint64_t full[WARPS][STAGES];
  __shared__ int abort_words[WARPS];
  constexpr int KEYS = Room<TMA>::KEYS, STAGE = Room<TMA>::STAGE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* base = narrow_smem + ((1024u - (smem_u32(narrow_smem) & 1023u)) & 1023u);
  unsigned char* stages = base + (size_t)warp * Room<TMA>::WARP;
  const Plan plan = plan_at(base + WARPS * Room<TMA>::WARP, c.n_groups + c.n_req);
  volatile int* abort_flag = &abort_words[warp];
  if (TMA && threadIdx.x < 2) tc_prefetch_map(threadIdx.x ? &v_map : &k_map);
  if (lane == 0) {
    abort_words[warp] = 0;
    if (TMA) {
      for (int st = 0; st < STAGES; ++st) tc_mbar_init(&full[warp][st], 1);
      asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    }
  }
  if (!beside) ifb_pdl_wait();
  ifb_pdl_trigger();
  make_plan(c, other, plan);
  const int G = c.heads / c.kv_heads;
  // the SMs that the wide owners' kernel leaves
  const int mine = sms - wide_sms(sms, plan.sums[63] * other.cost, plan.starts[c.n_groups + c.n_req] * c.cost);
  const int worker = blockIdx.x * WARPS + warp, limit = min(c.workers, mine * Room<TMA>::CTAS * WARPS);
  const long long values = (long long)c.kv_heads * c.page_size * D;

  // The copies' walk and the products' chunks, two steps apart.
  Walk walk;
  walk.begin(c, plan, worker, limit);
  Piece ap;
  ap.last = 0;
  int akey = 0, page0 = 0, id = 0;       // the next key to bring; the piece's pages page0 .. page0 + 31, one a lane
  int pushed = 0, requested = 0;
  bool more = true;
  Rows x;
  int key0 = 0, last = 0, lo = 0, pieces = 0;      // of the products' piece
  int rows = 0;
  const int pair = (lane & 3) << 1;      // the thread's rows of a tile of eight: pair, pair + 1
  // parts of an address: rows of 16 keys and halves of 16 columns for the keys, the other way round for the values; swizzled: 16 bytes j of row r lie at j ^ (r mod 8)
  const int krow = lane & 15, kcol = lane >> 4, vrow = (lane & 7) + ((lane >> 4) << 3), vcol = (lane >> 3) & 1;
  const uint32_t k_at = TMA ? krow * 128 + ((kcol ^ (krow & 7)) << 4) : krow * PITCH * 2 + kcol * 16;
  const uint32_t v_at = (TMA ? vrow * 128 + ((vcol ^ (vrow & 7)) << 4) : vrow * PITCH * 2 + vcol * 16) + KEYS;
  auto column = [](uint32_t at, int k) { return TMA ? (at ^ ((k & 3) << 5)) + (k >> 2) * (CHUNK * 128) : at + k * 32; };      // of the 16 columns from 16 k on
  bool ok = true;
  for (int step = 0;; ++step) {
    __syncwarp();                        // all lanes are done with the stage that is filled next
    if (more && akey >= ap.last) {
      more = walk.next(c, plan, ap);
      if (more) {
        akey = ap.first;
        const int2 workers = walk.item_workers(c, ap, worker);
        if (lane == 0) ring[warp][pushed % RING] = Entry{ap.w, ap.row0, ap.tokens, ap.kv_head, ap.item, ap.first, ap.last, ap.lo, workers};
        ++pushed;
        page0 = -32;
      }
    }
    if (more) {                          // the next chunk
      unsigned char* st = stages + step % STAGES * STAGE;
      if (TMA) {                         // it is within a page
        const int page = akey / c.page_size;
        if (page >= page0 + 32 || page0 < 0) {
          page0 = page;
          const int first = (page0 + lane) * c.page_size;      // of the lane's page
          id = first < ap.last ? c.block_tables[ap.w.table(first) * c.bt_stride + page0 + lane] : -1;
        }
        const int mine_id = __shfl_sync(0xffffffffu, id, page - page0);
        const bool there = mine_id >= 0 && mine_id < c.num_pages;
        if (!there && lane == 0) atomicExch(c.err, IFB_DEV_ERR_SHARED_PAGE);
        const int y = there ? mine_id * mrows.page + ap.kv_head * c.page_size + akey - page * c.page_size : mrows.total;      // (beyond the pool: zeros)
        uint64_t* bar = &full[warp][step % STAGES];
        if (lane == 0) tc_mbar_expect_tx(bar, STAGE);
        __syncwarp();
        if (lane < 2 * HALVES) {
          const int half = lane >> 1;
          tc_tma_2d(st + (lane & 1) * KEYS + half * (CHUNK * 128), lane & 1 ? &v_map : &k_map, bar, half * 64, y);
        }
      } else {
        const int key = akey + (lane & 15), page = key / c.page_size;      // lanes 16 .. 31 as 0 .. 15
        if (__shfl_sync(0xffffffffu, page, 15) >= page0 + 32 || page0 < 0) {
          page0 = __shfl_sync(0xffffffffu, page, 0);
          const int first = (page0 + lane) * c.page_size;
          id = first < ap.last ? c.block_tables[ap.w.table(first) * c.bt_stride + page0 + lane] : -1;
        }
        const int mine_id = __shfl_sync(0xffffffffu, id, page - page0 & 31);
        long long at = -1;
        if (key >= ap.lo && key < ap.last) {
          if (mine_id < 0 || mine_id >= c.num_pages) atomicExch(c.err, IFB_DEV_ERR_SHARED_PAGE);
          else at = mine_id * c.page_stride + ((long long)ap.kv_head * c.page_size + key - page * c.page_size) * D;
        }
        constexpr int PARTS = D / 8;      // 16-byte parts of a row
#pragma unroll
        for (int i = 0; i < (CHUNK * PARTS + 31) / 32; ++i) {
          const int e = i * 32 + lane, row = e / PARTS, col = e % PARTS * 8;
          const long long from = __shfl_sync(0xffffffffu, at, row & 15);
          if (e < CHUNK * PARTS) {
            const bf16* src = pages + (from < 0 ? 0 : from + col);
            copy16(st + (row * PITCH + col) * 2, src, from >= 0);
            copy16(st + KEYS + (row * PITCH + col) * 2, src + (from < 0 ? 0 : values), from >= 0);
          }
        }
      }
      akey += CHUNK;
      ++requested;
    }
    if (!TMA) asm volatile("cp.async.commit_group;\n" ::: "memory");
    const int done = step - (STAGES - 1);      // the products' chunk
    if (done < 0) continue;
    if (done >= requested) break;

    if (key0 >= last) {                  // the next piece
      __syncwarp();
      const Entry& p = ring[warp][pieces % RING];
      key0 = p.first; last = p.last; lo = p.lo;
      rows = p.tokens * G;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (t && rows <= 8) break;
        const int row = (lane >> 2) + 8 * t;
        const bool in = row < rows;
        const bf16* src = q + (p.row0 + (in ? row / G : 0)) * q_row + (long long)(p.kv_head * G + (in ? row % G : 0)) * D + pair;
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          x.q[t][k][0] = in ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
          x.q[t][k][1] = in ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * t + pair + e;
          const int pos = r < rows ? row_position(c, plan, p.w, p.row0 + r / G) : NO_POSITION;
          x.lo[t][e] = max(lo, c.window > 0 ? pos - c.window + 1 : 0);
          x.hi[t][e] = min(last, pos + 1);
          x.m[t][e] = -INFINITY; x.l[t][e] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < KB; ++n) x.o[t][n][0] = x.o[t][n][1] = x.o[t][n][2] = x.o[t][n][3] = 0.f;
      }
    }
    const uint32_t st = smem_u32(stages) + done % STAGES * STAGE;
    if (TMA) {
      ok = __all_sync(0xffffffffu, tc_mbar_wait(&full[warp][done % STAGES], done / STAGES & 1, abort_flag, c.err, 80)) != 0;
      if (!ok) break;
      if (key0 < lo || key0 + CHUNK > last) {      // values that no row sees: zeros
        for (int e = lane; e < CHUNK * HALVES * 8; e += 32) {
          const int row = e / (HALVES * 8), key = key0 + row;
          if (key < lo || key >= last)
            *reinterpret_cast<uint4*>(stages + done % STAGES * STAGE + KEYS + (e / 8 % HALVES) * (CHUNK * 128) + row * 128 + e % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");      // (a copy writes there again)
        __syncwarp();
      }
    } else {
      asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
    }
    auto products = [&](auto tiles) {      // with one tile of rows or with both
      constexpr int T = decltype(tiles)::value;
      float s[T][2][4];                // of even and of odd steps along the head: two chains of products in place of one
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][0][e] = s[t][1][e] = 0.f;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        uint32_t a[4];
        ldmatrix_x4(a, st + column(k_at, k));
#pragma unroll
        for (int t = 0; t < T; ++t) mma(s[t][k & 1], a, x.q[t][k][0], x.q[t][k][1]);
      }
      uint32_t b1[T][2], b2[T][2];      // weights as operands: keys 0 .. 7, 8 .. 15
#pragma unroll
      for (int t = 0; t < T; ++t) {
        // z[e + 2 h]: key key0 + 8 h + lane / 4, row pair + e
        float z[4], top[2];
        bool sees[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 8 * (e >> 1) + (lane >> 2);
          sees[e] = key >= x.lo[t][e & 1] && key < x.hi[t][e & 1];
          z[e] = sees[e] ? (s[t][0][e] + s[t][1][e]) * c.scale_log2 : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) top[e] = fmaxf(z[e], z[2 + e]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
#pragma unroll
          for (int e = 0; e < 2; ++e) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], d));
        if (__any_sync(0xffffffffu, top[0] > x.m[t][0] || top[1] > x.m[t][1])) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float next = fmaxf(x.m[t][e], top[e]);
            f[e] = next == x.m[t][e] ? 1.f : fast_exp2(x.m[t][e] - next);
            x.m[t][e] = next;
            x.l[t][e] *= f[e];
          }
#pragma unroll
          for (int n = 0; n < KB; ++n) { x.o[t][n][0] *= f[0]; x.o[t][n][1] *= f[1]; x.o[t][n][2] *= f[0]; x.o[t][n][3] *= f[1]; }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float ref = x.m[t][e & 1] == -INFINITY ? 0.f : x.m[t][e & 1];
          z[e] = sees[e] ? fast_exp2(z[e] - ref) : 0.f;
          x.l[t][e & 1] += z[e];
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
        ldmatrix_x4_trans(a, st + column(v_at, n));
#pragma unroll
        for (int t = 0; t < T; ++t) mma(x.o[t][n], a, b1[t][0], b1[t][1]);
#pragma unroll
        for (int t = 0; t < T; ++t) mma(x.o[t][n], a, b2[t][0], b2[t][1]);
      }
    };
    if (rows <= 8) products(std::integral_constant<int, 1>());
    else products(std::integral_constant<int, 2>());
    key0 += CHUNK;
    if (key0 < last) continue;

    // the piece's end
    const Entry& p = ring[warp][pieces % RING];
    Piece as;
    as.w = p.w;
    const bool sole = is_sole(as, p.workers);
    const long long slot = (long long)(p.item + worker) * c.rows;
    bool anew = false;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (t && rows <= 8) break;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = x.l[t][e];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        const int row = 8 * t + pair + e;
        if (row >= rows) continue;
        // columns 16 n + lane / 4 and the one eight on: eight lanes write 32 bytes (16 of bfloat16) together
        if (sole) {
          const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;      // (NaN stays)
          float finite = 0.f;      // NaN: not all of the thread's numbers are
#pragma unroll
          for (int n = 0; n < KB; ++n) finite = fmaf(x.o[t][n][e], 0.f, fmaf(x.o[t][n][2 + e], 0.f, finite));
          anew |= finite != finite;
          bf16* dst = reinterpret_cast<bf16*>(c.out) + ((long long)(p.row0 + row / G) * c.heads + p.kv_head * G + row % G) * D + (lane >> 2);
#pragma unroll
          for (int n = 0; n < KB; ++n) {
            dst[n * 16] = __float2bfloat16_rn(x.o[t][n][e] * inv);
            dst[n * 16 + 8] = __float2bfloat16_rn(x.o[t][n][2 + e] * inv);
          }
        } else {
          if (lane < 4) c.part_ml[slot + row] = make_float2(x.m[t][e], l);
          float* dst = c.part_o + (slot + row) * D + (lane >> 2);
#pragma unroll
          for (int n = 0; n < KB; ++n) { dst[n * 16] = x.o[t][n][e]; dst[n * 16 + 8] = x.o[t][n][2 + e]; }
        }
      }
    }
    anew = __any_sync(0xffffffffu, anew);
    if (lane == 0) c.pieces[p.item] = make_int2(p.workers.x, p.workers.y | (anew ? ANEW : 0));
    ++pieces;
  }
  if (TMA && !ok) {                      // a wait gave up: let copies in flight land
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  if (!TMA) asm volatile("cp.async.wait_all;\n" ::: "memory");
  write_parts(other, c, plan);
  if (beside && (blockIdx.x == 0 || (int)blockIdx.x * WARPS < limit)) ifb_pdl_wait();      // (one CTA that waits is enough for the grid)
}

// Whether chunks come by TMA: whole rows of 64 columns, pages that are whole chunks, the pool a matrix of rows.
static inline bool by_tma(int page_size, long long page_stride, long long num_pages) {
  return TMA_HEADS && page_size % CHUNK == 0 && page_stride % D == 0 && num_pages * (page_stride / D) < 0x7fffffffLL;
}
static inline Call call(bool tma, Class which, int n_tokens, int n_req, int n_groups, int kv_heads, int group) {
  Call c = {};
  c.which = which;
  c.n_tokens = n_tokens; c.n_req = n_req; c.n_groups = n_groups;
  c.kv_heads = kv_heads; c.heads = kv_heads * group;
  c.tokens = group <= NARROW_ROWS ? NARROW_ROWS / group : 1; c.rows = NARROW_ROWS; c.unit_log = 5; c.align_log = tma ? 4 : 0;
  c.workers = ifb_sm_count() * (tma ? Room<true>::CTAS : Room<false>::CTAS) * WARPS;
  c.cost = 1;
  c.extra = 1;
  return c;
}
template <bool TMA>
static int launch(const CUtensorMap& k_map, const CUtensorMap& v_map, PageRows rows, const Call& c, const Call& other, const bf16* q, long long q_row,
                  const bf16* pages, bool beside, cudaStream_t stream) {
  const size_t smem = 1024 + plan_bytes(c.n_req + c.n_groups) + WARPS * Room<TMA>::WARP;
  if (smem > MOST_SMEM) return IFB_ERR_SIZE;
  IFB_ALLOW_SMEM(shared_narrow_kernel<TMA>, smem);
  return ifb_launch(shared_narrow_kernel<TMA>, dim3(c.workers / WARPS), dim3(WARPS * 32), smem, stream, k_map, v_map, rows, c, other, q, q_row, pages,
                    ifb_sm_count(), beside ? 1 : 0);
}
static int run(bool tma, const Call& c, const Call& other, const bf16* q, long long q_row, const bf16* pages, bool beside, cudaStream_t stream) {
  CUtensorMap k_map = {}, v_map = {};
  if (!tma) return launch<false>(k_map, v_map, PageRows{}, c, other, q, q_row, pages, beside, stream);
  const long long page_rows = c.page_stride / D, all = (c.num_pages - 1) * page_rows + (long long)c.kv_heads * c.page_size;
  const unsigned long long dims[2] = {(unsigned long long)D, (unsigned long long)all}, strides[1] = {(unsigned long long)D * 2};
  const unsigned box[2] = {64, CHUNK};
  if (ifb_tensor_map_bf16(&k_map, pages, 2, dims, strides, box)) return IFB_ERR_ARG;
  if (ifb_tensor_map_bf16(&v_map, pages + (long long)c.kv_heads * c.page_size * D, 2, dims, strides, box)) return IFB_ERR_ARG;
  return launch<TMA_HEADS>(k_map, v_map, PageRows{(int)page_rows, (int)all}, c, other, q, q_row, pages, beside, stream);
}

}  // namespace narrow
