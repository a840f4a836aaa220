// Attention over shared pages on the fifth-generation tensor cores: wide owners of bfloat16 heads of HEAD_DIM, a multiple of 16 up to 128, in
// pages of 16, 32 or 64.  attention_shared.cuh says how the work is cut and joined.
//
// A tile is 128 score rows (query tokens times the heads of a key head's group: row = token * G + head-in-group), a unit 128 keys.  Decoded tokens
// of all requests of a group fill tiles together over the keys that they share; over its own keys a request of more than sixteen score rows has tiles to itself
// (those of fewer are narrow, and are worked on by warps beside this kernel).
//
// As in attention_tc.cu a CTA is a pipeline: warp 0 brings queries and keys by TMA, warp 3 values, warps 1 and 2 issue the products of two streams (stream x
// takes half x of every 128 keys), warps 4-7 and 8-11 do their softmax, a thread a row; scores, weights (over the scores' columns) and the sums stay in
// tensor memory.  Here the walk goes over pieces, which follow one another without a pause for the producers; a piece ends with its sums, not divided, in
// float32 to the room, and maximum and denominator beside them.  A weight is the sum of two bfloat16 numbers (16 of its bits).
//
// What no row sees may be anything: keys outside of a piece's are masked as scores; their values, which the product would multiply by a weight of zero, are
// overwritten with zeros in shared memory by the warp that issues it.  (A value that some rows of the tile see and others do not is in the product of these with
// weight zero: rows that come out infinite or NaN are worked out anew by the join.)
//
// What bounds it: a half's chain, 2,500 cycles, of which a softmax warp works 1,950 and waits for scores 300 and for the product before 240, two warps to a
// scheduler; tensor cores are busy 57% of the time and issue slots 41%.  Eight times 230 queries (32 heads of 128) to 6,000 shared keys take 296 us, 630 TFLOP/s not
// counting the second terms, or 940 with them, where the power limit lowers clocks to 1.2 to 1.5 GHz.
#pragma once
#include "tc_ops.cuh"
#include "attention_shared.cuh"

using namespace shared_attention;
typedef __nv_bfloat16 bf16;

constexpr int DH = (D + 63) / 64;                // swizzle rows of 64 columns that a row has
constexpr int DN = DH * 64;                      // columns of the output accumulator
constexpr int ROWS = 128, UNIT = 128, SUB = 64;
static_assert(UNIT == 1 << 7, "unit_log");
constexpr int THREADS = 384;
constexpr int HALF_BYTES = 128 * 128;            // [128 rows][64 columns] in the 128-byte swizzle
constexpr int TILE_BYTES = DH * HALF_BYTES;
constexpr int TILES_BYTES = 5 * TILE_BYTES + 1024;      // Q, two stages of K and of V, alignment
constexpr int STAGES_BYTES = 8 * 32 * 36 * 4;     // where sums turn from rows of a thread to rows of eight lanes
constexpr int COL_S = 0, COL_O = 128, COLS_PER_STREAM = 256, TMEM_COLS = 512;
constexpr uint64_t DESC = (1ull << 46) | (2ull << 61) | ((uint64_t)(1024 >> 4) << 32);      // 128-byte swizzle, groups of 8 rows 1,024 bytes apart
__device__ __forceinline__ uint64_t desc_k_major(uint32_t a) { return (uint64_t)((a >> 4) & 0x3FFF) | (1ull << 16) | DESC; }
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t a) { return (uint64_t)((a >> 4) & 0x3FFF) | ((uint64_t)(HALF_BYTES >> 4) << 16) | DESC; }
constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 4) << 24);      // float32 sums of bfloat16, M = 128
constexpr uint32_t IDESC_S = IDESC | ((uint32_t)(SUB >> 3) << 17);
constexpr uint32_t IDESC_PV = IDESC | ((uint32_t)(DN >> 3) << 17) | (1u << 16);

// Two float32 numbers in an instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair_of(float a, float b) { f32x2 r; asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void numbers_of(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
// Two weights as bfloat16 pairs: their upper 16 bits, and the rounding of the rest.  (One term alone, 8 bits of a weight, made outputs ten times less exact and
// the kernel 13% faster: 275 us in place of 316 for the questions below.)
__device__ __forceinline__ void weight_terms(f32x2 e, uint32_t& first, uint32_t& second) {
  float e0, e1, r0, r1;
  numbers_of(e, e0, e1);
  const uint32_t u0 = __float_as_uint(e0), u1 = __float_as_uint(e1);
  asm("prmt.b32 %0, %1, %2, 0x7632;\n" : "=r"(first) : "r"(u0), "r"(u1));
  numbers_of(add2(e, pair_of(__uint_as_float((u0 & 0xffff0000u) | 0x80000000u), __uint_as_float((u1 & 0xffff0000u) | 0x80000000u))), r0, r1);
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(second) : "f"(r1), "f"(r0));
}

struct Bars {
  uint64_t q_full, q_empty, o_free, k_full[2], v_full[2], k_empty[2][2], v_empty[2][2], s_full[2][2], p_ready[2][2], o_done[2];
};

__global__ void __launch_bounds__(THREADS, 1)
shared_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                 PageRows mrows, const __grid_constant__ Call c, const __grid_constant__ Call other, int parts) {
  extern __shared__ unsigned char tc_smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ float merge_m[2][2][ROWS], merge_l[2][2][ROWS];       // [piece parity][stream][row]
  volatile int* abort_flag = &abort_word;
  int* err = c.err;
  const uint32_t raw = tc_smem_u32(tc_smem_raw);
  unsigned char* smem = tc_smem_raw + (((raw + 1023u) & ~1023u) - raw);
  unsigned char *Qs = smem, *Ks = smem + TILE_BYTES, *Vs = smem + 3 * TILE_BYTES;
  const Plan plan = plan_at(smem + 5 * TILE_BYTES + STAGES_BYTES, c.n_groups + c.n_req);
  float* stages = reinterpret_cast<float*>(smem + 5 * TILE_BYTES);      // [8 warps][32][36]
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int G = c.heads / c.kv_heads;

  if (threadIdx.x < 3) tc_prefetch_map(threadIdx.x == 0 ? &q_map : threadIdx.x == 1 ? &k_map : &v_map);
  if (c.tokens * G < ROWS) {      // rows of the tile that no query fills: zeros, once
    for (int i = threadIdx.x; i < TILE_BYTES / 16; i += THREADS) reinterpret_cast<uint4*>(Qs)[i] = make_uint4(0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  if (threadIdx.x == 0) {
    tc_mbar_init(&bars.q_full, 1);
    tc_mbar_init(&bars.q_empty, 2);
    tc_mbar_init(&bars.o_free, 256);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      tc_mbar_init(&bars.k_full[i], 1); tc_mbar_init(&bars.v_full[i], 1);
      tc_mbar_init(&bars.o_done[i], 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        tc_mbar_init(&bars.k_empty[i][h], 1); tc_mbar_init(&bars.v_empty[i][h], 1);
        tc_mbar_init(&bars.s_full[i][h], 1); tc_mbar_init(&bars.p_ready[i][h], 128);
      }
    }
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc_smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  ifb_pdl_wait();
  ifb_pdl_trigger();
  make_plan(c, other, plan);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  Walk walk;
  walk.begin(c, plan, blockIdx.x, wide_sms(c.workers, plan.starts[c.n_groups + c.n_req] * c.cost, plan.sums[63] * other.cost));
  Piece p;
  if (parts) write_parts(c, other, plan);

  if (warp == 0 || warp == 3) {
    // ---------------- producers: queries and keys, and values
    const int kv = warp == 3;
    const int ps_shift = __ffs(c.page_size) - 1, ppt = UNIT >> ps_shift, n_ops = ppt * DH;      // boxes of a tile: at most 16
    bool ok = true;
    int jt = 0, ic = 0;                                      // tiles and pieces so far
    while (ok && walk.next(c, plan, p)) {
      if (!kv) {
        if (ic > 0) ok = tc_mbar_wait(&bars.q_empty, (ic - 1) & 1, abort_flag, err, 60);
        if (!ok) break;
        if (lane == 0) {
          tc_mbar_expect_tx(&bars.q_full, (uint32_t)(DH * c.tokens * G * 128));
#pragma unroll
          for (int hf = 0; hf < DH; ++hf) tc_tma_3d(Qs + hf * HALF_BYTES, &q_map, &bars.q_full, hf * 64, p.kv_head * G, p.row0);
        }
        __syncwarp();
      }
      const int n_tiles = (p.last - p.first + UNIT - 1) / UNIT;
      for (int j = 0; j < n_tiles && ok; ++j, ++jt) {
        const int st = jt & 1;
        uint64_t* full = kv ? &bars.v_full[st] : &bars.k_full[st];
        // where the tile's pages are, asked for before the stage is waited for
        const int pg = lane / DH, half = lane % DH, key0 = p.first + j * UNIT + pg * c.page_size;
        int y = mrows.total;                                 // beyond the pool: zeros
        if (lane < n_ops && key0 < p.last && key0 + c.page_size > p.lo) {
          const int id = c.block_tables[p.w.table(key0) * c.bt_stride + (key0 >> ps_shift)];
          if (id >= 0 && id < c.num_pages) y = id * mrows.page + p.kv_head * c.page_size;
          else atomicExch(err, IFB_DEV_ERR_SHARED_PAGE);
        }
        if (jt >= 2) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if (ok) ok = tc_mbar_wait(kv ? &bars.v_empty[x][st] : &bars.k_empty[x][st], ((jt >> 1) - 1) & 1, abort_flag, err, 61);
        }
        if (!ok) break;
        if (lane == 0) tc_mbar_expect_tx(full, TILE_BYTES);
        __syncwarp();
        if (lane < n_ops)
          tc_tma_2d((kv ? Vs : Ks) + st * TILE_BYTES + half * HALF_BYTES + pg * c.page_size * 128, kv ? &v_map : &k_map, full, half * 64, y);
      }
      ++ic;
    }
  } else if (warp == 1 || warp == 2) {
    // ---------------- issuers, one warp a stream: S(0) S(1) | O(i) S(i+2) | ... as in attention_tc.cu
    const int x = warp - 1;
    const uint32_t q_addr = tc_smem_u32(Qs), k_addr = tc_smem_u32(Ks) + x * (SUB * 128), v_addr = tc_smem_u32(Vs) + x * (SUB * 128);
    const uint32_t tb = tmem + x * COLS_PER_STREAM;
    bool ok = true;
    int kc = 0, hc = 0, ic = 0;                              // key tiles, this stream's halves, pieces so far
    while (ok && walk.next(c, plan, p)) {
      const int n_half = (p.last - p.first + SUB - 1) / SUB, n_tiles = (n_half + 1) / 2;
      const int n_mine = (n_half + 1 - x) / 2;
      ok = tc_mbar_wait(&bars.q_full, ic & 1, abort_flag, err, 62);
      auto issue_qk = [&](int i) {
        const int st = (kc + i) & 1, buf = (hc + i) & 1;
        ok = ok && tc_mbar_wait(&bars.k_full[st], ((kc + i) >> 1) & 1, abort_flag, err, 63);
        if (!ok) return;
        tc_fence_after();
        if (tc_elect_one()) {
          const uint64_t qd = desc_k_major(q_addr), kd = desc_k_major(k_addr + st * TILE_BYTES);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = ((ks >> 2) * HALF_BYTES + (ks & 3) * 32) >> 4;
            tc_mma_ss(tb + COL_S + buf * SUB, qd + off, kd + off, IDESC_S, ks != 0);
          }
          tc_commit(&bars.s_full[x][buf]);
          tc_commit(&bars.k_empty[x][st]);
          if (i == n_mine - 1) tc_commit(&bars.q_empty);
        }
        __syncwarp();
      };
      if (ok && n_mine > 0) issue_qk(0);
      if (ok && n_mine > 1) issue_qk(1);
      for (int i = 0; i < n_mine && ok; ++i) {
        const int st = (kc + i) & 1, buf = (hc + i) & 1;
        ok = tc_mbar_wait(&bars.v_full[st], ((kc + i) >> 1) & 1, abort_flag, err, 64);
        if (!ok) break;
        const int key0 = p.first + (2 * i + x) * SUB;
        if (key0 < p.lo || key0 + SUB > p.last) {            // values that no row sees: zeros
          for (int e = lane; e < SUB * DH * 8; e += 32) {
            const int row = e / (DH * 8), key = key0 + row;
            if (key < p.lo || key >= p.last)
              *reinterpret_cast<uint4*>(Vs + st * TILE_BYTES + (e / 8 % DH) * HALF_BYTES + (x * SUB + row) * 128 + e % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
          __syncwarp();
        }
        ok = tc_mbar_wait(&bars.p_ready[x][buf], ((hc + i) >> 1) & 1, abort_flag, err, 65);
        // the first product of a piece overwrites the sums of the piece before, which the softmax warps must have read
        if (ok && i == 0 && ic > 0) ok = tc_mbar_wait(&bars.o_free, (ic - 1) & 1, abort_flag, err, 66);
        if (!ok) break;
        tc_fence_after();
        if (tc_elect_one()) {
          const uint64_t vd = desc_mn_major(v_addr + st * TILE_BYTES);
#pragma unroll
          for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              tc_mma_ts(tb + COL_O, tb + COL_S + buf * SUB + term * 32 + ks * 8, vd + ks * (2048 >> 4), IDESC_PV, (i | ks | term) != 0);
          tc_commit(&bars.o_done[x]);
          tc_commit(&bars.v_empty[x][st]);
        }
        __syncwarp();
        if (i + 2 < n_mine) issue_qk(i + 2);
      }
      if (!ok) break;
      if (n_mine < n_tiles) {      // an odd number of halves: the last tile has none for stream 1; the producers count on both streams
        const int last = kc + n_tiles - 1;
        ok = tc_mbar_wait(&bars.k_full[last & 1], (last >> 1) & 1, abort_flag, err, 67) &&
             tc_mbar_wait(&bars.v_full[last & 1], (last >> 1) & 1, abort_flag, err, 68);
        if (!ok) break;
        if (tc_elect_one()) {
          const int st = last & 1;
          tc_commit(&bars.k_empty[x][st]);
          tc_commit(&bars.v_empty[x][st]);
          if (n_mine == 0) tc_commit(&bars.q_empty);
        }
        __syncwarp();
      }
      kc += n_tiles; hc += n_mine; ++ic;
    }
  } else if (warp >= 4) {
    // ---------------- softmax, one thread a row
    const int x = (warp - 4) >> 2;
    const int qd = warp & 3;                                 // this warp's quarter of the 128 lanes
    const int row = qd * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(qd * 32) << 16) + x * COLS_PER_STREAM;
    uint64_t* o_done = &bars.o_done[x];
    float* stage = stages + (warp - 4) * 32 * 36;
    bool ok = true;
    int hc = 0, ic = 0;                                      // this stream's halves and the pieces so far
    const float scale_log2 = c.scale_log2;
    while (walk.next(c, plan, p)) {
      const int n_half = (p.last - p.first + SUB - 1) / SUB;
      const int n_mine = (n_half + 1 - x) / 2;
      const bool exists = row < p.tokens * G;
      // the keys that the row sees, row_lo .. row_hi - 1; a row that does not exist sees none, and hinders no warp from working without masks
      int row_lo = 0, row_hi = 0;
      if (exists) {
        const int pos = row_position(c, plan, p.w, p.row0 + row / G);
        row_lo = max(p.lo, c.window > 0 ? pos - c.window + 1 : 0);
        row_hi = min(p.last, pos + 1);
      }
      const bool work = __any_sync(0xffffffffu, exists) != 0;
      const int all_lo = __reduce_max_sync(0xffffffffu, exists ? row_lo : -0x7fffffff), all_hi = __reduce_min_sync(0xffffffffu, exists ? row_hi : 0x7fffffff);
      float m_used = -INFINITY, l = 0.f;
      for (int u = 0; u < n_mine && ok; ++u) {
        const int cc_ = hc + u, h = cc_ & 1;
        ok = __all_sync(0xffffffffu, tc_mbar_wait(&bars.s_full[x][h], (cc_ >> 1) & 1, abort_flag, err, 70)) != 0;
        if (!ok) break;
        bool o_waited = false;
        if (work) {
          tc_fence_after();
          const int key0 = p.first + (2 * u + x) * SUB;
          const uint32_t s_addr = lane_addr + COL_S + h * SUB;
          const bool interior = key0 >= all_lo && key0 + SUB <= all_hi;
          const int vis_hi = row_hi - key0, vis_lo = row_lo - key0;
          uint32_t v[2][32];
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) tc_ld32(s_addr + cc * 32, v[cc]);
          tc_wait_ld();
          float mxc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          if (interior) {
#pragma unroll
            for (int cc = 0; cc < 2; ++cc)
#pragma unroll
              for (int i = 0; i < 32; i += 2)
                mxc[(cc << 1) | ((i >> 1) & 1)] = tc_max3(mxc[(cc << 1) | ((i >> 1) & 1)], __uint_as_float(v[cc][i]), __uint_as_float(v[cc][i + 1]));
          } else {
#pragma unroll
            for (int cc = 0; cc < 2; ++cc)
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const bool vis = cc * 32 + i < vis_hi && cc * 32 + i >= vis_lo;
                if (vis) mxc[(cc << 1) | (i & 1)] = fmaxf(mxc[(cc << 1) | (i & 1)], __uint_as_float(v[cc][i]));
              }
          }
          const float mx = fmaxf(fmaxf(mxc[0], mxc[1]), fmaxf(mxc[2], mxc[3])) * scale_log2;   // the scale is positive
          // the reference stays unless the new maximum is more than 2^8 above it (a warp's decision: tensor memory is accessed by warps)
          const float m_new = fmaxf(m_used, mx);
          const bool grow = m_new > m_used + 8.f;
          const bool any_grow = __any_sync(0xffffffffu, grow) != 0;
          float factor = 1.f;
          if (any_grow && grow) {
            factor = m_used == -INFINITY ? 0.f : tc_exp2(m_used - m_new);
            m_used = m_new;
          }
          const float ref = m_used == -INFINITY ? 0.f : m_used;
          if (u > 0 && any_grow) {
            ok = __all_sync(0xffffffffu, tc_mbar_wait(o_done, (cc_ - 1) & 1, abort_flag, err, 71)) != 0;
            if (!ok) break;
            o_waited = true;
            tc_fence_after();
            l *= factor;
#pragma unroll 1
            for (int cc = 0; cc < DN / 16; ++cc) {
              uint32_t o[16];
              tc_ld16(lane_addr + COL_O + cc * 16, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
              tc_st16(lane_addr + COL_O + cc * 16, o);
            }
          }
          f32x2 sums[2] = {0, 0};
          const f32x2 scales = pair_of(scale_log2, scale_log2), refs = pair_of(-ref, -ref);
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            uint32_t pk[16], pr[16];
            if (interior) {
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float z0, z1;
                numbers_of(fma2(pair_of(__uint_as_float(v[cc][i]), __uint_as_float(v[cc][i + 1])), scales, refs), z0, z1);
                const f32x2 e = pair_of(tc_exp2(z0), tc_exp2(z1));
                sums[i >> 1 & 1] = add2(sums[i >> 1 & 1], e);
                weight_terms(e, pk[i >> 1], pr[i >> 1]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const bool v0 = cc * 32 + i < vis_hi && cc * 32 + i >= vis_lo, v1 = cc * 32 + i + 1 < vis_hi && cc * 32 + i + 1 >= vis_lo;
                const float e0 = v0 ? tc_exp2(fmaf(__uint_as_float(v[cc][i]), scale_log2, -ref)) : 0.f;
                const float e1 = v1 ? tc_exp2(fmaf(__uint_as_float(v[cc][i + 1]), scale_log2, -ref)) : 0.f;
                const f32x2 e = pair_of(e0, e1);
                sums[i >> 1 & 1] = add2(sums[i >> 1 & 1], e);
                weight_terms(e, pk[i >> 1], pr[i >> 1]);
              }
            }
            tc_st16(s_addr + cc * 16, pk);
            tc_st16(s_addr + 32 + cc * 16, pr);
          }
          float l0, l1;
          numbers_of(add2(sums[0], sums[1]), l0, l1);
          l += l0 + l1;
          tc_wait_st();
          tc_fence_before();
        }
        // every step waits for the product of the half before, so that the wait after the last one is for it and not for the one two back
        if (u > 0 && !o_waited) {
          ok = __all_sync(0xffffffffu, tc_mbar_wait(o_done, (cc_ - 1) & 1, abort_flag, err, 72)) != 0;
          if (!ok) break;
        }
        tc_mbar_arrive(&bars.p_ready[x][h]);
      }
      if (ok && n_mine > 0) ok = __all_sync(0xffffffffu, tc_mbar_wait(o_done, (hc + n_mine - 1) & 1, abort_flag, err, 73)) != 0;
      // The streams hand each other their maxima and sums; each then joins and stores half of the columns.
      const int par = ic & 1;
      merge_m[par][x][row] = m_used;
      merge_l[par][x][row] = l;
      const int2 workers = walk.item_workers(c, p, blockIdx.x);
      if (threadIdx.x == 128) c.pieces[p.item] = workers;
      tc_fence_before();
      asm volatile("bar.sync 2, 256;\n" ::: "memory");          // the eight softmax warps, on every path
      tc_fence_after();
      const bool go = __all_sync(0xffffffffu, !*abort_flag) != 0;
      if (go && work) {
        const float m0 = merge_m[par][0][row], m1 = merge_m[par][1][row], l0 = merge_l[par][0][row], l1 = merge_l[par][1][row];
        const float m = fmaxf(m0, m1);
        const float a0 = m0 == -INFINITY ? 0.f : tc_exp2(m0 - m), a1 = m1 == -INFINITY ? 0.f : tc_exp2(m1 - m);
        const bool two = n_half > 1;                             // stream 1's accumulator holds something of this piece
        const uint32_t o_addr = tmem + ((uint32_t)(qd * 32) << 16) + COL_O;
        const float ml = (m0 == -INFINITY ? l0 : a0 * l0) + (m1 == -INFINITY ? l1 : a1 * l1);
        const bool sole = is_sole(p, workers);
        const float inv = !sole ? 1.f : ml > 0.f ? 1.f / ml : ml == 0.f ? 0.f : ml;      // (NaN stays)
        const float w0 = a0 * inv, w1 = a1 * inv;
        const long long slot = (long long)(p.item + blockIdx.x) * ROWS + row;
        float* dst = c.part_o + (slot - lane) * D;               // of the warp's first row
        const int count = min(32, p.tokens * G - qd * 32);       // its rows that exist
        if (x == 0 && exists && !sole) c.part_ml[slot] = make_float2(m, ml);
        float finite = 0.f;                                      // NaN: not all of the thread's numbers are
#pragma unroll 1
        for (int cc = 0; cc < DN / 64; ++cc) {
          const int col0 = x * (DN / 2) + cc * 32;
          uint32_t oa[32], ob[32];
          tc_ld32(o_addr + col0, oa);
          if (two) tc_ld32(o_addr + COLS_PER_STREAM + col0, ob);
          tc_wait_ld();
          float y[32];
          // (a stream in which the row sees nothing has sums of zero)
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(oa[i]) * w0;
          if (two) {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = fmaf(__uint_as_float(ob[i]), w1, y[i]);
          }
          if (sole && (DN == D || col0 < D)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) finite = fmaf(y[i], 0.f, finite);
          }
          // a row's 128 bytes by eight lanes: through shared memory, a row of it 36 numbers long (no two lanes of a quarter on a bank)
#pragma unroll
          for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(stage + lane * 36 + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
          __syncwarp();
          const int col = lane % 8 * 4;
          if (DN == D || col0 + col < D) {
            if (!sole) {
              for (int q = lane / 8; q < count; q += 4)
                *reinterpret_cast<float4*>(dst + q * D + col0 + col) = *reinterpret_cast<const float4*>(stage + q * 36 + col);
            } else {
              for (int q = lane / 8; q < count; q += 4) {
                const int r = qd * 32 + q;
                const float4 v = *reinterpret_cast<const float4*>(stage + q * 36 + col);
                const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
                bf16* to = reinterpret_cast<bf16*>(c.out) + ((long long)(p.row0 + r / G) * c.heads + p.kv_head * G + r % G) * D + col0 + col;
                *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
              }
            }
          }
          __syncwarp();
        }
        if (__any_sync(0xffffffffu, exists && finite != finite) && lane == 0) atomicOr(&c.pieces[p.item].y, ANEW);
      }
      tc_fence_before();
      tc_mbar_arrive(&bars.o_free);            // this piece's sums have been read
      if (!go) break;
      ok = true;
      hc += n_mine; ++ic;
    }
  }
  if (*abort_flag) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

static inline Call tc_call(int n_tokens, int n_req, int n_groups, int kv_heads, int group, int page_size) {
  Call c = {};
  c.which = WIDE;
  c.n_tokens = n_tokens; c.n_req = n_req; c.n_groups = n_groups;
  c.kv_heads = kv_heads; c.heads = kv_heads * group;
  c.tokens = ROWS / group; c.rows = ROWS; c.unit_log = 7; c.align_log = page_size == 16 ? 4 : page_size == 32 ? 5 : 6;
  c.workers = ifb_sm_count();
  // (with 5, 6 and 7: 64 answers to 8,000 keys 43.0, 41.8 and 41.9 us, 32 to 2,000 25.8, 25.5 and 25.3, groups of conversations 82.7, 81.2 and 81.4, others with heads of
  // 64 28.0, 27.5 and 29.2, with heads of 96 in pages of 64 23.8, 22.9 and 23.1, with eight heads to a key head 30.1, 28.4 and 28.4)
  c.cost = 6;
  c.extra = 2;
  return c;
}
static int tc_main(const Call& c, const Call& other, const bf16* q, long long q_row, const bf16* pages, bool parts, cudaStream_t stream) {
  const int group = c.heads / c.kv_heads;
  const long long page_rows = c.page_stride / D, rows = (c.num_pages - 1) * page_rows + (long long)c.kv_heads * c.page_size;
  CUtensorMap q_map, k_map, v_map;
  {
    const unsigned long long dims[3] = {(unsigned long long)D, (unsigned long long)c.heads, (unsigned long long)c.n_tokens};
    const unsigned long long strides[2] = {(unsigned long long)D * 2, (unsigned long long)q_row * 2};
    const unsigned box[3] = {64, (unsigned)group, (unsigned)c.tokens};
    if (ifb_tensor_map_bf16(&q_map, q, 3, dims, strides, box)) return IFB_ERR_ARG;
  }
  const unsigned long long dims[2] = {(unsigned long long)D, (unsigned long long)rows}, strides[1] = {(unsigned long long)D * 2};
  const unsigned box[2] = {64, (unsigned)c.page_size};
  if (ifb_tensor_map_bf16(&k_map, pages, 2, dims, strides, box)) return IFB_ERR_ARG;
  if (ifb_tensor_map_bf16(&v_map, pages + (long long)c.kv_heads * c.page_size * D, 2, dims, strides, box)) return IFB_ERR_ARG;
  const size_t smem = TILES_BYTES + STAGES_BYTES + plan_bytes(c.n_req + c.n_groups);
  IFB_ALLOW_SMEM(shared_tc_kernel, smem);
  return ifb_launch(shared_tc_kernel, dim3(c.workers), dim3(THREADS), smem, stream, q_map, k_map, v_map, PageRows{(int)page_rows, (int)rows}, c, other, parts ? 1 : 0);
}
