// Attention of requests whose block tables share leading pages: how the work is cut, and how its pieces are joined.
//
// Request r has the query rows cu_q[r] .. cu_q[r+1]-1 at the positions seq_lens[r] - (its rows) .. seq_lens[r] - 1; the query at position p sees the
// keys max(0, p - window + 1) .. p.  Group g is the requests cu_groups[g] .. cu_groups[g+1]-1, whose tables agree on the first shared_lens[g]
// keys.  With two sets of keys that do not meet, A (shared) and B (its own), a row's softmax is
//   m = max(m_A, m_B),  out = (2^(m_A - m) O_A + 2^(m_B - m) O_B) / (2^(m_A - m) l_A + 2^(m_B - m) l_B)
// with m the largest score (base 2), l the sum of weights 2^(s - m) and O their sum with the values; so it is for any number of pieces.  The rows of a
// group over its shared keys are one matrix product, in which a key is read once for all of them.
//
// Owners: the groups, then the requests.  An owner of at most 16 score rows (rows times the heads of a key head's group) is narrow, the others
// are wide: narrow ones are worked on by warps, sixteen rows each, wide ones by CTAs with larger tiles, in kernels of their own that run beside one another.
// For either an owner's rows are cut into tiles of `tokens` query tokens (a narrow owner is one tile), its keys into units of `unit` keys; a tile of one key
// head is an item.  All units of all items lie in one line, in the order of owner, tile, key head and key, and worker c of n takes those from
// c U / n to (c + 1) U / n: every worker has the same number but for one, however uneven the requests.  A stretch of one item's units within a worker
// is a piece; its sums go to slot (item + c), which no two pieces share, for along the line either the item or the worker moves on.  A last
// kernel joins a row's pieces in their order.  Item numbers leave gaps (an owner's first is floor(first row / tokens) + its place) so that they
// need no sum over the owners.
#pragma once
#include "common.cuh"
#include <math.h>

#define IFB_DEV_ERR_SHARED_PAGE 940   // a block-table entry that some query reads through is not a page of the pool (read as zeros)

namespace shared_attention {

constexpr int MAX_OWNERS = 2048;      // groups and requests of a call
constexpr int NO_POSITION = -1;

enum Class { EVERY, WIDE, NARROW };   // whose owners a kernel works on
constexpr int NARROW_ROWS = 16;

struct Call {
  const int* block_tables;
  const int* cu_q;
  const int* seq_lens;
  const int* cu_groups;
  const int* shared_lens;
  long long bt_stride;
  long long num_pages, page_stride;      // of the pool: elements from a page to the next
  int n_tokens, n_req, n_groups;
  int heads, kv_heads;
  int table_pages, page_size, window;
  float scale_log2;
  int* err;
  // of one class's kernel
  int which;
  int tokens, unit, rows;                // of a tile (rows = tokens x heads of a key head, at most), of a unit
  int align;                             // an item's first key is a multiple of this
  int workers;                           // at most
  int cost;                              // of a unit, to the other class's
  float* part_o;                         // [slots][rows][dim]
  float2* part_ml;                       // [slots][rows]: largest score (base 2), sum of weights
  int2* pieces;                          // [items]: first and last worker of an item that has units
};

__host__ __device__ inline int prefix_items(const Call& c) { return (c.n_tokens / c.tokens + c.n_groups + 1) * c.kv_heads; }
__host__ __device__ inline int all_items(const Call& c) { return prefix_items(c) + (c.n_tokens / c.tokens + c.n_req + 1) * c.kv_heads; }
__host__ inline long long room_align(long long x) { return (x + 255) & ~255LL; }
// The room of one class's kernel, in three parts.
__host__ inline long long room_bytes(const Call& c, int dim) {
  const long long slots = (long long)all_items(c) + c.workers;
  return room_align(slots * c.rows * dim * 4) + room_align(slots * c.rows * 8) + room_align((long long)all_items(c) * 8);
}
__host__ inline void room_at(Call& c, int dim, void* room) {
  const long long slots = (long long)all_items(c) + c.workers;
  c.part_o = (float*)room;
  c.part_ml = (float2*)((char*)room + room_align(slots * c.rows * dim * 4));
  c.pieces = (int2*)((char*)c.part_ml + room_align(slots * c.rows * 8));
}

__device__ __forceinline__ int clamp(int x, int lo, int hi) { return min(max(x, lo), hi); }

// What an owner's rows and keys are.
struct Owner {
  int row0, row1;            // query rows
  int request;               // whose table holds the keys (a group: its first request's)
  int lo, hi;                // keys lo .. hi - 1 at most
  int group;                 // whether it is one
  __device__ __forceinline__ int p_first() const { return hi - (row1 - row0); }      // a request: the position of its first row
};
__device__ __forceinline__ int request_row(const Call& c, int r) { return clamp(c.cu_q[r], 0, c.n_tokens); }
__device__ __forceinline__ int request_len(const Call& c, int r) { return clamp(c.seq_lens[r], 0, (int)min((long long)c.table_pages * c.page_size, 0x7fffff00LL)); }
__device__ __forceinline__ int group_start(const Call& c, int g) { return clamp(c.cu_groups[g], 0, c.n_req); }
__device__ __forceinline__ int shared_len(const Call& c, int g) { return clamp(c.shared_lens[g], 0, (int)min((long long)c.table_pages * c.page_size, 0x7fffff00LL)); }

// The group of a request, or -1.
__device__ __forceinline__ int group_of(const Call& c, int r) {
  if (c.n_groups == 0 || r < group_start(c, 0) || r >= group_start(c, c.n_groups)) return -1;
  int lo = 0, hi = c.n_groups - 1;      // the last group that begins at or before r
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (group_start(c, mid) <= r) lo = mid; else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ Owner owner_at(const Call& c, int o) {
  Owner w;
  w.group = o < c.n_groups;
  if (w.group) {
    const int r0 = group_start(c, o), r1 = max(r0, group_start(c, o + 1));
    w.request = min(r0, c.n_req - 1);
    w.row0 = request_row(c, r0);
    w.row1 = max(w.row0, request_row(c, r1));
    w.lo = 0;
    w.hi = shared_len(c, o);
    if (c.window > 0) {      // no row sees a key before this
      int first = w.hi;
      for (int r = r0; r < r1; ++r) first = min(first, request_len(c, r) - (request_row(c, r + 1) - request_row(c, r)) - c.window + 1);
      w.lo = max(0, first);
    }
  } else {
    const int r = o - c.n_groups;
    const int g = group_of(c, r);
    w.request = r;
    w.row0 = request_row(c, r);
    w.row1 = max(w.row0, request_row(c, r + 1));
    w.lo = g >= 0 ? shared_len(c, g) : 0;
    w.hi = request_len(c, r);
  }
  return w;
}
__device__ __forceinline__ int owner_tiles(const Call& c, const Owner& w) { return (w.row1 - w.row0 + c.tokens - 1) / c.tokens; }
__device__ __forceinline__ int owner_item(const Call& c, const Owner& w, int o) {
  return w.group ? (w.row0 / c.tokens + o) * c.kv_heads : prefix_items(c) + (w.row0 / c.tokens + o - c.n_groups) * c.kv_heads;
}

// The keys that a tile's rows can see (lo .. last - 1), and where their units begin.
struct Span { int first, last, lo, units; };
__device__ __forceinline__ Span tile_span(const Call& c, const Owner& w, int tile) {
  Span s;
  s.lo = w.lo;
  s.last = w.hi;
  if (!w.group) {
    const int t0 = tile * c.tokens, t1 = min(w.row1 - w.row0, t0 + c.tokens);
    if (c.window > 0) s.lo = max(s.lo, w.p_first() + t0 - c.window + 1);
    s.last = min(s.last, w.p_first() + t1);
  }
  s.first = s.lo / c.align * c.align;
  s.units = s.last > s.lo ? (s.last - s.first + c.unit - 1) / c.unit : 0;
  return s;
}
__device__ __forceinline__ bool is_narrow(const Call& c, const Owner& w) { return (w.row1 - w.row0) * (c.heads / c.kv_heads) <= NARROW_ROWS; }
__device__ inline long long owner_units(const Call& c, const Owner& w) {
  const int n = owner_tiles(c, w);
  if (n == 0) return 0;
  if (w.group) return (long long)n * tile_span(c, w, 0).units * c.kv_heads;
  long long u = 0;
  for (int t = 0; t < n; ++t) u += tile_span(c, w, t).units;
  return u * c.kv_heads;
}

// What a CTA knows of all owners, in shared memory: what they are, their first units, and behind those the sum of all.
struct Plan {
  long long* starts;      // [owners + 1]
  Owner* owners;          // [owners]
  long long* sums;        // [32]: of warps; the last: units of the other class
};
__host__ __device__ inline size_t plan_bytes(int owners) { return ((size_t)(owners + 1) * (8 + sizeof(Owner)) + 32 * 8 + 15) & ~(size_t)15; }
__device__ __forceinline__ Plan plan_at(unsigned char* at, int owners) {
  Plan p;
  p.starts = reinterpret_cast<long long*>(at);
  p.sums = p.starts + owners + 1;
  p.owners = reinterpret_cast<Owner*>(p.sums + 32);
  return p;
}
// All threads of a CTA (up to 31 warps) call it.  The kernel before this one has ended (the call's numbers are its to write).  `other`: the other class's call.
__device__ inline void make_plan(const Call& c, const Call& other, const Plan& plan) {
  long long *starts = plan.starts, *warp_sums = plan.sums;
  const int owners = c.n_groups + c.n_req, tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5;
  long long base = 0;
  if (tid == 0) plan.sums[31] = 0;
  for (int o0 = 0; o0 < owners; o0 += nt) {
    const int o = o0 + tid;
    long long u = 0, theirs = 0;
    if (o < owners) {
      const Owner w = owner_at(c, o);
      plan.owners[o] = w;
      if (c.which == EVERY || (c.which == NARROW) == is_narrow(c, w)) u = owner_units(c, w);
      else theirs += owner_units(other, w);
    }
    long long run = u;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const long long x = __shfl_up_sync(0xffffffffu, run, d); if (lane >= d) run += x; }
    if (lane == 31) warp_sums[warp] = run;
    __syncthreads();
    long long all = 0, before = 0;
    for (int v = 0; v < warps; ++v) { if (v < warp) before += warp_sums[v]; all += warp_sums[v]; }
    if (o < owners) starts[o] = base + before + run - u;
    if (theirs) atomicAdd(reinterpret_cast<unsigned long long*>(plan.sums + 31), (unsigned long long)theirs);
    base += all;
    __syncthreads();
  }
  if (tid == 0) starts[owners] = base;
  __syncthreads();
}

// How many of `sms` SMs the wide owners' kernel has: as much of them as of the cost; one at least where there is something to do, also for the other.
__device__ __forceinline__ int wide_sms(int sms, long long wide, long long narrow) {
  if (wide == 0) return 0;
  if (narrow == 0) return sms;
  return (int)max(1LL, min((long long)sms - 1, (sms * wide + (wide + narrow) / 2) / (wide + narrow)));
}

// A worker's walk over its pieces; `limit`: how many workers there are.
struct Piece {
  Owner w;
  int tile, kv_head, item;
  int first, last, lo;      // keys first .. last - 1 of whole units; visible ones are lo .. Span.last - 1 of these
  int row0, tokens;         // of the tile
};
struct Walk {
  long long at, end, total, workers;
  int o, tile;              // where `at` lies
  long long tile_start;     // the first unit of the tile
  int open;                 // the owner whose numbers are in w
  Owner w;
  __device__ __forceinline__ void begin(const Call& c, const Plan& plan, int worker, int limit) {
    const long long* starts = plan.starts;
    total = starts[c.n_groups + c.n_req];
    workers = min((long long)limit, total);      // each has a unit: an item's pieces leave none out
    at = end = 0;
    if (worker < workers) {
      at = worker * total / workers;
      end = (worker + 1) * total / workers;
    }
    open = -1;
    if (at >= end) return;
    int lo = 0, hi = c.n_groups + c.n_req - 1;      // the last owner that begins at or before `at`: it has units
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (starts[mid] <= at) lo = mid; else hi = mid - 1;
    }
    o = lo;
    tile = 0;
    tile_start = starts[o];
  }
  // The next piece; false: there is none.
  __device__ __forceinline__ bool next(const Call& c, const Plan& plan, Piece& p) {
    const long long* starts = plan.starts;
    if (at >= end) return false;
    while (at >= starts[o + 1]) { ++o; tile = 0; tile_start = starts[o]; }
    if (open != o) {
      w = plan.owners[o];
      open = o;
      if (w.group && at > tile_start) {      // tiles of a group are alike
        const long long per = (long long)tile_span(c, w, 0).units * c.kv_heads;
        tile = (int)((at - tile_start) / per);
        tile_start += tile * per;
      }
    }
    Span s = tile_span(c, w, tile);
    while (at >= tile_start + (long long)s.units * c.kv_heads) {
      tile_start += (long long)s.units * c.kv_heads;
      s = tile_span(c, w, ++tile);
    }
    const int in_tile = (int)(at - tile_start);
    p.w = w;
    p.tile = tile;
    p.kv_head = in_tile / s.units;
    const int u0 = in_tile % s.units;
    const long long rest = end - at;
    const int u1 = (int)min((long long)s.units, u0 + rest);
    p.item = owner_item(c, w, o) + tile * c.kv_heads + p.kv_head;
    p.first = s.first + u0 * c.unit;
    p.last = min(s.last, s.first + u1 * c.unit);
    p.lo = max(s.lo, p.first);
    p.row0 = w.row0 + tile * c.tokens;
    p.tokens = min(c.tokens, w.row1 - p.row0);
    at += u1 - u0;
    return true;
  }
  // The workers that have pieces of the item whose piece came last.
  __device__ __forceinline__ int2 item_workers(const Call& c, const Piece& p) const {
    const Span s = tile_span(c, p.w, p.tile);
    const long long a = tile_start + (long long)p.kv_head * s.units, b = a + s.units - 1;
    return make_int2((int)(((a + 1) * workers - 1) / total), (int)(((b + 1) * workers - 1) / total));
  }
};

// The position of a query row of an owner: of a group's row by its request.
__device__ __forceinline__ int row_position(const Call& c, const Plan& plan, const Owner& w, int row) {
  if (!w.group) return w.p_first() + row - w.row0;
  const Owner* requests = plan.owners + c.n_groups;      // the first whose rows end behind it
  int lo = w.request, hi = c.n_req - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (requests[mid].row1 <= row) lo = mid + 1; else hi = mid;
  }
  return requests[lo].hi - (requests[lo].row1 - row);
}

// The first elements of a page's keys (values: `kv_heads` page_size dim further on); -1: not a page of the pool.
__device__ __forceinline__ long long page_at(const Call& c, int request, int page) {
  const int id = c.block_tables[request * c.bt_stride + page];
  if (id < 0 || id >= c.num_pages) return -1;
  return id * c.page_stride;
}

// ---------------------------------------------------------------------------------------------------- the join
// A block takes a token's heads, a warp one head at a time; a lane has columns lane, lane + 32, ...  `wide` and `narrow`: the classes' calls (of
// `wide.which` EVERY there is no other).
constexpr int JOIN_WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const __grid_constant__ Call wide, const __grid_constant__ Call narrow, int dim, T* out) {
  __shared__ int found[1];
  ifb_pdl_wait();
  ifb_pdl_trigger();
  const int token = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  if (tid == 0) found[0] = -1;
  __syncthreads();
  for (int r = tid; r < wide.n_req; r += JOIN_WARPS * 32)
    if (request_row(wide, r) <= token && token < request_row(wide, r + 1)) found[0] = r;
  __syncthreads();
  const int r = found[0];
  if (r < 0) return;      // a row of no request: left as it is
  const int g = group_of(wide, r), group = wide.heads / wide.kv_heads;
  const int head = blockIdx.y * JOIN_WARPS + (tid >> 5);
  if (head >= wide.heads) return;
  const int kv_head = head / group;
  int first[2] = {0, 0}, last[2] = {-1, -1};
  const float2* ml_at[2] = {nullptr, nullptr};      // of the item's slot for worker 0
  const float* o_at[2] = {nullptr, nullptr};
  int rows[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int o = k == 0 ? g : wide.n_groups + r;
    if (o < 0) continue;
    const Owner w = owner_at(wide, o);
    const Call& c = wide.which != EVERY && is_narrow(wide, w) ? narrow : wide;
    const int tile = (token - w.row0) / c.tokens;
    if (tile_span(c, w, tile).units == 0) continue;
    const int item = owner_item(c, w, o) + tile * c.kv_heads + kv_head;
    const int2 workers = c.pieces[item];
    first[k] = max(0, workers.x); last[k] = min(workers.y, c.workers - 1);
    rows[k] = c.rows;
    const long long at = (long long)item * c.rows + (token - w.row0 - tile * c.tokens) * group + head % group;
    ml_at[k] = c.part_ml + at;
    o_at[k] = c.part_o + at * dim;
  }
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    for (int x = first[k] + lane; x <= last[k]; x += 32) m = fmaxf(m, ml_at[k][(long long)x * rows[k]].x);
  m = warp_max(m);
  constexpr int PER = 256 / 32;
  float acc[PER], den = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) acc[j] = 0.f;
  if (m == -INFINITY) m = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    for (int x = first[k]; x <= last[k]; ++x) {
      const float2 ml = ml_at[k][(long long)x * rows[k]];
      if (ml.y == 0.f) continue;      // a piece of which the row sees nothing
      const float f = exp2f(ml.x - m);
      den = fmaf(f, ml.y, den);
      const float* o = o_at[k] + (long long)x * rows[k] * dim;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (lane + j * 32 < dim) acc[j] = fmaf(f, o[lane + j * 32], acc[j]);
    }
  const float inv = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den;      // (NaN stays)
  T* dst = out + ((long long)token * wide.heads + head) * dim;
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (lane + j * 32 < dim) dst[lane + j * 32] = from_f32<T>(acc[j] * inv);
}

template <typename T> static int join(const Call& wide, const Call& narrow, int dim, T* out, cudaStream_t stream) {
  return ifb_launch(join_kernel<T>, dim3(wide.n_tokens, (wide.heads + JOIN_WARPS - 1) / JOIN_WARPS), dim3(JOIN_WARPS * 32), 0, stream, wide, narrow, dim, out);
}

}  // namespace shared_attention
