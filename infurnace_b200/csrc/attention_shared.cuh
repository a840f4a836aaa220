// Attention of requests whose block tables share leading pages: how the work is cut, and how its pieces are joined.
//
// Request r has the query rows cu_q[r] .. cu_q[r+1]-1 at the positions seq_lens[r] - (its rows) .. seq_lens[r] - 1; the query at position p sees the
// keys max(0, p - window + 1) .. p.  Group g is the requests cu_groups[g] .. cu_groups[g+1]-1, whose tables agree on the first shared_lens[g]
// keys.  With two sets of keys that do not meet, A (shared) and B (its own), a row's softmax is
//   m = max(m_A, m_B),  out = (2^(m_A - m) O_A + 2^(m_B - m) O_B) / (2^(m_A - m) l_A + 2^(m_B - m) l_B)
// with m the largest score (base 2), l the sum of weights 2^(s - m) and O their sum with the values; so it is for any number of pieces.  The rows of a
// group over its shared keys are one matrix product, in which a key is read once for all of them.
//
// Owners: the groups, then the requests.  Where the requests of a group bring many rows each (64 score rows on average, half a tile), their tiles are full
// without it: the group has no rows then, and each request has all its keys, the shared ones through the first request's table ("split" below).
// An owner of at most 16 score rows (rows times the heads of a key head's group) is narrow, the others are wide: narrow ones are worked on by warps,
// sixteen rows each, wide ones by CTAs with larger tiles, in kernels of their own that run beside one another.
// For either an owner's rows are cut into tiles of `tokens` query tokens (a narrow owner is one tile), its keys into units; a tile of one key
// head is an item.  All units of all items, and `extra` ones for an item's beginning and end, lie in one line, in the order of owner, tile, key
// head and key, and worker c of n takes those from c U / n to (c + 1) U / n: every worker has the same number but for one, however uneven the requests.
// A stretch of one item's units within a worker is a piece; its sums go to slot (item + c), which no two pieces share, for along the line
// either the item or the worker moves on.  A last kernel joins a row's pieces in their order; an item that is one piece, and the only one of its
// rows, is written out where it is worked on.  Item numbers leave gaps (an owner's first is floor(first row / tokens) + its place) so that they need no
// sum over the owners.
#pragma once
#include "common.cuh"
#include <math.h>

#define IFB_DEV_ERR_SHARED_PAGE 940   // a block-table entry that some query reads through is not a page of the pool (read as zeros)

namespace shared_attention {

constexpr int MAX_OWNERS = 2048;      // groups and requests of a call (512 for heads over 128, whose tiles leave less room beside them)
constexpr size_t MOST_SMEM = 224 * 1024;      // of a kernel, beside what it declares
constexpr int NO_POSITION = -1;
enum Class { EVERY, WIDE, NARROW };   // whose owners a kernel works on
constexpr int NARROW_ROWS = 16;
constexpr int FULL_ROWS = 64;         // score rows of a request, on average, from which a group is given up

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
  const void *q, *pages;                 // as they are given: rows `q_row` elements apart
  long long q_row;
  void* out;                             // [n_tokens, heads, dim]
  int4* parts;                           // [n_tokens]: where a row's pieces are (RowParts)
  int* err;
  // of one class's kernel
  int which;
  int tokens, rows;                      // of a tile (rows = tokens x heads of a key head, at most)
  int unit_log, align_log;               // keys of a unit; of which number an item's first key is a multiple: powers of two
  int extra;                             // units that an item's beginning and end cost
  int workers;                           // at most
  int cost;                              // of a unit, to the other class's
  float* part_o;                         // [slots][rows][dim]
  float2* part_ml;                       // [slots][rows]: largest score (base 2), sum of weights
  int2* pieces;                          // [items]: first and last worker of an item that has units
};

__host__ __device__ inline int prefix_items(const Call& c) { return (c.n_tokens / c.tokens + c.n_groups + 1) * c.kv_heads; }
// (a narrow owner beside wide ones is one tile, and the items of its class are numbered by owners)
__host__ __device__ inline int all_items(const Call& c) {
  return c.which == NARROW ? (c.n_groups + c.n_req) * c.kv_heads : prefix_items(c) + (c.n_tokens / c.tokens + c.n_req + 1) * c.kv_heads;
}
__host__ inline long long room_align(long long x) { return (x + 255) & ~255LL; }
// The room of one class's kernel, in three parts.
__host__ inline long long room_bytes(const Call& c, int dim) {
  const long long slots = (long long)all_items(c) + c.workers;
  return room_align(slots * c.rows * dim * 4) + room_align(slots * c.rows * 8) + room_align((long long)all_items(c) * 8);
}
__host__ inline long long parts_bytes(int n_tokens) { return room_align((long long)n_tokens * 16); }
__host__ inline void room_at(Call& c, int dim, void* room) {
  const long long slots = (long long)all_items(c) + c.workers;
  c.part_o = (float*)room;
  c.part_ml = (float2*)((char*)room + room_align(slots * c.rows * dim * 4));
  c.pieces = (int2*)((char*)c.part_ml + room_align(slots * c.rows * 8));
}

struct PageRows { int page, total; };      // the pool as a matrix of rows: rows of a page, rows in all

__device__ __forceinline__ int clamp(int x, int lo, int hi) { return min(max(x, lo), hi); }

// What an owner's rows and keys are.
struct Owner {
  int row0, row1;            // query rows
  int lo, hi;                // keys lo .. hi - 1 at most
  int request;               // whose table holds the keys (a group: its first request's)
  int first, split;          // keys below `split`, a whole number of pages, are in the table of `first` instead
  int group;                 // whether it is one
  __device__ __forceinline__ int p_first() const { return hi - (row1 - row0); }      // a request: the position of its first row
  __device__ __forceinline__ int table(int key) const { return key < split ? first : request; }
};

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
  s.first = s.lo >> c.align_log << c.align_log;
  s.units = s.last > s.lo ? (s.last - s.first - 1 >> c.unit_log) + 1 : 0;
  return s;
}
__device__ __forceinline__ int span_cost(const Call& c, const Span& s) { return s.units ? s.units + c.extra : 0; }
__device__ __forceinline__ int owner_tiles(const Call& c, const Owner& w) { return (w.row1 - w.row0 + c.tokens - 1) / c.tokens; }
__device__ __forceinline__ int owner_item(const Call& c, const Owner& w, int o) {
  if (c.which == NARROW) return o * c.kv_heads;
  return w.group ? (w.row0 / c.tokens + o) * c.kv_heads : prefix_items(c) + (w.row0 / c.tokens + o - c.n_groups) * c.kv_heads;
}
__device__ __forceinline__ bool is_narrow(const Call& c, const Owner& w) { return (w.row1 - w.row0) * (c.heads / c.kv_heads) <= NARROW_ROWS; }
__device__ inline long long owner_cost(const Call& c, const Owner& w) {
  const int n = owner_tiles(c, w);
  if (n == 0) return 0;
  if (w.group) return (long long)n * span_cost(c, tile_span(c, w, 0)) * c.kv_heads;
  long long u = 0;
  for (int t = 0; t < n; ++t) u += span_cost(c, tile_span(c, w, t));
  return u * c.kv_heads;
}

// What a CTA knows of all owners, in shared memory: what they are, their first units, and behind those the sum of all.
struct Plan {
  long long* starts;      // [owners + 1]; before it is made, the call's numbers lie there
  long long* sums;        // [64]: of warps; the second half: of the other class, its sum in the last
  Owner* owners;          // [owners]
};
__host__ __device__ inline size_t plan_bytes(int owners) { return (((size_t)(owners + 1) + 64) * 8 + 15 & ~(size_t)15) + (size_t)owners * sizeof(Owner); }
__device__ __forceinline__ Plan plan_at(unsigned char* at, int owners) {
  Plan p;
  p.starts = reinterpret_cast<long long*>(at);
  p.sums = p.starts + owners + 1;
  p.owners = reinterpret_cast<Owner*>(at + (((size_t)(owners + 1) + 64) * 8 + 15 & ~(size_t)15));
  return p;
}
// All threads of a CTA (up to 31 warps) call it.  The kernel before this one has ended (the call's numbers are its to write).  `other`: the other class's
// call.  The numbers are brought to shared memory first, all at once: read where they are needed they were a chain of seven trips to L2 (5 us).
__device__ inline void make_plan(const Call& c, const Call& other, const Plan& plan) {
  const int R = c.n_req, N = c.n_groups, owners = N + R;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5;
  {
    int* rows = reinterpret_cast<int*>(plan.starts);      // [R + 1] first rows, [R] lengths, [N + 1] first requests, [N] shared lengths
    int *lens = rows + R + 1, *members = lens + R, *shared = members + N + 1;
    const int most = (int)min((long long)c.table_pages * c.page_size, 0x7fffff00LL);
    for (int i = tid; i <= R; i += nt) {
      const int row = c.cu_q[i], len = i < R ? c.seq_lens[i] : 0;
      rows[i] = clamp(row, 0, c.n_tokens);
      if (i < R) lens[i] = clamp(len, 0, most);
    }
    for (int i = tid; i <= N; i += nt) {
      const int r = c.cu_groups[i], len = i < N ? c.shared_lens[i] : 0;
      members[i] = clamp(r, 0, R);
      if (i < N) shared[i] = clamp(len, 0, most);
    }
    __syncthreads();
    const int G = c.heads / c.kv_heads;
    auto full = [&](int g) {      // a group that is given up
      const int n = members[g + 1] - members[g];
      return n > 0 && (long long)(rows[members[g + 1]] - rows[members[g]]) * G >= (long long)FULL_ROWS * n && shared[g] % c.page_size == 0;
    };
    for (int o = tid; o < owners; o += nt) {
      Owner w;
      w.group = o < N;
      w.first = w.split = 0;
      if (w.group) {
        const int r0 = members[o], r1 = max(r0, members[o + 1]);
        w.request = min(r0, R - 1);
        w.row0 = rows[r0];
        w.row1 = full(o) ? w.row0 : max(w.row0, rows[r1]);
        w.lo = 0;
        w.hi = shared[o];
        if (c.window > 0) {      // no row sees a key before this
          int first = w.hi;
          for (int r = r0; r < r1; ++r) first = min(first, lens[r] - (rows[r + 1] - rows[r]) - c.window + 1);
          w.lo = max(0, first);
        }
      } else {
        const int r = o - N;
        w.request = r;
        w.row0 = rows[r];
        w.row1 = max(w.row0, rows[r + 1]);
        w.lo = 0;
        w.hi = lens[r];
        if (N > 0 && r >= members[0] && r < members[N]) {
          int a = 0, b = N - 1;      // the last group that begins at or before r
          while (a < b) {
            const int mid = (a + b + 1) >> 1;
            if (members[mid] <= r) a = mid; else b = mid - 1;
          }
          if (full(a)) { w.first = members[a]; w.split = shared[a]; }
          else w.lo = shared[a];
        }
      }
      plan.owners[o] = w;
    }
    __syncthreads();
  }
  long long base = 0, other_base = 0;
  for (int o0 = 0; o0 < owners; o0 += nt) {
    const int o = o0 + tid;
    long long u = 0, theirs = 0;
    if (o < owners) {
      const Owner w = plan.owners[o];
      if (c.which == EVERY || (c.which == NARROW) == is_narrow(c, w)) u = owner_cost(c, w);
      else theirs = owner_cost(other, w);
    }
    long long run = u;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const long long x = __shfl_up_sync(0xffffffffu, run, d); if (lane >= d) run += x; }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) theirs += __shfl_xor_sync(0xffffffffu, theirs, d);
    if (lane == 31) { plan.sums[warp] = run; plan.sums[32 + warp] = theirs; }
    __syncthreads();
    long long all = 0, before = 0;
    for (int v = 0; v < warps; ++v) { if (v < warp) before += plan.sums[v]; all += plan.sums[v]; other_base += plan.sums[32 + v]; }
    if (o < owners) plan.starts[o] = base + before + run - u;
    base += all;
    __syncthreads();
  }
  if (tid == 0) { plan.starts[owners] = base; plan.sums[63] = other_base; }
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
  int first, last, lo;      // keys first .. last - 1 of whole units; visible ones are lo .. last - 1 of these
  int row0, tokens;         // of the tile
  bool whole;               // the item is this piece
};
struct Walk {
  long long at, end, total, workers;
  int o, tile, cost;        // where the last piece was; what an item of the tile costs
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
    while (at < end) {
      while (at >= starts[o + 1]) { ++o; tile = 0; tile_start = starts[o]; }
      if (open != o) {
        w = plan.owners[o];
        open = o;
        if (w.group && at > tile_start) {      // tiles of a group are alike
          const long long per = (long long)span_cost(c, tile_span(c, w, 0)) * c.kv_heads;
          tile = (int)((at - tile_start) / per);
          tile_start += tile * per;
        }
      }
      Span s = tile_span(c, w, tile);
      cost = span_cost(c, s);
      while (at >= tile_start + (long long)cost * c.kv_heads) {
        tile_start += (long long)cost * c.kv_heads;
        s = tile_span(c, w, ++tile);
        cost = span_cost(c, s);
      }
      const int in_tile = (int)(at - tile_start), head = in_tile / cost, v0 = in_tile % cost;
      const int v1 = (int)min((long long)cost, v0 + (end - at));
      const int u0 = max(0, v0 - c.extra), u1 = v1 - c.extra;
      at += v1 - v0;
      if (u1 <= u0) continue;      // the worker's share is of the item's extra units
      p.w = w;
      p.tile = tile;
      p.kv_head = head;
      p.item = owner_item(c, w, o) + tile * c.kv_heads + head;
      p.first = s.first + (u0 << c.unit_log);
      p.last = min(s.last, s.first + (u1 << c.unit_log));
      p.lo = max(s.lo, p.first);
      p.row0 = w.row0 + tile * c.tokens;
      p.tokens = min(c.tokens, w.row1 - p.row0);
      p.whole = u0 == 0 && u1 == s.units;
      return true;
    }
    return false;
  }
  // The workers that have pieces of the item whose piece came last, this worker being one.
  __device__ __forceinline__ int2 item_workers(const Call& c, const Piece& p, int worker) const {
    if (p.whole) return make_int2(worker, worker);
    const long long a = tile_start + (long long)p.kv_head * cost, b = a + cost;
    return make_int2((int)(((a + c.extra + 1) * workers - 1) / total), (int)((b * workers - 1) / total));
  }
};
// Whether a piece is all that its rows have (`at`: its item's workers): it is written out where it is worked on.  Where something of it is not finite, its item's
// last worker gets ANEW.
constexpr int ANEW = 1 << 30;
__device__ __forceinline__ bool is_sole(const Piece& p, int2 at) { return !p.w.group && p.w.lo == 0 && at.x == at.y; }

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

// Where a row's pieces are, for the join: of its group's item (x, y) and its request's (z, w).  The item of key head 0, or -1: none (x = -2: no request's
// row); row of head 0 in the tile, NARROW_PART if its class is that, SOLE_PART if one piece of it would be all.
constexpr int NARROW_PART = 1 << 16, SOLE_PART = 1 << 17;
// The threads of all CTAs of a kernel call it together, each for some rows.
__device__ inline void write_parts(const Call& wide, const Call& narrow, const Plan& plan) {
  const int N = wide.n_groups, G = wide.heads / wide.kv_heads;
  auto find = [&](const Owner* owners, int n, int token) {      // the first that ends behind it, if it begins at or before it
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (owners[mid].row1 <= token) lo = mid + 1; else hi = mid;
    }
    return lo < n && owners[lo].row0 <= token ? lo : -1;
  };
  for (int token = blockIdx.x * blockDim.x + threadIdx.x; token < wide.n_tokens; token += gridDim.x * blockDim.x) {
    int at[4] = {-1, 0, -1, 0};
    const int r = find(plan.owners + N, wide.n_req, token), g = find(plan.owners, N, token);
    if (r < 0) at[0] = -2;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (r < 0 || (k == 0 && g < 0)) continue;
      const int o = k == 0 ? g : N + r;
      const Owner w = plan.owners[o];
      const bool few = wide.which != EVERY && is_narrow(wide, w);
      const Call& c = few ? narrow : wide;
      const int tile = (token - w.row0) / c.tokens;
      if (tile_span(c, w, tile).units == 0) continue;
      at[2 * k] = owner_item(c, w, o) + tile * c.kv_heads;
      at[2 * k + 1] = (token - w.row0 - tile * c.tokens) * G | (few ? NARROW_PART : 0) | (k == 1 && w.lo == 0 ? SOLE_PART : 0);
    }
    wide.parts[token] = make_int4(at[0], at[1], at[2], at[3]);
  }
}

// ---------------------------------------------------------------------------------------------------- rows worked out anew
// A token's row of one head, key by key over those that it sees, in two passes (maximum, sums): for rows that come out infinite or NaN.  In a matrix product a
// value that some rows of a tile see and others do not meets a weight of zero in these, and a weight's second term of zero in those: where the value is
// infinite or NaN the product is NaN.  All lanes of a warp call it; a lane has a key of 32 for the scores, and the join's columns for the sums.
template <typename T> __device__ __forceinline__ float dot16(const T* a, const T* b);      // of 16 bytes
template <> __device__ __forceinline__ float dot16<float>(const float* a, const float* b) {
  const float4 x = *reinterpret_cast<const float4*>(a), y = *reinterpret_cast<const float4*>(b);
  return fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, x.w * y.w)));
}
template <> __device__ __forceinline__ float dot16<__nv_bfloat16>(const __nv_bfloat16* a, const __nv_bfloat16* b) {
  const uint4 x = *reinterpret_cast<const uint4*>(a), y = *reinterpret_cast<const uint4*>(b);
  const uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fmaf(__uint_as_float(u[i] << 16), __uint_as_float(v[i] << 16), s);
    s = fmaf(__uint_as_float(u[i] & 0xffff0000u), __uint_as_float(v[i] & 0xffff0000u), s);
  }
  return s;
}
template <typename T> __device__ __noinline__ void row_anew(const Call& c, int token, int head, int dim) {
  const int lane = threadIdx.x & 31, N = c.n_groups, R = c.n_req, kv_head = head / (c.heads / c.kv_heads);
  const int most = (int)min((long long)c.table_pages * c.page_size, 0x7fffff00LL);
  auto row = [&](int i) { return clamp(c.cu_q[i], 0, c.n_tokens); };
  auto member = [&](int i) { return clamp(c.cu_groups[i], 0, R); };
  // as make_plan and write_parts have it: the request, its position, and the keys that it has from its group's first
  int lo = 0, hi = R;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (max(row(mid), row(mid + 1)) <= token) lo = mid + 1; else hi = mid;
  }
  if (lo >= R) return;
  const int r = lo, len = clamp(c.seq_lens[r], 0, most), pos = len - (max(row(r), row(r + 1)) - token);
  int first = r, split = 0;
  if (N > 0 && r >= member(0) && r < member(N)) {
    int a = 0, b = N - 1;
    while (a < b) {
      const int mid = (a + b + 1) >> 1;
      if (member(mid) <= r) a = mid; else b = mid - 1;
    }
    first = member(a);
    split = clamp(c.shared_lens[a], 0, most);
  }
  const int key_lo = c.window > 0 ? max(0, pos - c.window + 1) : 0, key_hi = min(len, pos + 1);
  const T* q = reinterpret_cast<const T*>(c.q) + token * c.q_row + (long long)head * dim;
  const T* pages = reinterpret_cast<const T*>(c.pages);
  const long long values = (long long)c.kv_heads * c.page_size * dim;
  auto score = [&](int key, long long& at) {      // (what is no page of the pool is zeros)
    at = page_at(c, key < split ? first : r, key / c.page_size);
    if (at < 0) return 0.f;
    at += ((long long)kv_head * c.page_size + key % c.page_size) * dim;
    float s = 0.f;
    for (int d = 0; d < dim; d += 16 / (int)sizeof(T)) s += dot16<T>(q + d, pages + at + d);
    return s * c.scale_log2;
  };
  float m = -INFINITY, den = 0.f, sums[8] = {};      // columns 4 lane .. 4 lane + 3, and those 128 on
  long long at;
  for (int key = key_lo + lane; key < key_hi; key += 32) m = fmaxf(m, score(key, at));
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  for (int key0 = key_lo; key0 < key_hi && den == den; key0 += 32) {
    at = -1;
    const float weight = key0 + lane < key_hi ? exp2f(score(key0 + lane, at) - ref) : 0.f;
    den += warp_sum(weight);
    for (int j = 0; j < min(32, key_hi - key0); ++j) {
      const float g = __shfl_sync(0xffffffffu, weight, j);
      const long long from = __shfl_sync(0xffffffffu, at, j);
      if (from < 0) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int col = (i >> 2) * 128 + lane * 4 + (i & 3);
        if (col < dim) sums[i] = fmaf(g, to_f32<T>(pages[from + values + col]), sums[i]);
      }
    }
  }
  const float inv = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den;      // (NaN stays)
  T* dst = reinterpret_cast<T*>(c.out) + ((long long)token * c.heads + head) * dim;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int col = (i >> 2) * 128 + lane * 4 + (i & 3);
    if (col < dim) dst[col] = from_f32<T>(sums[i] * inv);
  }
}

// ---------------------------------------------------------------------------------------------------- the join
// A warp takes a head of a token; a lane has the columns from 4 lane on (WIDTH 2, heads over 128: and from 128 + 4 lane on).  `wide` and `narrow`: the classes' calls (the same one where
// there is one kernel only).  Lane x first has piece x: its maximum and denominator, from which the factor that its sums get.
constexpr int JOIN_WARPS = 8;
template <typename T, int WIDTH>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const __grid_constant__ Call wide, const __grid_constant__ Call narrow, int dim) {
  ifb_pdl_wait();
  ifb_pdl_trigger();
  const int token = blockIdx.x, lane = threadIdx.x & 31, head = blockIdx.y * JOIN_WARPS + (threadIdx.x >> 5);
  if (head >= wide.heads) return;
  const int4 at = wide.parts[token];
  if (at.x == -2) return;      // a row of no request: left as it is
  const int group = wide.heads / wide.kv_heads, kv_head = head / group;
  int first[2] = {0, 0}, count[2] = {0, 0}, rows[2] = {0, 0};
  const float2* ml_at[2] = {nullptr, nullptr};      // of the item's slot for its first worker
  const float* o_at[2] = {nullptr, nullptr};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int item = (k ? at.z : at.x) + kv_head, how = k ? at.w : at.y;
    if (item < kv_head) continue;
    const Call& c = how & NARROW_PART ? narrow : wide;
    const int2 workers = c.pieces[item];
    if (how & SOLE_PART && workers.x == (workers.y & ~ANEW)) {      // it is written already
      if (workers.y == workers.x) return;
      const T* row = reinterpret_cast<const T*>(wide.out) + ((long long)token * wide.heads + head) * dim;
      float finite = 0.f;
      for (int col = lane; col < dim; col += 32) finite = fmaf(to_f32<T>(row[col]), 0.f, finite);
      if (__any_sync(0xffffffffu, finite != finite)) row_anew<T>(wide, token, head, dim);
      return;
    }
    first[k] = clamp(workers.x, 0, c.workers - 1);
    count[k] = clamp(workers.y, 0, c.workers - 1) - first[k] + 1;
    rows[k] = c.rows;
    const long long slot = (long long)(item + first[k]) * c.rows + (how & 0xffff) + head % group;
    ml_at[k] = c.part_ml + slot;
    o_at[k] = c.part_o + slot * dim;
  }
  const int n = max(0, count[0]) + max(0, count[1]);
  // in turns of 32 pieces, against a running maximum
  float m = -INFINITY, den = 0.f;
  float4 acc[WIDTH] = {};
  constexpr int ASK = 16 / WIDTH;      // pieces whose sums are asked for at once, the first with the maxima
  for (int x0 = 0; x0 < n; x0 += 32) {
    const int x = x0 + lane;
    const bool k = x >= count[0];
    const long long i = (long long)(k ? x - count[0] : x) * (k ? rows[1] : rows[0]);
    float2 ml = make_float2(-INFINITY, 0.f);
    const float* src = nullptr;
    if (x < n) {
      ml = (k ? ml_at[1] : ml_at[0])[i];
      src = (k ? o_at[1] : o_at[0]) + i * dim;
    }
    const int turn = min(32, n - x0);
    float4 v[WIDTH][ASK];
    auto ask = [&](int t0) {
#pragma unroll
      for (int t = 0; t < ASK; ++t) {
        const float* o = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)(uintptr_t)src, t0 + t & 31));
#pragma unroll
        for (int j = 0; j < WIDTH; ++j) {
          const int col = j * 128 + lane * 4;
          if (t0 + t < turn && col < dim) v[j][t] = *reinterpret_cast<const float4*>(o + col);
        }
      }
    };
    ask(0);
    const float next = fmaxf(m, warp_max(ml.y == 0.f ? -INFINITY : ml.x)), ref = next == -INFINITY ? 0.f : next;
    const float keep = exp2f(m - ref), f = ml.y == 0.f ? 0.f : exp2f(ml.x - ref);      // (a piece of which the row sees nothing has weight 0)
    m = next;
    den = fmaf(den, keep, warp_sum(f * ml.y));
#pragma unroll
    for (int j = 0; j < WIDTH; ++j) { acc[j].x *= keep; acc[j].y *= keep; acc[j].z *= keep; acc[j].w *= keep; }
    for (int t0 = 0; t0 < turn; t0 += ASK) {
      if (t0) ask(t0);
#pragma unroll
      for (int t = 0; t < ASK; ++t) {
        const float g = __shfl_sync(0xffffffffu, f, t0 + t & 31);
        if (g == 0.f || t0 + t >= turn) continue;      // (what has weight 0 may be infinite or NaN)
#pragma unroll
        for (int j = 0; j < WIDTH; ++j) {
          acc[j].x = fmaf(g, v[j][t].x, acc[j].x); acc[j].y = fmaf(g, v[j][t].y, acc[j].y);
          acc[j].z = fmaf(g, v[j][t].z, acc[j].z); acc[j].w = fmaf(g, v[j][t].w, acc[j].w);
        }
      }
    }
  }
  const float inv = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den;      // (NaN stays)
  float finite = 0.f;      // NaN: not all sums are
#pragma unroll
  for (int j = 0; j < WIDTH; ++j)
    if (j * 128 + lane * 4 < dim) finite += acc[j].x * 0.f + acc[j].y * 0.f + (acc[j].z * 0.f + acc[j].w * 0.f);
  if (__any_sync(0xffffffffu, finite != finite)) {
    row_anew<T>(wide, token, head, dim);
    return;
  }
  T* dst = reinterpret_cast<T*>(wide.out) + ((long long)token * wide.heads + head) * dim;
#pragma unroll
  for (int j = 0; j < WIDTH; ++j) {
    const int col = j * 128 + lane * 4;
    if (col < dim) {
      dst[col] = from_f32<T>(acc[j].x * inv); dst[col + 1] = from_f32<T>(acc[j].y * inv);
      dst[col + 2] = from_f32<T>(acc[j].z * inv); dst[col + 3] = from_f32<T>(acc[j].w * inv);
    }
  }
}

template <typename T> static int join(const Call& wide, const Call& narrow, int dim, cudaStream_t stream) {
  const dim3 grid(wide.n_tokens, (wide.heads + JOIN_WARPS - 1) / JOIN_WARPS), block(JOIN_WARPS * 32);
  return dim <= 128 ? ifb_launch(join_kernel<T, 1>, grid, block, 0, stream, wide, narrow, dim) : ifb_launch(join_kernel<T, 2>, grid, block, 0, stream, wide, narrow, dim);
}

// A call as the caller packs it: 8-byte fields first.
struct Packed {
  const void *q, *pages;
  const int *block_tables, *cu_q, *seq_lens, *cu_groups, *shared_lens;
  void *out, *room;
  int* err;
  cudaStream_t stream;
  long long q_row, page_stride, num_pages, bt_stride;
  double scale;
  int table_pages, n_tokens, n_req, n_groups, heads, kv_heads, dim, page_size, window, spare;
};
// What either class's call has from it.
static inline void fill(Call& c, const Packed& a) {
  c.block_tables = a.block_tables; c.cu_q = a.cu_q; c.seq_lens = a.seq_lens; c.cu_groups = a.cu_groups; c.shared_lens = a.shared_lens;
  c.bt_stride = a.bt_stride; c.num_pages = a.num_pages; c.page_stride = a.page_stride;
  c.table_pages = a.table_pages; c.page_size = a.page_size; c.window = a.window;
  c.scale_log2 = (float)(a.scale * 1.4426950408889634);
  c.q = a.q; c.pages = a.pages; c.q_row = a.q_row;
  c.out = a.out;
  c.parts = (int4*)a.room;
  c.err = a.err;
}
// The checks that do not depend on the type; `least`: elements of 16 bytes.
static inline int check(const Packed& a, int most_group, int least) {
  if (a.kv_heads < 1 || a.heads % a.kv_heads || a.heads / a.kv_heads > most_group || a.dim < 16 || a.dim > 256 || a.dim % 16 || a.n_groups < 0 ||
      a.n_req + a.n_groups > MAX_OWNERS || a.page_size < 1 || a.num_pages < 1)
    return IFB_ERR_SIZE;
  if ((((uintptr_t)a.q | (uintptr_t)a.pages | (uintptr_t)a.out) & 15) || a.q_row % least || a.page_stride % least || ((uintptr_t)a.room & 255)) return IFB_ERR_ALIGN;
  if (a.window < 0 || !a.err || !a.room || a.page_stride < 2LL * a.kv_heads * a.page_size * a.dim) return IFB_ERR_ARG;
  return IFB_OK;
}

}  // namespace shared_attention
