// Drawing a token for each row of logits under top-k, top-p and min-p, and the log probability and rank of given tokens.
//
// sample_cut.  With m the row's largest logit (NaN counts as -inf throughout) w_i = exp((l_i - m) / T); tokens are ordered by falling logit,
// equal ones by rising index.  A: the first k of the order (k < 1 or >= the vocabulary: all).  B: those of A before which A has less than p of its weight
// (p >= 1: all; at least the first).  C: those of B with w_i >= min_p (or l_i = m).  The token is the smallest index i of C with
// sum_{j <= i, j in C} w_j > u sum_C w; its log probability under C is (l_i - m) / T - log sum_C w.  T = 0 (or not above 0): the first of
// the order, log probability 0.  T NaN: the row is not drawn, nothing is written.  A row without a number above -inf: token 0, NaN.
//
// Weights are whole numbers W_i = round(2^44 w_i), from 64-bit arithmetic (so what is below 2^-45 of the largest is never drawn).  The borders between 150,000 tokens lie some 1e-6 of the sum apart, so that
// 32-bit sums (1e-7) would move one draw in tens to another token; with W one row in some 100,000 comes near a border (the errors of 150,000
// roundings add up to 1e-11).  And sums of whole numbers do not depend on their order: a row's token depends on the row alone, not on how many CTAs or
// threads share it.  2^44 times the largest vocabulary stays below 2^63.
//
// A row is shared by a cluster of C CTAs, which keep its slices in shared memory: it is read from memory once.  A cut is found by counts (top-k)
// or weights (top-p) in bins of equal width over (l - m) / T.  At first the bins reach 14 factors of two down, where nearly all cuts are and few tokens, so
// that few take part in the bins' atomics (what lies below is one sum); a cut that is not there is looked for over 24, and then over all 46.  The bin that the cut
// runs through is divided once more if it has many members; the members left, 512 at most (or all tokens of a row that has no more), go to every CTA, which puts them in order and finds the cut
// for itself.  Where too many are left (ties), a search over the ordered bits of their values finds the last value that is kept, and a count in index order the
// last of its tokens.
//
// What bounds it, by clock stamps in the kernel (one row of 151,936 under top-p, 16 CTAs, 17.2 us): its parameters 0.9 us, reading it 0.8, its maximum 1.2, weights
// and bins 3.2, their merging 2.9 and sum 0.4, the bin and its list in order 4.2, the weights of what is kept 1.3, prefix sums and draw 2.3.  The cluster meets six
// times: when all have begun, for the maximum, before and after the merging, for the list, for the prefix sums; twice more where the bin is divided, and for every further
// reach.  Rows with many tokens near the cut take 22 us (the divided bin, and weights of more tokens), rows whose cut the second reach holds 28.  Many rows are
// bound by the instructions of the bins and of the weights, and by how many clusters fit on the device (two CTAs to an SM): of 64 rows of all kinds
// those with cuts take 18 to 56 us each, 28 in the mean, the longest ones under top-p in the second reach.
#include "common.cuh"
#include <math.h>
#include <type_traits>

typedef unsigned long long u64;
typedef __nv_bfloat16 bf16;

constexpr int NT = 512;                  // threads of a CTA
constexpr int NW = NT / 32;
constexpr int BINS = 1023;               // over a reach of factors of two below the largest weight; place BINS holds the sum of what lies beyond
constexpr float REACH = 46.f;            // beyond it a weight is 0
constexpr int TRIES = 3;                 // reaches of the bins: 14, 24, 46
__device__ __forceinline__ float reach_of(int t) { return t == 0 ? 14.f : t == 1 ? 24.f : REACH; }
constexpr int SUBS = 256;                // parts of a bin
constexpr int LIST = NT;                 // members that are put in order, one a thread
constexpr int MAX_CLUSTER = 16;          // (beyond 8 a device may refuse: then no such cluster is taken)
constexpr int SURE_CLUSTER = 8;
constexpr int SLICE = 46080;             // most logits of a CTA: 180 KB (in 32 bits)
constexpr int SHARED_SLICE = 19072;      // up to here two CTAs fit on an SM
constexpr double UNIT = 17592186044416.0;      // 2^44
constexpr u64 ALL = ~0ull;

// ---------------------------------------------------------------------------------------------------- clusters
__device__ __forceinline__ uint32_t s_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t peer(const void* p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(s_addr(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ uint32_t peer_u32(const uint32_t* p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(peer(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ u64 peer_u64(const u64* p, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];\n" : "=l"(v) : "r"(peer(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void put_u32(uint32_t* p, int rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(peer(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void put_u64(u64* p, int rank, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;\n" ::"r"(peer(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t add_peer(uint32_t* p, int rank, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;\n" : "=r"(old) : "r"(peer(p, rank)), "r"(v) : "memory");
  return old;
}
__device__ __forceinline__ int cluster_rank() { int r; asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r)); return r; }
__device__ __forceinline__ int cluster_size() { int r; asm("mov.u32 %0, %%cluster_nctaid.x;\n" : "=r"(r)); return r; }
// All threads of all CTAs of the row; what was written to shared memory before it, one's own or a peer's, is seen after it.
__device__ __forceinline__ void row_sync(int ctas) {
  if (ctas == 1) { __syncthreads(); return; }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// ---------------------------------------------------------------------------------------------------- weights
// 2^(44 + j / 256), in shared memory.
constexpr int STEPS = 256;
struct Exp2Table { double t[STEPS]; };

// How a row's numbers become weights.
struct RowScale {
  double m, s;      // the largest logit, log2(e) / T
  float top;        // the largest logit
  float to_bin;     // bins per unit of m - l
  float to_log2;    // s, but at most 3e38 (temperatures below the smallest normal number have more): bins and floors by it are wider, no less right
  float low;        // a logit whose weight is far below a unit: what lies below it counts as it (a plain row's; see set)
  bool plain;       // whether that is so: no infinity among the largest, 500 factors of two are more than a rounding of m, and to_log2 is all of s
  __device__ __forceinline__ void set(float largest, float temperature) {
    top = largest;
    m = (double)largest;
    s = 1.4426950408889634074 / (double)temperature;
    to_log2 = (float)fmin(s, 3e38);
    to_bin = 0.f;
    low = largest - 500.f / to_log2;
    plain = fabsf(largest) * to_log2 < 1e9f && 500.f / to_log2 < 3e38f && s < 3e38;      // (false for NaN)
  }
};
// round(2^44 2^y), y = (l - m) s <= 0: 2^52 as a 64-bit number's bits, with the whole number in its last ones.  y = (n + f) / 256, n whole, |f| <= 1/2:
// 2^y = 2^(n / 256) e^x, x = f ln 2 / 256, by the first terms of its Taylor series (x^4 / 24 < 2e-13).  Eight operations in 64 bits and a conversion, without a
// branch, so that a thread has several numbers under way (one after the other they take 250 cycles each, four together 115); NaN counts as `low`.
constexpr u64 RAW = 0x4330000000000000ull;      // 2^52
constexpr double MAGIC = 6755399441055744.0 / STEPS;      // 1.5 2^52 / 256: the sum's last bit is 1/256
__device__ __forceinline__ double weight_parts(double d, const RowScale& rs, const Exp2Table& tab, double& scale, double& t) {      // (t: MAGIC + y)
  constexpr double LN2 = 0.693147180559945309417;
  t = fma(d, rs.s, MAGIC);
  const double r = fma(d, rs.s, -(t - MAGIC));
  const int n = __double2loint(t);
  const double step = tab.t[n & (STEPS - 1)];
  scale = __hiloint2double(__double2hiint(step) + (n & ~(STEPS - 1)) * 4096, __double2loint(step));      // n / 256 into the exponent
  double p = fma(r, LN2 * LN2 * LN2 / 6, LN2 * LN2 / 2);
  p = fma(r, p, LN2);
  return fma(r, p, 1.0);
}
__device__ __forceinline__ u64 plain_raw(float l, const RowScale& rs, const Exp2Table& tab) {
  double scale, t;
  const double p = weight_parts((double)fmaxf(l, rs.low) - rs.m, rs, tab, scale, t);
  return (u64)__double_as_longlong(fma(p, scale, 4503599627370496.0));
}
// The whole number of any row; `w`, if wanted: before rounding.  Weights below 2^-46 are 0.
__device__ __forceinline__ u64 row_weight(float l, const RowScale& rs, const Exp2Table& tab, double* w = nullptr) {
  double scale, t;
  const double p = weight_parts((double)l - rs.m, rs, tab, scale, t);
  const bool none = !(t > MAGIC - REACH), best = l == rs.top;      // (infinities too)
  if (w) *w = best ? UNIT : none ? 0.0 : p * scale;
  const u64 whole = (u64)__double_as_longlong(fma(p, scale, 4503599627370496.0)) & ((1ull << 52) - 1);
  return best ? (u64)UNIT : none ? 0 : whole;
}
// The same as a call, where rows that are not plain go once in a while.
__device__ __noinline__ u64 called_weight(float l, RowScale rs, const Exp2Table* tab) { return row_weight(l, rs, *tab); }

// What min_p asks of a logit, and a little less (of +inf: +inf, since what else there is has no weight).
__device__ __forceinline__ float least_floor(float m, float least, const RowScale& rs) {
  if (m == INFINITY) return m;
  const float l = m - (0.01f - log2f(fminf(least, 1.f))) / rs.to_log2;
  return l - fabsf(l) * 2.4e-7f;
}

// The place of a number in bins of equal width; BINS or more (NaN included): its weight is 0.
__device__ __forceinline__ float row_bin(float l, const RowScale& rs) { return l == rs.top ? 0.f : (rs.top - l) * rs.to_bin; }

// An order-preserving whole number of a float32 number that is not NaN (-0 was made 0).
__device__ __forceinline__ uint32_t ordered(float l) {
  const uint32_t b = __float_as_uint(l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// ---------------------------------------------------------------------------------------------------- sums over a row
struct Exchange { u64 a, b; };
struct CutShared {
  Exp2Table tab;
  Exchange swap[2][MAX_CLUSTER];        // what the CTAs of a row tell each other, in turn
  u64 warp_a[NW], warp_b[NW];
  u64 found[4];
  uint32_t listed[2], own, own_at;      // members of the row's lists, of this CTA's and where these begin
};

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int WARPS> struct RowOf {      // (of CTAs of so many warps)
  CutShared* sh;
  int ctas, rank, turn;
  // Every CTA's (a, b) to every CTA; read with got(r) until the call after the next.
  __device__ __forceinline__ const Exchange* tell(u64 a, u64 b) {      // called by all threads, with the CTA's numbers in thread 0
    Exchange* box = sh->swap[turn];
    turn ^= 1;
    if (threadIdx.x == 0)
      for (int r = 0; r < ctas; ++r) { put_u64(&box[rank].a, r, a); put_u64(&box[rank].b, r, b); }
    row_sync(ctas);
    return box;
  }
  // Sums of (a, b) over all threads of the row.
  __device__ __forceinline__ void sum(u64& a, u64& b) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    a = warp_add(a); b = warp_add(b);
    __syncthreads();
    if (lane == 0) { sh->warp_a[warp] = a; sh->warp_b[warp] = b; }
    __syncthreads();
    a = b = 0;
    if (threadIdx.x == 0)
      for (int w = 0; w < WARPS; ++w) { a += sh->warp_a[w]; b += sh->warp_b[w]; }
    const Exchange* box = tell(a, b);
    a = b = 0;
    for (int r = 0; r < ctas; ++r) { a += box[r].a; b += box[r].b; }
  }
  // Largest a and smallest b over all threads of the row.
  __device__ __forceinline__ void extremes(u64& a, u64& b) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 x = __shfl_xor_sync(0xffffffffu, a, o), y = __shfl_xor_sync(0xffffffffu, b, o);
      a = a > x ? a : x; b = b < y ? b : y;
    }
    __syncthreads();
    if (lane == 0) { sh->warp_a[warp] = a; sh->warp_b[warp] = b; }
    __syncthreads();
    if (threadIdx.x == 0)
      for (int w = 0; w < WARPS; ++w) { a = a > sh->warp_a[w] ? a : sh->warp_a[w]; b = b < sh->warp_b[w] ? b : sh->warp_b[w]; }
    const Exchange* box = tell(a, b);
    a = 0; b = ALL;
    for (int r = 0; r < ctas; ++r) { a = a > box[r].a ? a : box[r].a; b = b < box[r].b ? b : box[r].b; }
  }
  // Largest a and sum of b over all threads of the row.
  __device__ __forceinline__ void largest_and_sum(uint32_t& a, uint32_t& b) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    a = __reduce_max_sync(0xffffffffu, a);
    b = __reduce_add_sync(0xffffffffu, b);
    __syncthreads();
    if (lane == 0) sh->warp_a[warp] = (u64)a << 32 | b;
    __syncthreads();
    if (threadIdx.x == 0)
      for (int w = 1; w < WARPS; ++w) { a = max(a, (uint32_t)(sh->warp_a[w] >> 32)); b += (uint32_t)sh->warp_a[w]; }
    const Exchange* box = tell(a, b);
    a = b = 0;
    for (int r = 0; r < ctas; ++r) { a = max(a, (uint32_t)box[r].a); b += (uint32_t)box[r].b; }
  }
  // The sum of v over the threads of this CTA before this one and the CTAs before it (`total`: over all).
  __device__ __forceinline__ u64 before(u64 v, u64& total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    u64 run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const u64 x = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += x; }
    __syncthreads();
    if (lane == 31) sh->warp_a[warp] = run;
    __syncthreads();
    u64 mine = 0, at = run - v;
    for (int w = 0; w < WARPS; ++w) { const u64 x = sh->warp_a[w]; if (w < warp) at += x; mine += x; }
    const Exchange* box = tell(mine, 0);
    total = 0;
    for (int r = 0; r < ctas; ++r) { if (r < rank) at += box[r].a; total += box[r].a; }
    return at;
  }
};
using Row = RowOf<NW>;

// The counts and weights of `n` bins over all CTAs of the row, from each CTA's own (weights in two halves): to every CTA.
__device__ __forceinline__ void merge_bins(const Row& row, int n, const uint32_t* own_count, const uint32_t* own_lo, const uint32_t* own_hi,
                                           uint32_t* count, u64* mass, bool weighted) {
  row_sync(row.ctas);
  // a CTA has a share of the bins, four threads each of these: each takes a quarter of the CTAs
  const int share = (n + row.ctas - 1) / row.ctas, first = row.rank * share, last = min(n, first + share), q = threadIdx.x & 3;
  for (int b0 = first; b0 < last; b0 += NT / 4) {
    const int b = b0 + (int)(threadIdx.x >> 2);
    uint32_t c = 0;
    u64 w = 0;
    if (b < last)
      for (int r = q; r < row.ctas; r += 4) {
        c += peer_u32(own_count + b, r);
        if (weighted) w += ((u64)peer_u32(own_hi + b, r) << 32) + peer_u32(own_lo + b, r);
      }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) { c += __shfl_xor_sync(0xffffffffu, c, o); w += __shfl_xor_sync(0xffffffffu, w, o); }
    if (b < last)
      for (int r = q; r < row.ctas; r += 4) {
        put_u32(count + b, r, c);
        if (weighted) put_u64(mass + b, r, w);
      }
  }
  row_sync(row.ctas);
}

// The bin that the cut runs through: the first with count (by_mass: weight) before it below `goal` and with it at least that.
// Returns it, and what lies before it; n where the whole lies below the goal.  All threads of a CTA call it.
__device__ __forceinline__ int find_bin(CutShared* sh, int n, const uint32_t* count, const u64* mass, bool by_mass, u64 goal, u64& before_count,
                                        u64& before_mass, bool weighted) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (n + NT - 1) / NT;      // bins of a thread, one after the other
  u64 c = 0, w = 0;
  for (int j = 0; j < per; ++j) {
    const int b = threadIdx.x * per + j;
    if (b < n) { c += count[b]; if (weighted) w += mass[b]; }
  }
  u64 rc = c, rw = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, rc, o), y = __shfl_up_sync(0xffffffffu, rw, o);
    if (lane >= o) { rc += x; rw += y; }
  }
  __syncthreads();
  if (lane == 31) { sh->warp_a[warp] = rc; sh->warp_b[warp] = rw; }
  if (threadIdx.x == 0) { sh->found[0] = n; sh->found[1] = sh->found[2] = 0; }
  __syncthreads();
  rc -= c; rw -= w;
  for (int v = 0; v < warp; ++v) { rc += sh->warp_a[v]; rw += sh->warp_b[v]; }
  for (int j = 0; j < per; ++j) {
    const int b = threadIdx.x * per + j;
    if (b >= n) break;
    const u64 dc = count[b], dw = weighted ? mass[b] : 0;
    const u64 at = by_mass ? rw : rc, d = by_mass ? dw : dc;
    if (at < goal && at + d >= goal) { sh->found[0] = b; sh->found[1] = rc; sh->found[2] = rw; }
    rc += dc; rw += dw;
  }
  __syncthreads();
  before_count = sh->found[1]; before_mass = sh->found[2];
  return (int)sh->found[0];
}

// The last token that a cut keeps, and the weight that it keeps in all.
struct Cut { float l; int i; u64 mass; };
__device__ __forceinline__ bool kept(float l, int i, const Cut& c) { return l > c.l || (l == c.l && i <= c.i); }

// A CTA's slice of a row, in shared memory in the type that it comes in (of 16 bits twice the rows find room: 203 rows of 97,476 under top-p 184 to 145 us, 91 of
// 84,412 95 to 86).
template <typename T> struct Slice {
  T* at;
  __device__ __forceinline__ float operator[](int i) const { return to_f32<T>(at[i]); }
};

struct CutMemory {      // of a CTA, behind its slice of the row
  uint32_t* count; uint32_t* lo; uint32_t* hi;             // its own bins [BINS + 1] each
  uint32_t* row_count; u64* row_mass;                      // the row's bins [BINS + 1]
  uint32_t* sub_count; u64* sub_mass;                      // the row's parts of a bin [SUBS]
  u64* list;                                               // the members of a bin, for top-k and for top-p [2][LIST]: the logit in order, and behind it the index turned over
};
constexpr size_t CUT_BYTES = 16 + (size_t)(BINS + 1) * 24 + (size_t)SUBS * 12 + (size_t)LIST * 16;      // (16: the slice begins up to 3 numbers in)

__device__ __forceinline__ void add_mass(uint32_t* lo, uint32_t* hi, int b, u64 w) {
  const uint32_t x = (uint32_t)w, old = atomicAdd(lo + b, x);
  const uint32_t up = (uint32_t)(w >> 32) + (old + x < old ? 1u : 0u);
  if (up) atomicAdd(hi + b, up);
}

// The members that `in` tells by their logit, at most LIST of them in the row, to every CTA's list `which`, in one order for all.  (A CTA notes its own, in the place
// of its bins' counts, which are merged, and takes room for all of them at once: an addition over the cluster for each member took longer than all the rest.)
template <typename T, class In>
__device__ __forceinline__ void gather(const Row& row, const CutMemory& mem, Slice<T> vals, int n, int base, int which, In in) {
  CutShared* sh = row.sh;
  uint32_t* own = mem.count;
  for (int i0 = threadIdx.x; i0 < n; i0 += 4 * NT) {
    bool is[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) is[j] = i0 + j * NT < n && in(vals[i0 + j * NT]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (is[j]) {
        const uint32_t at = atomicAdd(&sh->own, 1u);
        if (at < LIST) own[at] = i0 + j * NT;      // (always: they were counted)
      }
  }
  __syncthreads();
  const int count = min(sh->own, (uint32_t)LIST);
  if (threadIdx.x == 0 && count) sh->own_at = add_peer(&sh->listed[which], 0, count);
  __syncthreads();
  if (threadIdx.x == 0) sh->own = 0;
  for (int j = threadIdx.x; j < count * row.ctas; j += NT) {
    const uint32_t i = own[j / row.ctas], at = sh->own_at + j / row.ctas;
    if (at < LIST) put_u64(mem.list + which * LIST + at, j % row.ctas, ((u64)ordered(vals[i]) << 32) | (uint32_t)~(base + i));
  }
  row_sync(row.ctas);
  // for the next list of this kind, which comes after another barrier of the row (as the next writes to this list do)
  if (row.rank == 0 && threadIdx.x == 0) sh->listed[which] = 0;
}
// A list in order, the best first: the thread's member, and 0 beyond the last.  A bitonic network, within a warp by shuffles, between warps through the list and
// the place `other` in turn.  (To count for each member what comes before it took 13 us for 512 of them.)
__device__ __forceinline__ u64 sorted_member(u64* list, u64* other, int members) {
  const int tid = threadIdx.x, lane = tid & 31;
  u64 x = tid < members ? list[tid] : 0;
  const bool some = (tid & ~31) < members;      // (a warp without members has zeros until others' come in)
  auto step = [&](int j, bool falling) {
    const u64 y = __shfl_xor_sync(0xffffffffu, x, j);
    if ((((lane & j) == 0) == falling) == (y > x)) x = y;
  };
  if (some) {
#pragma unroll
    for (int k = 2; k <= 32; k *= 2)
#pragma unroll
      for (int j = k / 2; j > 0; j /= 2) step(j, (tid & k) == 0);
  }
  for (int k = 64; k / 2 < members; k *= 2) {
    const bool falling = (tid & k) == 0;
    for (int j = k / 2; j >= 32; j /= 2) {
      other[tid] = x;
      __syncthreads();
      const u64 y = other[tid ^ j];
      if ((((tid & j) == 0) == falling) == (y > x)) x = y;
      u64* t = list; list = other; other = t;
    }
#pragma unroll
    for (int j = 16; j > 0; j /= 2) step(j, falling);
  }
  return x;
}
// The sum of v over this thread and those of the CTA before it.
__device__ __forceinline__ u64 running_sum(CutShared* sh, u64 v) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const u64 x = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += x; }
  __syncthreads();
  if (lane == 31) sh->warp_a[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; ++w) v += sh->warp_a[w];
  return v;
}
// The cut at the member that one thread holds, to all threads of the CTA.
__device__ __forceinline__ void tell_cut(CutShared* sh, bool last, u64 member, u64 mass, Cut& cut) {
  if (last) { sh->found[0] = member; sh->found[1] = mass; }
  __syncthreads();
  cut.l = unordered((uint32_t)(sh->found[0] >> 32));
  cut.i = (int)~(uint32_t)sh->found[0];
  cut.mass = sh->found[1];
  __syncthreads();
}

// The cut through the row's bins after which `goal` tokens (by_mass: at least `goal` of weight) are kept.  False: it does not run through them.
template <typename T>
__device__ __forceinline__ bool find_cut(Row& row, const CutMemory& mem, Slice<T> vals, int n, int base, const RowScale& rs, bool by_mass, u64 goal, bool weighted,
                         Cut& cut) {
  constexpr int key_shift = sizeof(T) == 2 ? 16 : 0;
  CutShared* sh = row.sh;
  u64 bc, bm;
  const int b0 = find_bin(sh, BINS, mem.row_count, mem.row_mass, by_mass, goal, bc, bm, weighted);
  if (b0 >= BINS) return false;
  uint32_t members = mem.row_count[b0];
  int b1 = -1;
  if (members > LIST) {
    __syncthreads();
    for (int b = threadIdx.x; b < SUBS; b += NT) mem.count[b] = mem.lo[b] = mem.hi[b] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) {
      const float f = row_bin(vals[i], rs);
      if (!(f < BINS) || (int)f != b0) continue;
      const int b = (int)((f - b0) * SUBS);      // exact until the last step
      atomicAdd(mem.count + b, 1u);
      if (weighted) add_mass(mem.lo, mem.hi, b, row_weight(vals[i], rs, sh->tab));
    }
    merge_bins(row, SUBS, mem.count, mem.lo, mem.hi, mem.sub_count, mem.sub_mass, weighted);
    u64 c1, m1;
    b1 = find_bin(sh, SUBS, mem.sub_count, mem.sub_mass, by_mass, goal - (by_mass ? bm : bc), c1, m1, weighted);
    if (b1 >= SUBS) return false;      // (never: the parts have what the bin has)
    bc += c1; bm += m1;
    members = mem.sub_count[b1];
  }
  auto member = [&](float l) {
    const float f = row_bin(l, rs);
    return f < BINS && (int)f == b0 && (b1 < 0 || (int)((f - b0) * SUBS) == b1);
  };
  if (members <= LIST) {
    const float f0 = b1 < 0 ? (float)b0 : b0 + b1 * (1.f / SUBS), f1 = b1 < 0 ? b0 + 1.f : b0 + (b1 + 1) * (1.f / SUBS);      // (exact)
    gather(row, mem, vals, n, base, by_mass, [&](float l) { const float f = row_bin(l, rs); return f >= f0 && f < f1; });
    const int i = threadIdx.x;
    const u64 member = sorted_member(mem.list + by_mass * LIST, reinterpret_cast<u64*>(mem.count), (int)members);
    const bool in = i < (int)members;
    const u64 w = in && weighted ? row_weight(unordered((uint32_t)(member >> 32)), rs, sh->tab) : 0;
    const u64 mass = bm + (weighted ? running_sum(sh, w) : 0), next = by_mass ? mass : bc + i + 1, at = by_mass ? mass - w : bc + i;
    tell_cut(sh, in && at < goal && (next >= goal || i + 1 == (int)members), member, mass, cut);
    return true;
  }
  // Many members within a hundred-thousandth of a factor of two: the smallest key above which less than the goal lies, by halving, then its ties in order.
  // (`key_shift`: of 16-bit logits the upper half says all: sixteen halvings fewer.)
  u64 top = 0, low = ALL;
  for (int i = threadIdx.x; i < n; i += NT)
    if (member(vals[i])) { const u64 k = ordered(vals[i]) >> key_shift; top = top > k ? top : k; low = low < k ? low : k; }
  row.extremes(top, low);
  auto above = [&](u64 key, u64& c, u64& w, u64& ties) {      // what lies above a key among the members, and before them
    c = w = 0;
    u64 t = 0, unused = 0;
    for (int i = threadIdx.x; i < n; i += NT) {
      const float l = vals[i];
      if (!member(l)) continue;
      const u64 k = ordered(l) >> key_shift;
      if (k > key) { ++c; if (weighted) w += row_weight(l, rs, sh->tab); }
      t += k == key;
    }
    row.sum(c, w);
    row.sum(t, unused);
    c += bc; w += bm; ties = t;
  };
  u64 c = 0, w = 0, ties = 0;
  while (low < top) {
    const u64 mid = (low + top) >> 1;
    above(mid, c, w, ties);
    if ((by_mass ? w : c) < goal) top = mid; else low = mid + 1;
  }
  above(top, c, w, ties);
  const uint32_t whole = (uint32_t)top << key_shift;
  cut.l = unordered(whole >> 31 ? whole : whole | ((1u << key_shift) - 1));      // (a negative number's bits are turned over)
  const u64 each = weighted ? row_weight(cut.l, rs, sh->tab) : 0;
  u64 take = by_mass ? (each ? (goal - w + each - 1) / each : ties) : goal - c;
  if (take > ties) take = ties;
  cut.mass = w + take * each;
  // the take-th tie in the order of indices
  const int chunk = ((n + NT - 1) / NT) | 1, first = min(n, (int)threadIdx.x * chunk), last = min(n, first + chunk);
  u64 mine = 0, total;
  for (int i = first; i < last; ++i) mine += vals[i] == cut.l;
  u64 at = row.before(mine, total);
  if (at < take && at + mine >= take)
    for (int i = first; i < last; ++i)
      if (vals[i] == cut.l && ++at == take)
        for (int r = 0; r < row.ctas; ++r) put_u64(&sh->found[0], r, (u64)(base + i));
  row_sync(row.ctas);
  cut.i = (int)sh->found[0];
  __syncthreads();
  return true;
}

// Both cuts at once from the order of a list, without weights of any other token: of all tokens that are above -inf (`whole`), or of those that the bins up to `end`
// counted, where the cut to the first k lies above it (`members` of them, k at most).  (Asked as the bins asked: beside an infinite largest logit a finite one's bin may
// be NaN, which no bin counts.)
template <typename T>
__device__ __forceinline__ void list_cut(Row& row, const CutMemory& mem, Slice<T> vals, int n, int base, const RowScale& rs, bool whole, float end, uint32_t members,
                         uint32_t k, float p, Cut& cut) {
  CutShared* sh = row.sh;
  gather(row, mem, vals, n, base, 0, [&](float l) { return whole ? l > -INFINITY : row_bin(l, rs) < end; });
  const uint32_t i = threadIdx.x, most = members < k ? members : k;
  const u64 member = sorted_member(mem.list, reinterpret_cast<u64*>(mem.count), (int)members);
  const u64 w = i < most ? row_weight(unordered((uint32_t)(member >> 32)), rs, sh->tab) : 0, mass = running_sum(sh, w);
  u64 goal = ALL;
  if (p < 1.f) {
    __syncthreads();
    if (i + 1 == most) sh->warp_a[0] = mass;
    __syncthreads();
    const double want = ceil((double)p * (double)sh->warp_a[0]);
    goal = want >= 1.0 ? (u64)want : 1;
  }
  tell_cut(sh, i < most && mass - w < goal && (i + 1 == most || mass >= goal), member, mass, cut);      // the last that is kept
}

template <typename T> struct Vec16;
template <> struct Vec16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& x, float (&v)[4]) {
    v[0] = __uint_as_float(x.x); v[1] = __uint_as_float(x.y); v[2] = __uint_as_float(x.z); v[3] = __uint_as_float(x.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  static __device__ __forceinline__ void read(const float* p, float (&v)[4]) { unpack(*reinterpret_cast<const uint4*>(p), v); }
};
template <> struct Vec16<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {      // of numbers that have 16 bits
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ void read(const bf16* p, float (&v)[8]) { unpack(*reinterpret_cast<const uint4*>(p), v); }
  static __device__ __forceinline__ void unpack(const uint4& x, float (&v)[8]) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
  }
};

struct CutArgs {
  long long pitch;
  int vocab, per;      // of a CTA's slice
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int* out;
  float* logprobs;
};

// The drawn token is the first with more than this of the weight up to it.
__device__ __forceinline__ u64 draw_goal(float u, u64 total) {
  const u64 goal = u > 0.f ? (u64)((double)u * (double)total) : 0;
  return goal < total ? goal : total - 1;
}
__device__ __forceinline__ float drawn_logprob(float l, float m, float temp, u64 total) {
  return (float)((l == m ? 0.0 : ((double)l - (double)m) / (double)temp) - log((double)total / UNIT));
}

// Whether a row is drawn, and top-k or top-p may cut something of it.  (What it takes is asked for at once.)
__device__ __forceinline__ bool has_cuts(const CutArgs& a, long long r) {
  const float t = a.temperature[r], p = a.top_p ? a.top_p[r] : 1.f;
  const int k = a.top_k ? a.top_k[r] : 0;
  return (t > 0.f) & (((k >= 1) & (k < a.vocab)) | (p < 1.f));
}

// `everything`: rows without top-k and top-p too (of few rows, which all find their SMs at once; a second kernel would cost 2 us).
template <typename T>
__global__ void __launch_bounds__(NT, 2) sample_cut_kernel(const T* logits, CutArgs a, int everything) {
  extern __shared__ __align__(16) unsigned char cut_smem[];
  __shared__ CutShared shared;
  CutShared* sh = &shared;
  CutMemory mem;
  mem.row_mass = reinterpret_cast<u64*>(cut_smem + 16 + (size_t)a.per * sizeof(T));      // (a slice is a multiple of eight numbers)
  mem.sub_mass = mem.row_mass + BINS + 1;
  mem.list = mem.sub_mass + SUBS;
  mem.count = reinterpret_cast<uint32_t*>(mem.list + 2 * LIST);
  mem.lo = mem.count + BINS + 1;
  mem.hi = mem.lo + BINS + 1;
  mem.row_count = mem.hi + BINS + 1;
  mem.sub_count = mem.row_count + BINS + 1;
  Row row = {sh, cluster_size(), cluster_rank(), 0};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long r = blockIdx.x / row.ctas;
  const int base = min((long long)a.vocab, (long long)row.rank * a.per), n = min(a.vocab - base, a.per);
  ifb_pdl_wait();
  ifb_pdl_trigger();
  const float temp = a.temperature[r], u = a.uniform[r], p = a.top_p ? a.top_p[r] : 1.f, least = a.min_p ? a.min_p[r] : 0.f;
  const int k = a.top_k ? a.top_k[r] : 0;
  if (tid < STEPS) sh->tab.t[tid] = UNIT * exp2(tid / (double)STEPS);
  if (tid == 0) sh->listed[0] = sh->listed[1] = sh->own = 0;
  for (int b = tid; b <= BINS; b += NT) mem.count[b] = mem.lo[b] = mem.hi[b] = 0;
  bool by_count = k >= 1 && k < a.vocab;
  const bool by_mass = p < 1.f, by_least = least > 0.f, cuts = by_count | by_mass;
  if (everything ? temp != temp : !((temp > 0.f) & cuts)) return;      // the other kernel's row, or one that is not to be drawn
  if (row.ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");

  // ---- the slice into shared memory, and its largest logit
  // (rows of an odd vocabulary begin anywhere: `head` numbers come before the first boundary of 16 bytes, and what follows them is on one here, too)
  constexpr int N = Vec16<T>::N;
  const T* src = logits + r * a.pitch + base;
  const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / (int)sizeof(T)), done = head + (n - head) / N * N;
  const Slice<T> vals = {reinterpret_cast<T*>(cut_smem) + (-head & N - 1)};
  float bv = -INFINITY;
  uint32_t live = 0;
  auto take = [&](float v) {
    v = v == v ? v + 0.f : -INFINITY;      // -0 becomes 0
    bv = fmaxf(bv, v);
    live += v > -INFINITY;
    return v;
  };
  auto put = [&](int i) { vals.at[i] = from_f32<T>(take(to_f32<T>(src[i]))); };      // (exact)
  if (tid < head) put(tid);
#pragma unroll 4
  for (int i = head + tid * N; i < done; i += NT * N) {
    float v[N];
    Vec16<T>::read(src + i, v);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = take(v[j]);
    *reinterpret_cast<uint4*>(vals.at + i) = Vec16<T>::pack(v);
  }
  for (int i = done + tid; i < n; i += NT) put(i);
  if (row.ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");      // every peer has begun: its shared memory may be written
  uint32_t best = ordered(bv);
  row.largest_and_sum(best, live);
  const float m = unordered(best);
  if (m == -INFINITY) {
    if (row.rank == 0 && tid == 0) {
      a.out[r] = 0;
      if (a.logprobs) a.logprobs[r] = __uint_as_float(0x7fc00000u);
    }
    return;
  }
  if (!(temp > 0.f)) {      // the lowest index of the largest
    u64 where = ALL, unused = 0;
    for (int i = n - 1 - tid; i >= 0; i -= NT)
      if (vals[i] == m) where = base + i;
    row.extremes(unused, where);
    if (row.rank == 0 && tid == 0) {
      a.out[r] = (int)where;
      if (a.logprobs) a.logprobs[r] = 0.f;
    }
    return;
  }
  RowScale rs;
  rs.set(m, temp);

  // ---- what top-k and top-p keep
  Cut cut = {-INFINITY, 0x7fffffff, 0};
  bool found = !cuts, used = false;
  // Tokens of a small vocabulary, or that a grammar leaves: a list's worth (104 rows of 316 21.6 to 7.9 us, 176 of 2,971 of which 97 in 100 are forbidden 29.6 to 11.5).
  const bool few = cuts && live <= LIST;
  if (few || (by_count && k <= LIST)) {       // or by counts alone, if the first k and what shares the last one's bin are
    for (int t = 0; t < TRIES && !found; ++t) {
      uint32_t members = live;
      float end = 0.f;
      if (!few) {
        rs.to_bin = (float)fmin(rs.s * (BINS / (double)reach_of(t)), 3e38);
        if (used) {
          for (int b = tid; b < BINS; b += NT) mem.count[b] = 0;
          __syncthreads();
        }
        used = true;
        for (int i0 = tid; i0 < n; i0 += 4 * NT) {
          float f[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] = i0 + j * NT < n ? row_bin(vals[i0 + j * NT], rs) : INFINITY;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (f[j] < BINS) atomicAdd(mem.count + (int)f[j], 1u);
        }
        merge_bins(row, BINS, mem.count, mem.lo, mem.hi, mem.row_count, mem.row_mass, false);
        u64 before, unused;
        const int b = find_bin(sh, BINS, mem.row_count, mem.row_mass, false, (u64)k, before, unused, false);
        if (b >= BINS) {
          if (t == TRIES - 1) { by_count = false; found = !by_mass; }      // fewer than k tokens have a weight: top-k keeps them all
          continue;
        }
        if (before + mem.row_count[b] > LIST) break;
        members = (uint32_t)before + mem.row_count[b];
        end = b + 1.f;
      }
      list_cut(row, mem, vals, n, base, rs, few, end, members, by_count ? (uint32_t)k : (uint32_t)LIST, p, cut);
      found = true;
    }
  }
  if (!found) {
    for (int t = 0; t < TRIES && !found; ++t) {
      const bool last_try = t == TRIES - 1;
      rs.to_bin = (float)fmin(rs.s * (BINS / (double)reach_of(t)), 3e38);
      if (t || used) {      // (no peer reads these any more)
        for (int b = tid; b <= BINS; b += NT) mem.count[b] = mem.lo[b] = mem.hi[b] = 0;
        __syncthreads();
      }
      u64 beyond = 0;
      for (int i0 = tid; i0 < n; i0 += 4 * NT) {
        float f[4], v[4];
        u64 w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = i0 + j * NT;
          const float l = i < n ? vals[i] : -INFINITY;
          v[j] = l;
          f[j] = row_bin(l, rs);
        }
        if (by_mass) {
          if (rs.plain) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = plain_raw(v[j], rs, sh->tab) - RAW;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = called_weight(v[j], rs, &sh->tab);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (f[j] < BINS) {
            atomicAdd(mem.count + (int)f[j], 1u);
            if (by_mass) add_mass(mem.lo, mem.hi, (int)f[j], w[j]);
          } else {
            beyond += w[j];
          }
        }
      }
      beyond = warp_add(beyond);
      if (lane == 0 && beyond) add_mass(mem.lo, mem.hi, BINS, beyond);
      merge_bins(row, BINS + 1, mem.count, mem.lo, mem.hi, mem.row_count, mem.row_mass, by_mass);
      u64 all = 0;
      if (by_mass) {      // every CTA has the row's bins: their sum needs no peer
        u64 x = 0;
        for (int b = tid; b <= BINS; b += NT) x += mem.row_mass[b];
        x = warp_add(x);
        __syncthreads();
        if (lane == 0) sh->warp_a[warp] = x;
        __syncthreads();
        for (int w = 0; w < NW; ++w) all += sh->warp_a[w];
        __syncthreads();
      }
      cut.mass = all;
      // top-k, then top-p in what it left
      for (int what = by_count ? 0 : 1; what < 2; ++what) {
        if (what && !by_mass) { found = true; break; }
        const double want = ceil((double)p * (double)cut.mass);
        const u64 goal = what == 0 ? (u64)k : want >= 1.0 ? (u64)want : 1;
        found = find_cut(row, mem, vals, n, base, rs, what, goal, by_mass, cut);
        if (!found && !(what == 0 && last_try)) break;      // (with fewer than k tokens in the last try's bins top-k keeps everything)
      }
    }
  }

  // ---- the draw: a thread has tokens one after the other
  const int chunk = ((n + NT - 1) / NT) | 1, first = min(n, tid * chunk), last = min(n, first + chunk);      // (odd: no two threads of a warp on a bank)
  auto weigh = [&](int i) -> u64 {
    const float l = vals[i];
    double w;
    const u64 whole = row_weight(l, rs, sh->tab, &w);
    return kept(l, base + i, cut) && (!by_least || w >= (double)least * UNIT || l == m) ? whole : 0;
  };
  u64 mine = 0, total;
  int i = first;
  float floor = cut.l;      // most are not kept
  if (by_least) floor = fmaxf(floor, least_floor(m, least, rs));
  if (!cuts && !by_least && rs.plain) {
    const int from = i;
    for (; i + 4 <= last; i += 4)
      mine += (plain_raw(vals[i], rs, sh->tab) + plain_raw(vals[i + 1], rs, sh->tab)) + (plain_raw(vals[i + 2], rs, sh->tab) + plain_raw(vals[i + 3], rs, sh->tab));
    mine -= (u64)(i - from) * RAW;
  }
  const bool quick = !by_least && rs.plain;
  for (; i + 4 <= last; i += 4)
    if (fmaxf(fmaxf(vals[i], vals[i + 1]), fmaxf(vals[i + 2], vals[i + 3])) >= floor) {
      if (quick) {
#pragma unroll
        for (int j = 0; j < 4; ++j) mine += kept(vals[i + j], base + i + j, cut) ? plain_raw(vals[i + j], rs, sh->tab) - RAW : 0;
      } else {
        mine += (weigh(i) + weigh(i + 1)) + (weigh(i + 2) + weigh(i + 3));
      }
    }
  for (; i < last; ++i) mine += weigh(i);
  const u64 at = row.before(mine, total);
  const u64 goal = draw_goal(u, total);
  const unsigned owner = __ballot_sync(0xffffffffu, at <= goal && at + mine > goal);
  if (owner) {      // the warp weighs that thread's tokens anew, a lane each
    const int from = __ffs(owner) - 1, i0 = __shfl_sync(0xffffffffu, first, from), i1 = __shfl_sync(0xffffffffu, last, from);
    u64 run = __shfl_sync(0xffffffffu, at, from);
    for (int j = i0; j < i1; j += 32) {
      const int i = j + lane;
      const u64 w = i < i1 ? weigh(i) : 0;
      u64 x = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const u64 y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
      if (run + x > goal && run + x - w <= goal) {
        a.out[r] = base + i;
        if (a.logprobs) a.logprobs[r] = drawn_logprob(vals[i], m, temp, total);
      }
      run += __shfl_sync(0xffffffffu, x, 31);
    }
  }
}

// ---------------------------------------------------------------------------------------------------- rows without top-k and top-p
// Greedy rows, and such as are drawn from all tokens or from those that min_p leaves: nothing has to be looked for, so nothing is kept; a row is read for its
// largest logit, and a second time, from L2, for its weights.  A CTA needs no shared memory to speak of and four are on an SM, which matters where there are
// many rows: 256 rows of 151,936 held in shared memory, two CTAs on an SM, took 135 us, so they take 85 (a read takes 24; a weight's twenty instructions fill half
// of the issue slots, and warps wait for the second pass's loads longer than for anything else).  A warp has a stretch of the row, which it
// takes in blocks of 512; a block's sum is kept, so that the draw goes over 512 tokens anew and no more.
constexpr int ST_NT = 256, ST_NW = ST_NT / 32, ST_BLOCK = 512, ST_BLOCKS = 16;      // (a CTA has 65,536 logits at most)

// Four numbers from index i on, where row + i is aligned to them; -inf before 0 and from `end` on.  (NaN passes: a maximum and a comparison take no notice of
// it, and its weight is 0.)
template <typename T> __device__ __forceinline__ void stream_read(const T* row, int i, int end, float (&v)[4]) {
  if (i >= 0 && i + 4 <= end) {
    if constexpr (sizeof(T) == 4) {
      const float4 x = *reinterpret_cast<const float4*>(row + i);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(row + i);
      v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u); v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j >= 0 && i + j < end ? to_f32<T>(row[i + j]) : -INFINITY;
  }
}

// `beside`: the kernel before this one in the stream has the other rows (attention_shared_narrow.cuh has the argument): this one waits for it at its end.
template <typename T>
__global__ void __launch_bounds__(ST_NT, 4) sample_stream_kernel(const T* logits, CutArgs a, int beside) {
  __shared__ CutShared shared;
  __shared__ u64 blocks[ST_NW][ST_BLOCKS];
  CutShared* sh = &shared;
  RowOf<ST_NW> row = {sh, cluster_size(), cluster_rank(), 0};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long r = blockIdx.x / row.ctas;
  sh->tab.t[tid] = UNIT * exp2(tid / (double)STEPS);
  static_assert(STEPS == ST_NT, "a thread makes a step of the table");
  if (row.ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  if (!beside) ifb_pdl_wait();
  ifb_pdl_trigger();
  auto draw = [&]() {
    const float temp = a.temperature[r], u = a.uniform[r], least = a.min_p ? a.min_p[r] : 0.f;
    const bool greedy = !(temp > 0.f), mine = (temp == temp) & !has_cuts(a, r);
    if (row.ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");      // every peer has begun: its shared memory may be written
    if (!mine) return;
    const T* src = logits + r * a.pitch;
    // (the stretches of a row that begins behind a boundary of four numbers begin at that boundary)
    const int early = (int)(reinterpret_cast<uintptr_t>(src) / sizeof(T)) & 3, stretch = a.per / ST_NW;
    const int from = (int)min((long long)a.vocab, (long long)row.rank * a.per + warp * stretch - early), end = min(a.vocab, from + stretch);
    float bv = -INFINITY;
    int bi = 0x7fffffff;
    for (int i0 = from; i0 < end; i0 += ST_BLOCK) {
      float v[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) stream_read<T>(src, i0 + j * 128 + lane * 4, end, v[j]);
      if (greedy) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (v[j][e] > bv) { bv = v[j][e]; bi = i0 + j * 128 + lane * 4 + e; }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) bv = fmaxf(fmaxf(fmaxf(bv, v[j][0]), fmaxf(v[j][1], v[j][2])), v[j][3]);
      }
    }
    bv += 0.f;      // (-0 becomes 0; a largest one is no NaN)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
    }
    // (largest first, then lowest index, as one whole number)
    u64 best = ((u64)ordered(bv) << 32) | (uint32_t)~bi, unused = ALL;
    row.extremes(best, unused);
    const float m = unordered((uint32_t)(best >> 32));
    if (greedy || m == -INFINITY) {
      if (row.rank == 0 && tid == 0) {
        a.out[r] = m == -INFINITY ? 0 : (int)~(uint32_t)best;
        if (a.logprobs) a.logprobs[r] = m == -INFINITY ? __uint_as_float(0x7fc00000u) : 0.f;
      }
      return;
    }
    RowScale rs;
    rs.set(m, temp);
    const bool by_least = least > 0.f;
    const float floor = by_least ? least_floor(m, least, rs) : -INFINITY;
    auto weigh = [&](float l) -> u64 {
      if (!by_least) return row_weight(l, rs, sh->tab);
      double w;
      const u64 whole = row_weight(l, rs, sh->tab, &w);
      return w >= (double)least * UNIT || l == m ? whole : 0;
    };
    u64 all = 0;
    for (int i0 = from, b = 0; i0 < end; i0 += ST_BLOCK, ++b) {
      float v[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) stream_read<T>(src, i0 + j * 128 + lane * 4, end, v[j]);
      u64 sum = 0;
      if (rs.plain && !by_least) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sum += (plain_raw(v[j][0], rs, sh->tab) + plain_raw(v[j][1], rs, sh->tab)) + (plain_raw(v[j][2], rs, sh->tab) + plain_raw(v[j][3], rs, sh->tab));
        sum -= 16 * RAW;
      } else
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!by_least || fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])) >= floor)
          sum += (weigh(v[j][0]) + weigh(v[j][1])) + (weigh(v[j][2]) + weigh(v[j][3]));
      sum = warp_add(sum);
      if (lane == 0) blocks[warp][b] = sum;
      all += sum;
    }
    u64 total, at = row.before(lane == 0 ? all : 0, total);
    at = __shfl_sync(0xffffffffu, at, 0);
    const u64 goal = draw_goal(u, total);
    if (at > goal || at + all <= goal) return;
    // the warp's block that the draw falls into, and the token of it
    int b = 0;
    for (; at + blocks[warp][b] <= goal; ++b) at += blocks[warp][b];
    for (int j = 0; j < 4; ++j) {
      const int i = from + b * ST_BLOCK + j * 128 + lane * 4;
      float v[4];
      stream_read<T>(src, i, end, v);
      u64 w[4], x = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) { w[e] = weigh(v[e]); x += w[e]; }
      u64 run = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const u64 y = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += y; }
      const u64 sum = __shfl_sync(0xffffffffu, run, 31);
      if (at + sum <= goal) { at += sum; continue; }
      u64 c = at + run - x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c <= goal && c + w[e] > goal) {
          a.out[r] = i + e;
          if (a.logprobs) a.logprobs[r] = drawn_logprob(v[e], m, temp, total);
        }
        c += w[e];
      }
      break;
    }
  };
  draw();
  if (beside) ifb_pdl_wait();
}

constexpr size_t MOST_CUT_SMEM = (size_t)SLICE * 4 + CUT_BYTES;
// How many clusters of `ctas` CTAs with so much shared memory (MOST_CUT_SMEM is allowed) the device holds at a time (remembered by what they fit: two of them on an SM, or one); negative: an
// error.
static int cut_clusters(const void* kernel, int dtype, int ctas, size_t smem) {
  static std::atomic<int> known[IFB_MAX_DEVICES][2][2][MAX_CLUSTER + 1];      // (host threads ask at once; they find the same)
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= IFB_MAX_DEVICES) return 0;
  const bool pair = smem <= (size_t)SHARED_SLICE * 4 + CUT_BYTES;
  std::atomic<int>& held = known[dev][dtype][pair][ctas];
  if (const int n = held.load(std::memory_order_relaxed)) return n;
  const size_t size = pair ? (size_t)SHARED_SLICE * 4 + CUT_BYTES : MOST_CUT_SMEM;
  cudaError_t e = cudaSuccess;
  if (ctas > SURE_CLUSTER) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) { cudaGetLastError(); return -(int)e; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = size;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int found = 0;
  e = cudaOccupancyMaxActiveClusters(&found, kernel, &cfg);
  if (e != cudaSuccess) { cudaGetLastError(); return -(int)e; }
  held.store(found, std::memory_order_relaxed);
  return found;
}

// logits [rows, vocab] with rows `pitch` elements apart (dtype IFB_F32 or IFB_BF16); per row: temperature, uniform number, and top_k, top_p, min_p (each or
// null); out int32, logprobs float32 or null.
IFB_EXPORT int ifb_sample_cut_max_vocab() { return SURE_CLUSTER * SLICE; }
struct CutPacked {      // a call as the caller packs it: 8-byte fields first
  const void* logits;
  const float *temperature, *uniform;
  const int* top_k;
  const float *top_p, *min_p;
  int* out;
  float* logprobs;
  cudaStream_t stream;
  long long pitch;
  int dtype, rows, vocab, spare;
};
IFB_EXPORT int ifb_sample_cut(const CutPacked* call) {
  const int dtype = call->dtype, rows = call->rows, vocab = call->vocab;
  if (rows <= 0) return IFB_OK;
  if (vocab < 1 || vocab > SURE_CLUSTER * SLICE || rows > (1 << 27)) return IFB_ERR_SIZE;
  if (!call->temperature || !call->uniform || !call->out) return IFB_ERR_ARG;
  // As few CTAs of a row as let two share an SM (of 16-bit numbers counted as 32-bit ones, but for half as many where there are rows for several rounds: 203
  // rows of 97,476 under top-p take 191 us in eight CTAs each and 150 in four, 91 of 84,412 101 and 87); more while all rows' clusters find their SMs at once.
  const void* kernel = dtype == IFB_F32 ? (const void*)sample_cut_kernel<float> : dtype == IFB_BF16 ? (const void*)sample_cut_kernel<bf16> : nullptr;
  if (!kernel) return IFB_ERR_DTYPE;
  if (dtype == IFB_F32) IFB_ALLOW_SMEM(sample_cut_kernel<float>, MOST_CUT_SMEM);
  else IFB_ALLOW_SMEM(sample_cut_kernel<bf16>, MOST_CUT_SMEM);
  auto slice = [&](int n) { return ((vocab + n - 1) / n + 7) & ~7; };
  const int width = dtype == IFB_F32 ? 4 : 2;
  auto room_for = [&](int n) { return cut_clusters(kernel, dtype, n, (size_t)slice(n) * width + CUT_BYTES); };
  int ctas = 1;
  while (ctas < SURE_CLUSTER && slice(ctas) > SHARED_SLICE) ctas *= 2;
  int clusters = room_for(ctas);
  if (ctas > 1 && slice(ctas / 2) * width <= SHARED_SLICE * 4 && rows > clusters + clusters / 2) {
    ctas /= 2;
    clusters = room_for(ctas);
  } else {
    while (ctas < MAX_CLUSTER && vocab / ctas >= 2048 && clusters >= 0) {
      const int next = room_for(ctas * 2);
      if (next < rows) break;
      ctas *= 2;
      clusters = next;
    }
  }
  if (clusters < 0) return clusters;
  const bool everything = rows <= clusters, cuts = everything || call->top_k || call->top_p;
  CutArgs a = {call->pitch, vocab, slice(ctas), call->temperature, call->top_k, call->top_p, call->min_p, call->uniform, call->out, call->logprobs};
  auto go = [&](auto kernel, int count, int n, int threads, size_t smem, auto... args) -> int {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)count * n);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = call->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = n;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ifb_pdl_enabled() ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) { cudaGetLastError(); return -(int)e; }
    return IFB_OK;
  };
  if (cuts) {
    const size_t smem = (size_t)a.per * width + CUT_BYTES;
    const int st = dtype == IFB_F32 ? go(sample_cut_kernel<float>, rows, ctas, NT, smem, (const float*)call->logits, a, everything ? 1 : 0)
                                    : go(sample_cut_kernel<bf16>, rows, ctas, NT, smem, (const bf16*)call->logits, a, everything ? 1 : 0);
    if (st || everything) return st;
  }
  // the other rows: as many CTAs of a row as leave no SM idle, each with whole blocks for its warps
  const int sms = ifb_sm_count();
  int n = 1;
  const int early = (call->pitch | (long long)((uintptr_t)call->logits / width)) & 3 ? 3 : 0;      // (rows may begin up to 3 numbers early)
  auto stretch = [&](int ctas) { return ((vocab + early + ctas * ST_NW - 1) / (ctas * ST_NW) + ST_BLOCK - 1) / ST_BLOCK * ST_BLOCK; };
  while (n < SURE_CLUSTER && (stretch(n) > ST_BLOCKS * ST_BLOCK || ((long long)rows * n * 2 <= 8LL * sms && stretch(n) > 2 * ST_BLOCK))) n *= 2;
  a.per = stretch(n) * ST_NW;
  return dtype == IFB_F32 ? go(sample_stream_kernel<float>, rows, n, ST_NT, 0, (const float*)call->logits, a, cuts ? 1 : 0)
                          : go(sample_stream_kernel<bf16>, rows, n, ST_NT, 0, (const bf16*)call->logits, a, cuts ? 1 : 0);
}

// ---------------------------------------------------------------------------------------------------- log probabilities
// token_logprobs.  log p = l_t - m - log(1 + s), m the row's largest logit and s the sum of e^(l - m) over all tokens but one of the largest: with
// log(1 + s) apart from the leading 1 a token that is nearly certain keeps its digits.  The rank is the number of tokens that come before t in the order of
// falling logits, equal ones by rising index.  One pass over the row: running maximum and sum (32 bits, combined in 64 at the end), and two counts:
// what lies at or above l_t ahead of t, and above it behind t.  A row with a NaN or +inf, or with no number above -inf, gives NaN; a token outside the
// vocabulary NaN and -1.
constexpr int LP_NT = 256;
constexpr int LP_NW = LP_NT / 32;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
struct LpSum { float m, s; };      // the largest number so far, and the sum over all but one of it
__device__ __forceinline__ LpSum lp_join(LpSum a, LpSum b) {
  if (a.m < b.m) { const LpSum t = a; a = b; b = t; }
  if (b.m != -INFINITY) a.s += (1.f + b.s) * lp_exp2((b.m - a.m) * LOG2E);
  else a.s += b.s;      // (0, or NaN)
  return a;
}
// Two numbers per instruction.
__device__ __forceinline__ u64 lp_pair(float a, float b) { u64 r; asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void lp_unpair(u64 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ u64 lp_add2(u64 a, u64 b) { u64 r; asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ u64 lp_mul2(u64 a, u64 b) { u64 r; asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ float lp_min(float a, float b) { float y; asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(y) : "f"(a), "f"(b)); return y; }
// A thread's running state: its largest number, and the sum of e^(l - m) over all others.  The sum is brought to a new largest number without asking whether it is
// one: a branch would be taken by one of 32 threads in nearly every step, and a reference left behind would round what is added at its distance (left up to 40
// behind, two near-equal tokens far above what their thread saw first came out 8e-7 off).
struct LpRun { float m, s; };
// N more numbers (a power of two).  They are paired off: of two the smaller goes into the sum, the larger on to the next round, so that the sum is over all
// but one of the largest without a subtraction; NaN goes into the sum.  `count`: those at or above (AHEAD) or above `lt` are counted, which
// takes a look at the largest first.
template <int N, bool AHEAD> __device__ __forceinline__ void lp_take(LpRun& t, const float (&v)[N], float lt, int& count) {
  float up[N], out[N];
#pragma unroll
  for (int j = 0; j < N; ++j) up[j] = v[j];
#pragma unroll
  for (int n = N, k = 0; n > 1; n /= 2) {
#pragma unroll
    for (int j = 0; j < n / 2; ++j, ++k) {
      out[k] = lp_min(up[2 * j], up[2 * j + 1]);
      up[j] = fmaxf(up[2 * j], up[2 * j + 1]);
    }
  }
  if (up[0] >= lt) {
#pragma unroll
    for (int j = 0; j < N; ++j) count += AHEAD ? v[j] >= lt : v[j] > lt;
  }
  out[N - 1] = lp_min(t.m, up[0]);
  const float before = t.m;
  t.m = fmaxf(t.m, up[0]);
  const float ref = t.m == -INFINITY ? 0.f : t.m;
  t.s *= lp_exp2((before - ref) * LOG2E);      // (1 where it is the same)
  if (N > 1) {
    const u64 minus = lp_pair(-ref, -ref), log2e = lp_pair(LOG2E, LOG2E);
    u64 s[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      float a, b;
      lp_unpair(lp_mul2(lp_add2(lp_pair(out[j], out[(j + 1) % N]), minus), log2e), a, b);
      s[j / 2 & 1] = lp_add2(s[j / 2 & 1], lp_pair(lp_exp2(a), lp_exp2(b)));
    }
    float a, b;
    lp_unpair(lp_add2(s[0], s[1]), a, b);
    t.s += a + b;
  } else {
    t.s += lp_exp2((out[0] - ref) * LOG2E);
  }
}
struct LpBox { LpSum sum; int count; int pad; };

template <typename T>
__global__ void __launch_bounds__(LP_NT) token_logprob_kernel(const T* logits, long long pitch, int vocab, int per, const int* tokens, float* out, int* ranks) {
  __shared__ LpBox warps[LP_NW];
  __shared__ LpBox boxes[MAX_CLUSTER];
  const int ctas = cluster_size(), rank = cluster_rank(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long r = blockIdx.x / ctas;
  if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  ifb_pdl_wait();
  ifb_pdl_trigger();
  const int token = tokens[r];
  const T* row = logits + r * pitch;
  const int base = min((long long)vocab, (long long)rank * per);
  int n = min(vocab - base, per);
  const bool valid = token >= 0 && token < vocab;
  const float lt = valid ? to_f32<T>(row[token]) : 0.f;
  const T* src = row + base;
  int t = max(0, min(n, token - base));      // numbers of this slice ahead of the token
  constexpr int N = Vec16<T>::N;
  LpRun own = {-INFINITY, 0.f};
  int count = 0;
  auto one = [&](int i) {
    const float v[1] = {to_f32<T>(src[i])};
    if (i < t) lp_take<1, true>(own, v, lt, count); else lp_take<1, false>(own, v, lt, count);
  };
  // up to the first boundary of 16 bytes (rows of an odd vocabulary begin anywhere)
  const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / (int)sizeof(T));
  if (tid < head) one(tid);
  src += head;
  n -= head;
  t = max(0, t - head);
  const int vecs = n / N;
  // whole vectors ahead of the token, then those behind it
  auto run = [&](int from, int to, auto ahead) {
    constexpr bool AHEAD = decltype(ahead)::value;
    constexpr int U = sizeof(T) == 4 ? 4 : 2;      // vectors at a time: 16 numbers
    // 16 bits: the next ones are asked for before these are worked on (1,000 rows of 32,768 20.1 to 16.9 us; float32 rows, which have twice the bytes on their
    // way, took 194 in place of 184 so)
    constexpr bool EARLY = sizeof(T) == 2;
    constexpr int STEP = U * LP_NT, REST = (U - 1) * LP_NT;
    const uint4* vec = reinterpret_cast<const uint4*>(src);
    int i = from + tid;
    uint4 x[U];
    if (EARLY && i + REST < to) {
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = vec[i + u * LP_NT];
    }
    for (; i + REST < to; i += STEP) {
      float v[U * N];
      if (!EARLY) {
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = vec[i + u * LP_NT];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float w[N];
        Vec16<T>::unpack(x[u], w);
#pragma unroll
        for (int j = 0; j < N; ++j) v[u * N + j] = w[j];
      }
      if (EARLY && i + STEP + REST < to) {
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = vec[i + STEP + u * LP_NT];
      }
      lp_take<U * N, AHEAD>(own, v, lt, count);
    }
    for (; i < to; i += LP_NT) {
      float v[N];
      Vec16<T>::read(src + (size_t)i * N, v);
      lp_take<N, AHEAD>(own, v, lt, count);
    }
  };
  const int split = min(vecs, t / N);
  run(0, split, std::true_type());
  if (split < vecs && tid < N) one(split * N + tid);      // the vector that the token may be in
  run(split + 1, vecs, std::false_type());
  for (int i = vecs * N + tid; i < n; i += LP_NT) one(i);
  LpSum sum = {own.m, own.s};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const LpSum x = {__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.s, o)};
    sum = lp_join(sum, x);
    count += __shfl_xor_sync(0xffffffffu, count, o);
  }
  if (lane == 0) warps[warp] = {sum, count, 0};
  if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < LP_NW; ++w) { sum = lp_join(sum, warps[w].sum); count += warps[w].count; }
    if (ctas > 1) {
      put_u64(reinterpret_cast<u64*>(&boxes[rank].sum), 0, ((u64)__float_as_uint(sum.s) << 32) | __float_as_uint(sum.m));
      put_u32(reinterpret_cast<uint32_t*>(&boxes[rank].count), 0, (uint32_t)count);
    }
  }
  if (ctas > 1) {
    row_sync(ctas);
    if (rank != 0) return;
  }
  if (tid == 0) {
    if (ctas > 1) {
      sum = boxes[0].sum; count = boxes[0].count;
      for (int c = 1; c < ctas; ++c) { sum = lp_join(sum, boxes[c].sum); count += boxes[c].count; }
    }
    const bool nan = !valid || sum.m == INFINITY || sum.m == -INFINITY;
    out[r] = nan ? __uint_as_float(0x7fc00000u) : (float)((double)lt - (double)sum.m - log1p((double)sum.s));
    if (ranks) ranks[r] = valid ? count : -1;
  }
}

struct LpPacked {      // a call as the caller packs it: 8-byte fields first
  const void* logits;
  const int* tokens;
  float* out;
  int* ranks;
  cudaStream_t stream;
  long long pitch;
  int dtype, rows, vocab, spare;
};
IFB_EXPORT int ifb_token_logprobs(const LpPacked* call) {
  const int dtype = call->dtype, rows = call->rows, vocab = call->vocab;
  const int* tokens = call->tokens;
  float* out = call->out;
  if (rows <= 0) return IFB_OK;
  if (vocab < 1 || vocab > (1 << 30) || rows > (1 << 27)) return IFB_ERR_SIZE;
  if (!tokens || !out) return IFB_ERR_ARG;
  // several CTAs of a row while the rows leave room on the SMs (eight CTAs fit on each)
  const int sms = ifb_sm_count();
  int ctas = 1;
  while (ctas < SURE_CLUSTER && (long long)rows * ctas * 2 <= 4 * sms && vocab / ctas >= 4096) ctas *= 2;
  const int per = ((vocab + ctas - 1) / ctas + 7) & ~7;
  auto go = [&](auto kernel, auto typed) -> int {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * ctas);
    cfg.blockDim = dim3(LP_NT);
    cfg.stream = call->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ifb_pdl_enabled() ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, typed, call->pitch, vocab, per, tokens, out, call->ranks);
    if (e != cudaSuccess) { cudaGetLastError(); return -(int)e; }
    return IFB_OK;
  };
  if (dtype == IFB_F32) return go(token_logprob_kernel<float>, (const float*)call->logits);
  if (dtype == IFB_BF16) return go(token_logprob_kernel<bf16>, (const bf16*)call->logits);
  return IFB_ERR_DTYPE;
}
