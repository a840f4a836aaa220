// Attention over shared pages in bfloat16, compiled for one head size: -DHEAD_DIM=<multiple of 16, at most 256> (default 128).  Narrow owners by
// attention_shared_narrow.cuh, wide ones beside them by attention_shared_tc.cuh where heads and pages allow.  Where they do not, all owners by
// attention_shared_narrow.cuh, in tiles of sixteen rows; groups of more than 16 heads, of which a tile would not hold one token, by
// attention_shared_simt.cuh, which is several times slower (11 requests of 173 queries and 189 to 316 keys, 40 on 8 heads of 256: 2,027 us, and 390 in tiles of sixteen).
#include <cuda.h>

#ifndef HEAD_DIM
#define HEAD_DIM 128
#endif
#if HEAD_DIM % 16 || HEAD_DIM < 16 || HEAD_DIM > 256
#error "HEAD_DIM is a multiple of 16 between 16 and 256"
#endif
constexpr int D = HEAD_DIM;
#include "attention_shared_narrow.cuh"
#include "attention_shared_simt.cuh"
#if HEAD_DIM <= 128
#include "attention_shared_tc.cuh"
constexpr int MOST_PLAN = 227 * 1024 - 5 * 1024 - TILES_BYTES - STAGES_BYTES;      // beside the tiles and what the kernel holds besides
#endif

// Whether the wide owners run on tcgen05.
static bool on_tc(int page_size, int owners, float scale, long long page_stride, long long num_pages) {
#if HEAD_DIM <= 128
  return (page_size == 16 || page_size == 32 || page_size == 64) && scale > 0.f && plan_bytes(owners) <= MOST_PLAN && page_stride % D == 0 &&
         num_pages * (page_stride / D) < 0x7fffffffLL;
#else
  return false;
#endif
}
// Bytes of room for a call's sums at most, whichever kernels it takes.
IFB_EXPORT long long ifb_attention_shared_bf16_room(int n_tokens, int n_req, int n_groups, int kv_heads, int group) {
  const bool any_narrow = group <= NARROW_ROWS;
  // one kernel for all owners (by TMA or not: with it the narrow one has as many workers or more)
  long long most = any_narrow ? room_bytes(narrow::call(true, EVERY, n_tokens, n_req, n_groups, kv_heads, group), D)
                              : room_bytes(sh_call(n_tokens, n_req, n_groups, kv_heads, group, 1), D);
#if HEAD_DIM <= 128
  // tcgen05, and narrow owners beside it
  long long both = room_bytes(tc_call(n_tokens, n_req, n_groups, kv_heads, group, 16), D);
  if (any_narrow) both += room_bytes(narrow::call(true, NARROW, n_tokens, n_req, n_groups, kv_heads, group), D);
  if (both > most) most = both;
#endif
  return parts_bytes(n_tokens) + most;
}

// As ifb_attention_shared.
IFB_EXPORT int ifb_attention_shared_bf16(const Packed* call) {
  const Packed& a = *call;
  if (a.n_tokens <= 0 || a.n_req <= 0) return IFB_OK;
  if (a.dim != D) return IFB_ERR_SIZE;
  if (const int st = check(a, SH_ROWS, 8)) return st;
  const __nv_bfloat16 *q = (const __nv_bfloat16*)a.q, *pages = (const __nv_bfloat16*)a.pages;
  const int group = a.heads / a.kv_heads;
  const bool tc = on_tc(a.page_size, a.n_req + a.n_groups, (float)a.scale, a.page_stride, a.num_pages);
  const bool by_tma = narrow::by_tma(a.page_size, a.page_stride, a.num_pages);
  const bool any_narrow = group <= NARROW_ROWS;
  char* rest = (char*)a.room + parts_bytes(a.n_tokens);
  int st = IFB_OK;
  if (!tc) {      // one kernel for all owners
    Call every = any_narrow ? narrow::call(by_tma, EVERY, a.n_tokens, a.n_req, a.n_groups, a.kv_heads, group)
                            : sh_call(a.n_tokens, a.n_req, a.n_groups, a.kv_heads, group, 1);
    fill(every, a);
    room_at(every, D, rest);
    st = any_narrow ? narrow::run(by_tma, every, every, q, a.q_row, pages, false, a.stream)
                    : sh_main<__nv_bfloat16, (D + 31) / 32>(every, q, a.q_row, pages, D, a.stream);
    return st ? st : join<__nv_bfloat16>(every, every, D, a.stream);
  }
#if HEAD_DIM <= 128
  Call wide = tc_call(a.n_tokens, a.n_req, a.n_groups, a.kv_heads, group, a.page_size);
  Call few = narrow::call(by_tma, NARROW, a.n_tokens, a.n_req, a.n_groups, a.kv_heads, group);
  fill(wide, a);
  fill(few, a);
  room_at(wide, D, rest);
  room_at(few, D, rest + room_bytes(wide, D));
  const bool any_wide = (long long)a.n_tokens * group > NARROW_ROWS;      // no owner has more rows than all
  if (any_wide) {
    st = tc_main(wide, few, q, a.q_row, pages, !any_narrow, a.stream);
    if (st) return st;
  }
  if (any_narrow) {      // (in groups of more heads no owner with rows is)
    st = narrow::run(by_tma, few, wide, q, a.q_row, pages, any_wide, a.stream);
    if (st) return st;
  }
  st = join<__nv_bfloat16>(wide, few, D, a.stream);
#endif
  return st;
}
