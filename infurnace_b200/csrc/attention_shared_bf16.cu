// Attention over shared pages in bfloat16, compiled for one head size: -DHEAD_DIM=<multiple of 16, at most 256> (default 128).  Narrow owners by
// attention_shared_narrow.cuh, wide ones by attention_shared_tc.cuh where heads and pages allow, else by attention_shared_simt.cuh, beside one another.
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
static Call wide_call(bool tc, int n_tokens, int n_req, int n_groups, int kv_heads, int group, int page_size) {
#if HEAD_DIM <= 128
  if (tc) return tc_call(n_tokens, n_req, n_groups, kv_heads, group, page_size);
#endif
  return sh_call(n_tokens, n_req, n_groups, kv_heads, group, WIDE);
}

// Bytes of room for a call's sums at most, whichever kernels it takes.
IFB_EXPORT long long ifb_attention_shared_bf16_room(int n_tokens, int n_req, int n_groups, int kv_heads, int group) {
  const long long a = room_bytes(wide_call(true, n_tokens, n_req, n_groups, kv_heads, group, 16), D);
  const long long b = room_bytes(wide_call(false, n_tokens, n_req, n_groups, kv_heads, group, 16), D);
  return parts_bytes(n_tokens) + (a > b ? a : b) + room_bytes(narrow::call(true, n_tokens, n_req, n_groups, kv_heads, group), D);      // (either has as many workers)
}

// As ifb_attention_shared.
IFB_EXPORT int ifb_attention_shared_bf16(const __nv_bfloat16* q, long long q_row, const __nv_bfloat16* pages, long long page_stride, long long num_pages,
                                         const int* block_tables, long long bt_stride, int table_pages, const int* cu_q, const int* seq_lens,
                                         const int* cu_groups, const int* shared_lens, __nv_bfloat16* out, void* room, int* err, int n_tokens, int n_req,
                                         int n_groups, int heads, int kv_heads, int dim, int page_size, float scale, int window, cudaStream_t stream) {
  if (n_tokens <= 0 || n_req <= 0) return IFB_OK;
  if (dim != D || kv_heads < 1 || heads % kv_heads || heads / kv_heads > SH_ROWS || n_groups < 0 || n_req + n_groups > MAX_OWNERS || page_size < 1 ||
      num_pages < 1)
    return IFB_ERR_SIZE;
  if ((((uintptr_t)q | (uintptr_t)pages) & 15) || q_row % 8 || page_stride % 8 || ((uintptr_t)room & 255)) return IFB_ERR_ALIGN;
  if (window < 0 || !err || page_stride < 2LL * kv_heads * page_size * D) return IFB_ERR_ARG;
  const int group = heads / kv_heads;
  const bool tc = on_tc(page_size, n_req + n_groups, scale, page_stride, num_pages);
  const bool by_tma = narrow::by_tma(page_size, page_stride, num_pages);
  Call wide = wide_call(tc, n_tokens, n_req, n_groups, kv_heads, group, page_size), few = narrow::call(by_tma, n_tokens, n_req, n_groups, kv_heads, group);
  for (Call* c : {&wide, &few}) {
    c->block_tables = block_tables; c->cu_q = cu_q; c->seq_lens = seq_lens; c->cu_groups = cu_groups; c->shared_lens = shared_lens;
    c->bt_stride = bt_stride; c->num_pages = num_pages; c->page_stride = page_stride;
    c->table_pages = table_pages; c->page_size = page_size; c->window = window;
    c->scale_log2 = scale * 1.4426950408889634f;
    c->err = err;
    c->out = out;
    c->parts = (int4*)room;
  }
  char* rest = (char*)room + parts_bytes(n_tokens);
  room_at(wide, D, rest);
  room_at(few, D, rest + room_bytes(wide, D));
  const bool any_wide = (long long)n_tokens * group > NARROW_ROWS;      // no owner has more rows than all
  const bool any_narrow = group <= NARROW_ROWS;
  int st = IFB_OK;
  if (any_wide) {
#if HEAD_DIM <= 128
    if (tc) st = tc_main(wide, few, q, q_row, pages, !any_narrow, stream);
    else
#endif
      st = sh_main<__nv_bfloat16, (D <= 64 ? 8 : D <= 128 ? 16 : 32)>(wide, few, q, q_row, pages, D, !any_narrow, stream);
    if (st) return st;
  }
  if (any_narrow) {
    st = narrow::run(by_tma, few, wide, q, q_row, pages, any_wide, stream);
    if (st) return st;
  }
  return join<__nv_bfloat16>(wide, few, D, stream);
}
