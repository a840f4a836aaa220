// Attention over shared pages in float32: every owner by the kernel of attention_shared_simt.cuh.
#include "attention_shared_simt.cuh"

// (two CTAs of heads up to 128 find registers and shared memory on an SM)
static Call call_of(int n_tokens, int n_req, int n_groups, int kv_heads, int group, int dim) {
  return sh_call(n_tokens, n_req, n_groups, kv_heads, group, dim <= 128 ? 2 : 1);
}

// Bytes of room for a call's sums.
IFB_EXPORT long long ifb_attention_shared_room(int n_tokens, int n_req, int n_groups, int kv_heads, int group, int dim) {
  return parts_bytes(n_tokens) + room_bytes(call_of(n_tokens, n_req, n_groups, kv_heads, group, dim), dim);
}

// q [n_tokens, heads, dim] with rows `q_row` elements apart; pages [num_pages][2][kv_heads][page_size][dim], pages `page_stride` elements apart; out dense.
IFB_EXPORT int ifb_attention_shared(const Packed* call) {
  const Packed& a = *call;
  if (a.n_tokens <= 0 || a.n_req <= 0) return IFB_OK;
  if (const int st = check(a, SH_ROWS, 4)) return st;
  Call c = call_of(a.n_tokens, a.n_req, a.n_groups, a.kv_heads, a.heads / a.kv_heads, a.dim);
  fill(c, a);
  room_at(c, a.dim, (char*)a.room + parts_bytes(a.n_tokens));
  const float *q = (const float*)a.q, *pages = (const float*)a.pages;
  const int st = a.dim <= 64    ? sh_main<float, 2>(c, q, a.q_row, pages, a.dim, a.stream)
                 : a.dim <= 96  ? sh_main<float, 3>(c, q, a.q_row, pages, a.dim, a.stream)
                 : a.dim <= 128 ? sh_main<float, 4>(c, q, a.q_row, pages, a.dim, a.stream)
                 : a.dim <= 192 ? sh_main<float, 6>(c, q, a.q_row, pages, a.dim, a.stream)
                                : sh_main<float, 8>(c, q, a.q_row, pages, a.dim, a.stream);
  return st ? st : join<float>(c, c, a.dim, a.stream);
}
