// Attention over shared pages in float32: every owner by the kernel of attention_shared_simt.cuh.
#include "attention_shared_simt.cuh"

// Bytes of room for a call's sums.
IFB_EXPORT long long ifb_attention_shared_room(int n_tokens, int n_req, int n_groups, int kv_heads, int group, int dim) {
  return parts_bytes(n_tokens) + room_bytes(sh_call(n_tokens, n_req, n_groups, kv_heads, group, EVERY), dim);
}

// q [n_tokens, heads, dim] with rows `q_row` elements apart; pages [num_pages][2][kv_heads][page_size][dim], pages `page_stride` elements apart; out dense.
IFB_EXPORT int ifb_attention_shared(const float* q, long long q_row, const float* pages, long long page_stride, long long num_pages,
                                    const int* block_tables, long long bt_stride, int table_pages, const int* cu_q, const int* seq_lens,
                                    const int* cu_groups, const int* shared_lens, float* out, void* room, int* err, int n_tokens, int n_req, int n_groups,
                                    int heads, int kv_heads, int dim, int page_size, float scale, int window, cudaStream_t stream) {
  if (n_tokens <= 0 || n_req <= 0) return IFB_OK;
  if (kv_heads < 1 || heads % kv_heads || heads / kv_heads > SH_ROWS || dim < 4 || dim > 256 || dim % 4 || n_groups < 0 ||
      n_req + n_groups > MAX_OWNERS || page_size < 1 || num_pages < 1)
    return IFB_ERR_SIZE;
  if ((((uintptr_t)q | (uintptr_t)pages) & 15) || q_row % 4 || page_stride % 4 || ((uintptr_t)room & 255)) return IFB_ERR_ALIGN;
  if (window < 0 || !err) return IFB_ERR_ARG;
  Call c = sh_call(n_tokens, n_req, n_groups, kv_heads, heads / kv_heads, EVERY);
  c.block_tables = block_tables; c.cu_q = cu_q; c.seq_lens = seq_lens; c.cu_groups = cu_groups; c.shared_lens = shared_lens;
  c.bt_stride = bt_stride; c.num_pages = num_pages; c.page_stride = page_stride;
  c.table_pages = table_pages; c.page_size = page_size; c.window = window;
  c.scale_log2 = scale * 1.4426950408889634f;
  c.err = err;
  c.out = out;
  c.parts = (int4*)room;
  room_at(c, dim, (char*)room + parts_bytes(n_tokens));
  const int st = dim <= 64    ? sh_main<float, 8>(c, c, q, q_row, pages, dim, true, stream)
                 : dim <= 128 ? sh_main<float, 16>(c, c, q, q_row, pages, dim, true, stream)
                              : sh_main<float, 32>(c, c, q, q_row, pages, dim, true, stream);
  return st ? st : join<float>(c, c, dim, stream);
}
