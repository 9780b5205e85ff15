// Attention of drafted tokens that form a tree over a paged cache: each sees what is in front of the tree, its ancestors and itself.
#include "paged_attn.h"

extern "C" {

size_t ftk_paged_tree_attn_workspace_bytes(const ftk_kv_pages* pages, const ftk_kv_batch* batch, int heads, int window, int max_queries, int max_keys) {
  return ftk::attend_workspace_bytes(pages, batch, heads, window, max_queries, max_keys, true);
}

int ftk_paged_tree_attn(const void* q, int type, long long q_token_stride, long long q_head_stride, const ftk_kv_pages* pages, const ftk_kv_batch* batch,
                        const int* parents, void* o, float* lse, int heads, float scale, int window, int max_queries, int max_keys, void* workspace,
                        size_t workspace_bytes, ftk_stream_t stream) {
  return ftk::attend<true>("ftk_paged_tree_attn", q, type, q_token_stride, q_head_stride, pages, batch, parents, o, lse, heads, scale, 1, window, max_queries, max_keys,
                           workspace, workspace_bytes, stream);
}

}  // extern "C"
