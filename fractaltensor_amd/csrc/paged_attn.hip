// Attention of new tokens over a paged cache: prompts, chunks, drafts and single tokens, each of which sees what is in front of it.
#include "paged_attn.h"

extern "C" {

size_t ftk_paged_attn_workspace_bytes(const ftk_kv_pages* pages, const ftk_kv_batch* batch, int heads, int window, int max_queries, int max_keys) {
  return ftk::attend_workspace_bytes(pages, batch, heads, window, max_queries, max_keys, false);
}

int ftk_paged_attn(const void* q, int type, long long q_token_stride, long long q_head_stride, const ftk_kv_pages* pages, const ftk_kv_batch* batch,
                   void* o, float* lse, int heads, float scale, int causal, int window, int max_queries, int max_keys, void* workspace,
                   size_t workspace_bytes, ftk_stream_t stream) {
  return ftk::attend<false>("ftk_paged_attn", q, type, q_token_stride, q_head_stride, pages, batch, nullptr, o, lse, heads, scale, causal, window, max_queries, max_keys,
                            workspace, workspace_bytes, stream);
}

}  // extern "C"
