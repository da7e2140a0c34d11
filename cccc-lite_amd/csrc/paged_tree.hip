// C-ABI entry points for new tokens that form trees, or whose positions lie on several axes (kernels in paged.h and paged_attention.h).
#include "paged_host.h"

using namespace ccq;

int hip_qk_norm_rope_kv_paged_at_bf16(const hip_paged_kv* cache, const void* q, const void* k, const void* v, const void* q_norm_w, const void* k_norm_w, const void* cos_tab, const void* sin_tab,
                                      int n_positions, const void* positions, int n_axes, long long position_stride, const void* axis, void* q_out, int n_q_heads, int n_tokens, int ldq, int ldk, int ldv,
                                      float epsilon)
{
    return launch_append<true>("qk_norm_rope_kv_paged_at", cache, q, k, v, q_norm_w, k_norm_w, cos_tab, sin_tab, n_positions, positions, n_axes, position_stride, axis, q_out, n_q_heads, n_tokens, ldq,
                               ldk, ldv, epsilon);
}

unsigned long long hip_attention_paged_tree_workspace_bytes(const hip_paged_kv* cache, int n_q_heads, int n_tokens, int max_new, int max_ctx, int window, int n_sink)
{
    return attention_workspace_bytes(cache, n_q_heads, n_tokens, max_new, max_ctx, window, n_sink, true);
}

int hip_attention_paged_tree_bf16(const hip_paged_kv* cache, const void* q, void* y, const void* seen, long long seen_stride, void* workspace, unsigned long long workspace_bytes, int n_q_heads,
                                  int n_tokens, int max_new, int max_ctx, int window, int n_sink, int ldq, int ldy)
{
    return launch_attention<true>("attention_paged_tree", cache, q, y, (const unsigned long long*)seen, seen_stride, workspace, workspace_bytes, n_q_heads, n_tokens, max_new, max_ctx, window, n_sink,
                                  ldq, ldy);
}
