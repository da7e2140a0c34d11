// C-ABI entry points of the paged key / value cache (kernels in paged.h and paged_attention.h).
#include "paged_host.h"

using namespace ccq;

namespace
{
// Tokens per workgroup of the read back (and of the append, in paged_host.h): one up to 32 workgroups per CU, which then share their trips to memory.  MI355X, 32 / 8 heads, E4M3, one / these,
// us: append of 512 tokens 5.1 / 6.8, 2048 (6144 workgroups) 12.8 / 13.5, 8192 48.6 / 41.7; read of 2048 rows 4.7 / 5.5, 8192 (8192 workgroups) 12.0 / 10.9, 32000 54.6 / 43.2.
constexpr int READ_TOKENS = 8;
}    // namespace

int hip_qk_norm_rope_kv_paged_bf16(const hip_paged_kv* cache, const void* q, const void* k, const void* v, const void* q_norm_w, const void* k_norm_w, const void* cos_tab, const void* sin_tab,
                                   int n_positions, void* q_out, int n_q_heads, int n_tokens, int ldq, int ldk, int ldv, float epsilon)
{
    return launch_append<false>("qk_norm_rope_kv_paged", cache, q, k, v, q_norm_w, k_norm_w, cos_tab, sin_tab, n_positions, nullptr, 1, 0, nullptr, q_out, n_q_heads, n_tokens, ldq, ldk, ldv, epsilon);
}

int hip_kv_paged_read_bf16(const hip_paged_kv* cache, void* k_out, void* v_out, int n_tokens, long long token_stride, long long head_stride)
{
    PagedArgs a;
    if (!paged_args(cache, a) || n_tokens < 0 || !k_out || !v_out || !aligned(k_out, 16) || !aligned(v_out, 16)) { return -1; }
    if (token_stride % 8 != 0 || head_stride % 8 != 0 || token_stride < cache->head_dim || head_stride < cache->head_dim) { return -1; }
    const int per_wg = 256 * 8 / cache->head_dim;
    const int parts = (2 * a.n_kv + per_wg - 1) / per_wg;
    const long long blocks = (long long)n_tokens * parts;
    if (blocks > MOST_BLOCKS) { return -1; }
    if (n_tokens == 0) { return 0; }
    if (blocks < 32LL * cu_count())
    {
        const auto kernel = CCQ_PAGED_KERNEL(paged_read_kernel, cache, 1);
        kernel<<<(unsigned)blocks, 256, 0, stream()>>>(a, (uint16_t*)k_out, (uint16_t*)v_out, n_tokens, token_stride, head_stride);
    }
    else
    {
        const auto kernel = CCQ_PAGED_KERNEL(paged_read_kernel, cache, READ_TOKENS);
        kernel<<<(unsigned)((n_tokens + READ_TOKENS - 1) / READ_TOKENS * parts), 256, 0, stream()>>>(a, (uint16_t*)k_out, (uint16_t*)v_out, n_tokens, token_stride, head_stride);
    }
    return finish("kv_paged_read");
}

unsigned long long hip_attention_paged_workspace_bytes(const hip_paged_kv* cache, int n_q_heads, int n_tokens, int max_new, int max_ctx, int window, int n_sink)
{
    return attention_workspace_bytes(cache, n_q_heads, n_tokens, max_new, max_ctx, window, n_sink, false);
}

int hip_attention_paged_bf16(const hip_paged_kv* cache, const void* q, void* y, void* workspace, unsigned long long workspace_bytes, int n_q_heads, int n_tokens, int max_new, int max_ctx,
                             int window, int n_sink, int ldq, int ldy)
{
    return launch_attention<false>("attention_paged", cache, q, y, nullptr, 0, workspace, workspace_bytes, n_q_heads, n_tokens, max_new, max_ctx, window, n_sink, ldq, ldy);
}
