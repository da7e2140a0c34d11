// What the entry points of the paged cache share on the host: descriptors and their checks, how an attention call is cut into workgroups, its launches.
#pragma once
#include "../../include/cccc_hip_quant.h"
#include "paged_attention.h"
#include "runtime.h"
#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>

namespace ccq
{
constexpr long long MOST_BLOCKS = 0xFFFFFF;        // of 256 lanes: a grid has fewer than 2^32

inline bool aligned(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Whether two buffers of so many bytes have any in common (NULL: none).
inline bool overlap(const void* a, unsigned long long n_a, const void* b, unsigned long long n_b)
{
    return a && b && n_a && n_b && (uintptr_t)a < (uintptr_t)b + n_b && (uintptr_t)b < (uintptr_t)a + n_a;
}

// The descriptor as the kernels take it; false: refused.
inline bool paged_args(const hip_paged_kv* c, PagedArgs& a)
{
    if (!c || (c->type != CCCC_BFLOAT16 && c->type != CCCC_FP8_E4M3 && c->type != CCCC_FP8_E5M2) || (c->head_dim != 64 && c->head_dim != 128)) { return false; }
    if (c->n_kv_heads <= 0 || c->n_kv_heads > 1024 || c->n_pages <= 0 || c->n_seqs <= 0 || c->n_seqs > 65536 || c->table_stride <= 0) { return false; }
    if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)) != 0) { return false; }
    if (!c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16) || !c->page_table || !c->ctx_len || !c->seq_start) { return false; }
    if (!aligned(c->page_table, 4) || !aligned(c->ctx_len, 4) || !aligned(c->seq_start, 4)) { return false; }
    const bool fp8 = c->type != CCCC_BFLOAT16;
    const size_t rows = (size_t)c->n_kv_heads * c->page_size, dense = rows * c->head_dim * (fp8 ? 1 : 2);
    if (c->page_stride % 16 != 0 || (c->page_stride != 0 && c->page_stride < dense)) { return false; }
    if (fp8 && (!aligned(c->k_scale, 16) || !aligned(c->v_scale, 16))) { return false; }
    if (fp8 && (!c->k_scale || !c->v_scale || c->scale_stride % 16 != 0 || (c->scale_stride != 0 && c->scale_stride < rows))) { return false; }
    a.k = (const uint8_t*)c->k;
    a.v = (const uint8_t*)c->v;
    a.k_scale = (const uint8_t*)c->k_scale;
    a.v_scale = (const uint8_t*)c->v_scale;
    a.table = (const int*)c->page_table;
    a.ctx_len = (const int*)c->ctx_len;
    a.seq_start = (const int*)c->seq_start;
    a.page_stride = c->page_stride ? (size_t)c->page_stride : dense;
    a.scale_stride = c->scale_stride ? (size_t)c->scale_stride : rows;
    a.n_pages = c->n_pages;
    a.n_kv = c->n_kv_heads;
    a.n_seqs = c->n_seqs;
    a.table_stride = c->table_stride;
    a.shift = __builtin_ctz((unsigned)c->page_size);
    a.max_ctx = (int)std::min((long long)c->table_stride << a.shift, 1LL << 30);
    return true;
}

// KERNEL for the type and head length of a cache, with further template arguments.
#define CCQ_PAGED_KERNEL(KERNEL, c, ...)                                                                               \
    ((c)->head_dim == 64 ? CCQ_PAGED_TYPE(KERNEL, c, 64, __VA_ARGS__) : CCQ_PAGED_TYPE(KERNEL, c, 128, __VA_ARGS__))
#define CCQ_PAGED_TYPE(KERNEL, c, DIM, ...)                                                                            \
    ((c)->type == CCCC_BFLOAT16 ? KERNEL<DT_BF16, DIM, __VA_ARGS__> : (c)->type == CCCC_FP8_E4M3 ? KERNEL<DT_E4M3, DIM, __VA_ARGS__> : KERNEL<DT_E5M2, DIM, __VA_ARGS__>)

// Tokens per workgroup of the append: one up to 32 workgroups per CU, which then share their trips to memory (figures in paged.hip).
constexpr int APPEND_TOKENS = 4;

// AT: positions of the rotation as given.
template <bool AT>
int launch_append(const char* name, const hip_paged_kv* cache, const void* q, const void* k, const void* v, const void* q_norm_w, const void* k_norm_w, const void* cos_tab, const void* sin_tab, int n_positions,
                  const void* positions, int n_axes, long long position_stride, const void* axis, void* q_out, int n_q_heads, int n_tokens, int ldq, int ldk, int ldv, float epsilon)
{
    PagedArgs a;
    if (!paged_args(cache, a) || n_q_heads < 0 || n_q_heads > 65536 || n_tokens < 0) { return -1; }
    const int dim = cache->head_dim;
    if ((n_q_heads > 0 && (!q || !q_out)) || !k || !v || (q_norm_w == nullptr) != (k_norm_w == nullptr) || (cos_tab == nullptr) != (sin_tab == nullptr)) { return -1; }
    if (cos_tab && n_positions <= 0) { return -1; }
    for (const void* p : { q, k, v, q_norm_w, k_norm_w, cos_tab, sin_tab, (const void*)q_out })
    {
        if (!aligned(p, 16)) { return -1; }
    }
    if ((n_q_heads > 0 && (ldq % 8 != 0 || ldq < (long long)n_q_heads * dim)) || ldk % 8 != 0 || ldv % 8 != 0 || ldk < (long long)a.n_kv * dim || ldv < (long long)a.n_kv * dim) { return -1; }
    if (n_q_heads > 0 && q_out == q && n_tokens > 1 && ldq != (long long)n_q_heads * dim) { return -1; }       // a row's result would land on another's input
    if (AT && (!positions || !cos_tab || n_axes < 1 || n_axes > 4 || !aligned(positions, 4) || !aligned(axis, 4) || (n_axes > 1 && position_stride < n_tokens))) { return -1; }
    const int per_wg = 256 * 8 / dim;
    const int parts = (n_q_heads + 2 * a.n_kv + per_wg - 1) / per_wg;
    const long long blocks = (long long)n_tokens * parts;
    if (blocks > MOST_BLOCKS) { return -1; }
    if (n_tokens == 0) { return 0; }
    const PagedAppend p = { (const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (const uint16_t*)q_norm_w, (const uint16_t*)k_norm_w, (const uint16_t*)cos_tab, (const uint16_t*)sin_tab,
                            (uint16_t*)q_out, n_q_heads, n_tokens, n_positions, (size_t)ldq, (size_t)ldk, (size_t)ldv, epsilon, (const int*)positions, (const uint8_t*)axis, n_axes, (size_t)position_stride };
    if (blocks < 32LL * cu_count())
    {
        const auto kernel = CCQ_PAGED_KERNEL(paged_append_kernel, cache, 1, AT);
        kernel<<<(unsigned)blocks, 256, 0, stream()>>>(a, p);
    }
    else
    {
        const auto kernel = CCQ_PAGED_KERNEL(paged_append_kernel, cache, APPEND_TOKENS, AT);
        kernel<<<(unsigned)((n_tokens + APPEND_TOKENS - 1) / APPEND_TOKENS * parts), 256, 0, stream()>>>(a, p);
    }
    return finish(name);
}

// keys of a block of paged_attention_kernel's rows (RowsForm)
inline int keys_per_block(const hip_paged_kv* c) { return c->type == CCCC_BFLOAT16 && c->head_dim == 128 ? 32 : 64; }

inline bool attention_args(const hip_paged_kv* c, PagedArgs& a, int n_q_heads, int n_tokens, int& max_new, int max_ctx, int& window, int& n_sink)
{
    if (!paged_args(c, a) || n_q_heads <= 0 || n_q_heads % c->n_kv_heads != 0 || n_q_heads / c->n_kv_heads > 64) { return false; }
    if (n_tokens < 0 || max_new <= 0 || max_ctx <= 0 || window < 0 || n_sink < 0) { return false; }
    if ((long long)n_tokens * n_q_heads > MOST_BLOCKS) { return false; }
    a.max_ctx = std::min(a.max_ctx, max_ctx);
    // sums and differences of positions stay within 32 bits
    max_new = std::min(max_new, 1 << 24);
    n_sink = std::min(n_sink, a.max_ctx);
    window = window >= a.max_ctx ? 0 : window;          // all keys
    return true;
}
// How a call's rows are taken: in tiles, each over so many ranges of keys at most; as sequences of up to 16 rows per kv head, whose keys are shared out over
// so many workgroups (0: one each); or both.
struct Plan
{
    int tiles, tile_split;          // at most
    bool rows;
    int min_rows, row_slots, row_parts;
    size_t tile_bytes, row_bytes;   // of partial sums
    int piece_slots;                 // trees (find_piece): tiles counts their pieces, at most, and how many run at once per kv head
};

// Ranges of keys for tiles that are few workgroups.  A tile takes 5 us and 1.35 per block of 64 keys where a CU has one workgroup, 2.15 for two side by side (heads of
// 64: 0.6 of it); ranges add 10 us for the launch that adds them and for the start of more workgroups, and 0.3 per MB of FP32 sums written and read.  5 % to gain
// at least.  Measured with 1 / 2 / 4 / 8 / 16 ranges, 32 / 8 heads BF16: 512 tokens behind 3000 71.5 / 52.0 / 50.2, 1024 behind 500 37.2 / 46.0, 1024 behind 3000 80.1 / 83.7,
// 128 behind 3000 61.4 / 40.7 / 29.7 / 27.8 / 30.9, 64 behind 8000 - / - / 47.4 / 33.9 / 30.1, 512 from 0 18.2 / 20.1.
inline int tile_ranges(long long workgroups, int blocks, size_t outputs, int dim)
{
    const double cus = cu_count(), mb = (double)outputs * (dim + 2) * 4.0 * 1e-6;
    int best = 1;
    double least = 0.0;
    for (int n = 1; n <= 64 && n <= std::max(blocks / 4, 1); n++)
    {
        const double all = (double)workgroups * n, rounds = std::max(1.0, all / (2.0 * cus));
        const double time = 5.0 + std::ceil((double)blocks / n) * rounds * (all > cus ? 2.15 : 1.35) * (dim == 64 ? 0.6 : 1.0) + (n > 1 ? 10.0 + 0.3 * mb * n : 0.0);
        if (n == 1 || time < 0.95 * least)
        {
            best = n;
            least = time;
        }
    }
    return best;
}

// Workspace for each of the pieces per kv head that run at once: two, since tiles of little more than one range's keys are in two.  Every slot has them,
// whatever the call's lengths (8 kv heads of 128 on 256 CUs: 68 MB).
inline size_t piece_bytes(const PagedArgs& a, int dim) { return (size_t)2 * a.n_kv * 128 * (dim + 2) * 4; }

// False: more than a launch can have.
inline bool plan_attention(const PagedArgs& a, int keys_per_block, int n_q, int dim, int n_tokens, int max_new, int window, int n_sink, bool tree, Plan& plan)
{
    const int group = n_q / a.n_kv;
    const long long rows = (long long)n_tokens * group, slots = 2LL * cu_count();
    // Sequences of up to 16 rows per kv head have a form of their own, also beside longer ones -- unless every sequence has max_new tokens, as far as
    // their number tells.
    plan = { 0, 1, true, 0, 0, 0, 0, 0, 0 };
    const long long keys = window == 0 ? a.max_ctx : std::min<long long>(a.max_ctx, (long long)window + n_sink + max_new);
    if ((long long)std::min(max_new, n_tokens) * group > PA_ROWS)
    {
        plan.rows = group <= PA_ROWS && n_tokens < (long long)a.n_seqs * max_new;
        plan.min_rows = plan.rows ? PA_ROWS : 0;
        const long long cut = std::min<long long>(a.n_seqs, rows / (plan.min_rows + 1));       // sequences, at most
        const long long tiles = (rows - cut) / 128 + cut;
        if (tiles * a.n_kv * 64 > MOST_BLOCKS) { return false; }
        plan.tiles = (int)tiles;
        if (tree)
        {
            plan.piece_slots = (int)std::max<long long>(1, slots / a.n_kv);
            if ((tiles + plan.piece_slots) * a.n_kv * 64 > MOST_BLOCKS) { return false; }
            plan.tile_bytes = 16 + plan.piece_slots * piece_bytes(a, dim);
        }
        else
        {
            plan.tile_split = tile_ranges(tiles * a.n_kv, (int)((keys + PA_TILE_KEYS - 1) / PA_TILE_KEYS), (size_t)n_tokens * n_q, dim);
            plan.tile_bytes = plan.tile_split > 1 ? ((size_t)n_tokens * n_q * plan.tile_split * (dim + 2) * 4 + 15) & ~(size_t)15 : 0;
        }
    }
    if (plan.rows)
    {
        // shares of four blocks (Parts): of a sequence at most, with a block at either end and one more for the first keys in part; all fit 32 bits
        const long long shares = (keys / keys_per_block + 3 + 3) / 4 + 1, all = shares * a.n_seqs, part = keys_per_block == 32 ? 2 : 1;
        const long long at_once = std::max<long long>(1, slots / a.n_kv);
        if (all > 0x3FFFFFFFLL || (a.n_seqs + 3 * at_once + 1) * a.n_kv * 2 > MOST_BLOCKS) { return false; }
        if (a.n_seqs > PA_CUT_SEQS) { return true; }
        plan.row_slots = (int)at_once;
        plan.row_parts = (int)(a.n_seqs + std::max<long long>(1, std::min(3 * at_once, all / part)));
        plan.row_bytes = ((size_t)plan.row_parts * a.n_kv * (PA_ROWS * (dim + 2) * 4 + 8) + 15) & ~(size_t)15;
    }
    return true;
}

// A name for a call's counters that no other call has: what lies in a workspace before is not taken for counts of this one.
inline unsigned long long name_call()
{
    static std::atomic<unsigned long long> next{ (unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count() * 0x9E3779B97F4A7C15ull };
    unsigned long long name;
    do { name = next.fetch_add(0x9E3779B97F4A7C15ull) >> 16; } while (name == 0);
    return name;
}

inline unsigned long long attention_workspace_bytes(const hip_paged_kv* cache, int n_q_heads, int n_tokens, int max_new, int max_ctx, int window, int n_sink, bool tree)
{
    PagedArgs a;
    if (!attention_args(cache, a, n_q_heads, n_tokens, max_new, max_ctx, window, n_sink) || n_tokens == 0) { return 0; }
    Plan plan;
    return plan_attention(a, keys_per_block(cache), n_q_heads, cache->head_dim, n_tokens, max_new, window, n_sink, tree, plan) ? plan.tile_bytes + plan.row_bytes : 0;
}

template <bool TREE>
int launch_attention(const char* name, const hip_paged_kv* cache, const void* q, void* y, const unsigned long long* seen, long long seen_stride, void* workspace, unsigned long long workspace_bytes,
                     int n_q_heads, int n_tokens, int max_new, int max_ctx, int window, int n_sink, int ldq, int ldy)
{
    PagedArgs a;
    if (!attention_args(cache, a, n_q_heads, n_tokens, max_new, max_ctx, window, n_sink)) { return -1; }
    if (!q || !y || !aligned(q, 16) || !aligned(y, 16) || !aligned(workspace, 16) || (workspace == nullptr && workspace_bytes != 0)) { return -1; }
    const int dim = cache->head_dim;
    const long long width = (long long)n_q_heads * dim;
    if (ldq % 8 != 0 || ldy % 8 != 0 || ldq < width || ldy < width) { return -1; }
    if (TREE && (!seen || !aligned(seen, 8) || seen_stride < (max_new + 63) / 64)) { return -1; }
    if (n_tokens == 0) { return 0; }
    if (y == q) { return -1; }
    Plan plan;
    if (!plan_attention(a, keys_per_block(cache), n_q_heads, dim, n_tokens, max_new, window, n_sink, TREE, plan)) { return -1; }
    // too little workspace: tiles and sequences in one piece each, tiles of trees in fewer
    if (workspace_bytes < plan.tile_bytes + plan.row_bytes)
    {
        plan.tile_split = 1;
        plan.tile_bytes = 0;
        if (workspace_bytes < plan.row_bytes) { plan.row_parts = 0; }
        const size_t rest = workspace_bytes - (plan.row_parts ? plan.row_bytes : 0);
        plan.piece_slots = plan.piece_slots == 0 || rest < 16 ? 0 : (int)((rest - 16) / piece_bytes(a, dim));
    }
    const int most_added = TREE ? std::min(plan.tiles, plan.piece_slots) : plan.tiles;         // tiles in several ranges
    plan.tiles += plan.piece_slots;
    const long long tiles = (long long)plan.tiles * a.n_kv * plan.tile_split, parts = plan.rows ? (long long)(plan.row_parts ? plan.row_parts : a.n_seqs) * a.n_kv : 0;
    // the workspace: the parts' words, sums and statistics, then the tiles'
    const size_t words = (size_t)plan.row_parts * a.n_kv;
    char* const part_sums = (char*)workspace + words * 8;
    const PagedAttention p = { (const uint16_t*)q, (uint16_t*)y, (float*)((char*)workspace + (plan.row_parts ? plan.row_bytes : 0) + (TREE ? 16 : 0)), (size_t)ldq, (size_t)ldy, n_q_heads, n_q_heads / a.n_kv,
                               n_tokens, max_new, window, n_sink, plan.tiles, plan.tile_split, plan.row_slots, plan.row_parts, (float*)part_sums, (unsigned long long*)workspace,
                               plan.row_parts ? name_call() : 0, plan.min_rows, tiles <= 2LL * cu_count() ? 1 : 0, 1.4426950408889634f / sqrtf((float)dim), seen, (size_t)seen_stride, plan.piece_slots };
    const auto kernel = CCQ_PAGED_KERNEL(paged_attention_kernel, cache, TREE);
    kernel<<<(unsigned)(tiles + parts), 256, 0, stream()>>>(a, p);
    if (plan.tile_split > 1 || plan.piece_slots > 0)
    {
        const unsigned blocks = (unsigned)(most_added * a.n_kv * 8);
        if (dim == 64) { paged_attention_combine_kernel<64, TREE><<<blocks, 256, 0, stream()>>>(a, p); }
        else { paged_attention_combine_kernel<128, TREE><<<blocks, 256, 0, stream()>>>(a, p); }
    }
    return finish(name);
}

}    // namespace ccq
