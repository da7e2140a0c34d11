// C-ABI entry points that move rows and pages of a paged key / value cache in all layers (kernels in paged_moves.h).
#include "paged_host.h"
#include "paged_moves.h"
#include <iterator>

using namespace ccq;

namespace
{
// The layers' common descriptor; false: refused, or not alike.
bool layers_args(const hip_paged_kv* caches, int n_layers, PagedArgs& a)
{
    if (!caches || n_layers <= 0 || n_layers > 65536 || !paged_args(caches, a)) { return false; }
    for (int i = 1; i < n_layers; i++)
    {
        const hip_paged_kv &c = caches[i], &first = caches[0];
        PagedArgs other;
        if (!paged_args(&c, other) || c.type != first.type || c.head_dim != first.head_dim || c.n_kv_heads != first.n_kv_heads || c.page_size != first.page_size || c.n_pages != first.n_pages ||
            c.n_seqs != first.n_seqs || c.table_stride != first.table_stride || c.page_stride != first.page_stride || c.scale_stride != first.scale_stride || c.page_table != first.page_table ||
            c.ctx_len != first.ctx_len || c.seq_start != first.seq_start)
        {
            return false;
        }
    }
    return true;
}

// Layers from `first` on that one launch takes: 64 of up to 2 * 65536 workgroups each are half of what a grid can have.
PagedLayers some_layers(const hip_paged_kv* caches, int first, int n_layers)
{
    PagedLayers l = {};
    l.n = std::min(n_layers - first, MOVE_LAYERS);
    l.row = caches->head_dim * (caches->type == CCCC_BFLOAT16 ? 2 : 1);
    for (int i = 0; i < l.n; i++)
    {
        const hip_paged_kv& c = caches[first + i];
        l.k[i] = (uint8_t*)c.k;
        l.v[i] = (uint8_t*)c.v;
        l.k_scale[i] = c.type == CCCC_BFLOAT16 ? nullptr : (uint8_t*)c.k_scale;
        l.v_scale[i] = c.type == CCCC_BFLOAT16 ? nullptr : (uint8_t*)c.v_scale;
    }
    return l;
}

size_t padded(size_t bytes) { return (bytes + 15) & ~(size_t)15; }
}    // namespace

int hip_kv_paged_keep(const hip_paged_kv* caches, int n_layers, const void* keep, const void* n_keep, int n_tokens, int max_new, void* ctx_out)
{
    PagedArgs a;
    if (!layers_args(caches, n_layers, a) || !keep || !n_keep || n_tokens < 0 || max_new <= 0) { return -1; }
    if (!aligned(keep, 4) || !aligned(n_keep, 4) || !aligned(ctx_out, 4)) { return -1; }
    // the lengths are written while other workgroups, and launches for further layers, read these
    const unsigned long long n = 4ull * a.n_seqs;
    if (overlap(ctx_out, n, keep, 4ull * n_tokens) || overlap(ctx_out, n, n_keep, n) || overlap(ctx_out, n, a.ctx_len, n) || overlap(ctx_out, n, a.seq_start, n + 4) ||
        overlap(ctx_out, n, a.table, n * a.table_stride))
    {
        return -1;
    }
    if (n_tokens == 0 && !ctx_out) { return 0; }
    const long long per_layer = 2LL * a.n_seqs;
    for (int first = 0; first < n_layers;)
    {
        const PagedLayers layers = some_layers(caches, first, n_layers);
        const PagedKeep p = { (const int*)keep, (const int*)n_keep, first == 0 ? (int*)ctx_out : nullptr, n_tokens, max_new };
        paged_keep_kernel<<<(unsigned)(per_layer * layers.n), 256, 0, stream()>>>(a, layers, p);
        first += layers.n;
    }
    return finish("kv_paged_keep");
}

unsigned long long hip_kv_paged_fork_workspace_bytes(const hip_paged_kv* caches, int n_layers, int n_out)
{
    PagedArgs a;
    if (!layers_args(caches, n_layers, a) || n_out <= 0 || n_out > 65536 || (long long)n_out * a.table_stride > 0x3FFFFFFFLL) { return 0; }
    return 16 + padded((size_t)n_out * 8) + 2 * padded((size_t)a.n_pages * 4);
}

int hip_kv_paged_fork(const hip_paged_kv* caches, int n_layers, int n_out, const void* parent, const void* rows, const void* grow, const void* reserved, void* table_out, void* ctx_out, void* missing,
                      void* workspace, unsigned long long workspace_bytes)
{
    PagedArgs a;
    if (!layers_args(caches, n_layers, a) || n_out <= 0 || n_out > 65536 || !parent || !grow || !table_out || !ctx_out || !missing || !workspace) { return -1; }
    for (const void* p : { parent, rows, grow, (const void*)table_out, (const void*)ctx_out, (const void*)missing })
    {
        if (!aligned(p, 4)) { return -1; }
    }
    const unsigned long long need = hip_kv_paged_fork_workspace_bytes(caches, n_layers, n_out);
    if ((long long)n_out * a.table_stride > 0x3FFFFFFFLL || !aligned(workspace, 16) || workspace_bytes < need) { return -1; }
    // what a launch writes, the next one and other workgroups still read beside
    struct Buffer
    {
        const void* at;
        unsigned long long bytes;
    };
    const unsigned long long n = 4ull * n_out, n_old = 4ull * a.n_seqs;
    const Buffer buffers[] = { { table_out, n * a.table_stride }, { ctx_out, n }, { missing, 4 }, { workspace, need },       // written
                               { parent, n }, { rows, n }, { grow, n }, { reserved, (unsigned long long)a.n_pages }, { a.table, n_old * a.table_stride }, { a.ctx_len, n_old } };
    for (int i = 0; i < 4; i++)
    {
        for (const Buffer* b = buffers + i + 1; b != std::end(buffers); b++)
        {
            if (overlap(buffers[i].at, buffers[i].bytes, b->at, b->bytes)) { return -1; }
        }
    }
    char* at = (char*)workspace;
    PagedFork f = { (const int*)parent, (const int*)rows, (const int*)grow, (const uint8_t*)reserved, (int*)table_out, (int*)ctx_out, (int*)missing, n_out };
    f.n_free = (int*)at;
    at += 16;
    f.base = (int*)at;
    at += padded((size_t)n_out * 8);
    f.holder = (int*)at;
    at += padded((size_t)a.n_pages * 4);
    f.free_pages = (int*)at;
    if (a.n_pages <= FORK_LDS_PAGES) { paged_fork_kernel<true><<<1, FORK_THREADS, 0, stream()>>>(a, f); }
    else { paged_fork_kernel<false><<<1, FORK_THREADS, 0, stream()>>>(a, f); }
    const long long per_layer = 2LL * n_out, tables = (long long)n_out * ((a.table_stride + 255) / 256);
    for (int first = 0; first < n_layers;)
    {
        const PagedLayers layers = some_layers(caches, first, n_layers);
        const unsigned n_copies = (unsigned)(per_layer * layers.n);
        paged_fork_copy_kernel<<<n_copies + (first == 0 ? (unsigned)tables : 0), 256, 0, stream()>>>(a, layers, f, (int)n_copies);
        first += layers.n;
    }
    return finish("kv_paged_fork");
}
