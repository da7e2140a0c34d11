// Rows and pages of a paged key / value cache moved about, in all layers at once: what is kept of a sequence's new tokens, and batches that fork.
#pragma once
#include "paged.h"

namespace ccq
{

// The pools of up to this many layers travel with a launch.
constexpr int MOVE_LAYERS = 64;

struct PagedLayers
{
    uint8_t *k[MOVE_LAYERS], *v[MOVE_LAYERS], *k_scale[MOVE_LAYERS], *v_scale[MOVE_LAYERS];
    int n;
    int row;                        // bytes of a row of one kv head: 64, 128 or 256
};

// The sequence of a workgroup, n workgroups for each layer and side: turned by one from one to the next, so that a sequence with much to move is not always on the same XCD
// (workgroups go round them by eights, and so may sequences: MI355X, 64 sequences of which every second one is copied 35.6 us, not turned, for 25.8).
__device__ __forceinline__ int turned(unsigned block, int n) { return (int)((block % n + block / n) % n); }

struct PagedKeep
{
    const int *keep, *n_keep;
    int* ctx_out;
    int n_tokens, max_new;
};

// Rows of a sequence's kept tokens, KEEP_ROWS at a time and KEEP_UNITS times 256 pieces of 16 bytes, through registers.
// Kept indices ascend and none is below its place, so that a place is never a source of later rows: what a chunk reads is read before it writes, and nothing else has to
// wait.  MI355X, 36 layers of 8 heads of 128: one BF16 sequence 4.6 us, 32 E4M3 ones with one to nine kept rows 9.2 us.  Bound by the launch and four trips to memory in a row (places, pages, rows, and the way back).
// Grid: sequences x layers x (keys, values).
constexpr int KEEP_ROWS = 16, KEEP_UNITS = 8;

__global__ __launch_bounds__(256) void paged_keep_kernel(const PagedArgs a, const PagedLayers layers, const PagedKeep p)
{
    // where the chunk's rows come from and go to: page (-1: no move) and row of kv head 0
    __shared__ int from_page[KEEP_ROWS], from_row[KEEP_ROWS], to_page[KEEP_ROWS], to_row[KEEP_ROWS];
    const int of = blockIdx.x / a.n_seqs, s = turned(blockIdx.x, a.n_seqs), side = of % 2, layer = of / 2;
    const int begin = a.seq_start[s], end = a.seq_start[s + 1], rows = paged_rows(a, a.ctx_len[s]);
    int kept = p.n_keep[s];
    const bool mine = begin >= 0 && end <= p.n_tokens && begin < end && (long long)end - begin <= p.max_new;
    const int n = mine ? end - begin : 0, first = rows - n;
    kept = min(max(kept, 0), n);
    if (p.ctx_out && threadIdx.x == 0 && of == 0) { p.ctx_out[s] = max(first + kept, 0); }
    uint8_t* const pool = side ? layers.v[layer] : layers.k[layer];
    uint8_t* const scale = side ? layers.v_scale[layer] : layers.k_scale[layer];
    const int pieces = layers.row / 16, i = threadIdx.x / pieces % KEEP_ROWS, heads_at_once = 256 / pieces / KEEP_ROWS, h0 = threadIdx.x / pieces / KEEP_ROWS;
    const size_t piece = threadIdx.x % pieces * 16;
    for (int i0 = 0; i0 < kept; i0 += KEEP_ROWS)
    {
        if (threadIdx.x < KEEP_ROWS)
        {
            const int at = i0 + threadIdx.x, of = at < kept ? p.keep[begin + at] : 0;
            const int src = first + of, dst = first + at;
            int page = -1, place = -1;
            if (at < kept && of > at && of < n && dst >= 0)
            {
                page = paged_page(a, s, src);
                place = paged_page(a, s, dst);
            }
            from_page[threadIdx.x] = place < 0 ? -1 : page;
            to_page[threadIdx.x] = place;
            from_row[threadIdx.x] = paged_row(a, 0, max(src, 0));
            to_row[threadIdx.x] = paged_row(a, 0, max(dst, 0));
        }
        __syncthreads();
        const bool moves = from_page[i] >= 0;
        for (int h1 = 0; h1 < a.n_kv; h1 += KEEP_UNITS * heads_at_once)
        {
            u32x4 unit[KEEP_UNITS];
#pragma unroll
            for (int u = 0; u < KEEP_UNITS; u++)
            {
                const int h = h1 + u * heads_at_once + h0;
                if (moves && h < a.n_kv) { unit[u] = *(const u32x4*)(pool + from_page[i] * a.page_stride + (((size_t)h << a.shift) + from_row[i]) * layers.row + piece); }
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < KEEP_UNITS; u++)
            {
                const int h = h1 + u * heads_at_once + h0;
                if (moves && h < a.n_kv) { *(u32x4*)(pool + to_page[i] * a.page_stride + (((size_t)h << a.shift) + to_row[i]) * layers.row + piece) = unit[u]; }
            }
        }
        if (scale)
        {
            const int row = threadIdx.x % KEEP_ROWS;
            for (int h1 = 0; h1 < a.n_kv; h1 += 256 / KEEP_ROWS)
            {
                const int h = h1 + threadIdx.x / KEEP_ROWS;
                const bool moves = from_page[row] >= 0 && h < a.n_kv;
                uint8_t unit = 0;
                if (moves) { unit = scale[from_page[row] * a.scale_stride + ((size_t)h << a.shift) + from_row[row]]; }
                __syncthreads();
                if (moves) { scale[to_page[row] * a.scale_stride + ((size_t)h << a.shift) + to_row[row]] = unit; }
            }
        }
        __syncthreads();
    }
}

struct PagedFork
{
    const int *parent, *rows, *grow;
    const uint8_t* reserved;
    int *table_out, *ctx_out, *missing;
    int n_out;
    int* holder;                    // [n_pages] who holds a page: nobody, a sequence's number + 1 (as its last one, the lowest such), 0 (as a whole one, or reserved)
    int* free_pages;                // [n_pages] pages of nobody, lowest first
    int* base;                      // [n_out][2] new pages handed out to the sequences in front; whether the last page is a new one
    int* n_free;
};

constexpr int FORK_NOBODY = 0x7FFFFFFF, FORK_THREADS = 1024, FORK_AT_ONCE = 4;

// What sequence s of the new batch is to hold.
struct Forked
{
    const int* old;                 // its parent's pages
    int rows, total;                // rows taken over, and with those to come
    int whole, taken, all;          // pages taken over as whole ones, with a last one, and with new ones

    __device__ __forceinline__ Forked(const PagedArgs& a, const PagedFork& f, int s)
    {
        const int parent = f.parent[s], want = f.rows ? f.rows[s] : a.max_ctx, grow = f.grow[s];
        const bool has = parent >= 0 && parent < a.n_seqs;
        const int have = has ? paged_rows(a, a.ctx_len[parent]) : 0;
        rows = min(max(want, 0), have);
        total = (int)min((long long)rows + max(grow, 0), (long long)a.max_ctx);
        old = a.table + (size_t)(has ? parent : 0) * a.table_stride;
        whole = rows >> a.shift;
        const int more = (1 << a.shift) - 1;
        taken = (rows + more) >> a.shift;
        all = (total + more) >> a.shift;
    }
    __device__ __forceinline__ bool has_last() const { return taken > whole; }
};

__device__ __forceinline__ int fork_page(const PagedArgs& a, int page) { return page >= 0 && page < a.n_pages ? page : -1; }

// Sum of v over the threads in front of this one, and over all.
__device__ __forceinline__ int fork_scan(int v, int& all, int* lds)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int upto = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
    {
        const int other = __shfl_up(upto, d);
        upto += lane >= d ? other : 0;
    }
    __syncthreads();
    if (lane == 63) { lds[wave] = upto; }
    __syncthreads();
    int before = 0;
    all = 0;
    for (int w = 0; w < FORK_THREADS / 64; w++)
    {
        before += w < wave ? lds[w] : 0;
        all += lds[w];
    }
    return before + upto - v;
}

// Who holds each page, which are free, and how many new ones go to the sequences in front of each: one workgroup.  The holders of up to FORK_LDS_PAGES pages are in LDS (IN_LDS).
// A sequence's pages are gone through by 2^k neighbouring threads, as many as the table's rows have entries, so that short rows leave no thread without.  Bound by its chain of trips: MI355X,
// 4 sequences of 63 pages 4.0 us, 64 of up to 32 pages 7.0 us (with the holders in memory and fences between the steps 15 and 21).  The pool's pages are all cleared, and gone through up to the last one that is handed
// out: 64 sequences of 500 pages of 16 rows, one E4M3 layer, both launches, in a pool of 16384 pages (a common prefix of 450 pages per four sequences) 13 us, of 40000 (holders in memory) 66, of 200000 75, 104 with `reserved`.
constexpr int FORK_LDS_PAGES = 16384;

template <bool IN_LDS>
__global__ __launch_bounds__(FORK_THREADS) void paged_fork_kernel(const PagedArgs a, const PagedFork f)
{
    __shared__ int lds[FORK_THREADS / 64];
    __shared__ int lds_holder[IN_LDS ? FORK_LDS_PAGES : 1];
    auto clear = [&](int i, int v) {
        if constexpr (IN_LDS) { lds_holder[i] = v; }
        else { f.holder[i] = v; }
    };
    auto hold = [&](int i, int v) {
        if constexpr (IN_LDS) { atomicMin(lds_holder + i, v); }
        else { atomicMin(f.holder + i, v); }
    };
    auto holder = [&](int i) {
        if constexpr (IN_LDS) { return lds_holder[i]; }
        else { return __hip_atomic_load(f.holder + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
    };
    for (int i = threadIdx.x; i < a.n_pages; i += FORK_THREADS) { clear(i, f.reserved && f.reserved[i] ? 0 : FORK_NOBODY); }
    __syncthreads();
    const int log2 = min(32 - __builtin_clz(a.table_stride - 1 | 1), 6), group = 1 << log2, within = threadIdx.x & (group - 1);
    for (int s = threadIdx.x >> log2; s < f.n_out; s += FORK_THREADS >> log2)
    {
        const Forked mine(a, f, s);
        for (int i0 = within; i0 < mine.taken; i0 += FORK_AT_ONCE * group)
        {
            int page[FORK_AT_ONCE];
#pragma unroll
            for (int n = 0; n < FORK_AT_ONCE; n++) { page[n] = i0 + n * group < mine.taken ? mine.old[i0 + n * group] : -1; }
#pragma unroll
            for (int n = 0; n < FORK_AT_ONCE; n++)
            {
                if (fork_page(a, page[n]) >= 0) { hold(page[n], i0 + n * group < mine.whole ? 0 : s + 1); }
            }
        }
    }
    __syncthreads();
    int needed = 0;
    for (int s0 = 0; s0 < f.n_out; s0 += FORK_THREADS)
    {
        const int s = s0 + threadIdx.x;
        int need = 0, is_new = 0;
        if (s < f.n_out)
        {
            const Forked mine(a, f, s);
            const int last = mine.has_last() ? fork_page(a, mine.old[mine.whole]) : -1;
            is_new = last >= 0 && holder(last) != s + 1;
            need = mine.all - mine.taken + is_new;
            f.ctx_out[s] = mine.total;
        }
        int all;
        const int before = fork_scan(need, all, lds);
        if (s < f.n_out)
        {
            f.base[2 * s] = needed + before;
            f.base[2 * s + 1] = is_new;
        }
        needed += all;
    }
    int n_free = 0;
    for (int i0 = 0; i0 < a.n_pages && n_free < needed; i0 += FORK_THREADS)
    {
        const int i = i0 + threadIdx.x;
        const bool free = i < a.n_pages && holder(i) == FORK_NOBODY;
        int all;
        const int before = fork_scan(free ? 1 : 0, all, lds);
        if (free) { f.free_pages[n_free + before] = i; }
        n_free += all;
    }
    if (threadIdx.x == 0)
    {
        *f.missing = max(needed - n_free, 0);
        *f.n_free = n_free;
    }
}

constexpr int COPY_AT_ONCE = 8;

// The new tables (workgroups from n_copies on, 256 entries each of one sequence) and the rows of last pages that became a sequence's own: sequences x layers x (keys, values),
// pieces of 16 bytes, COPY_AT_ONCE per thread on their way at once.  Bound by memory: MI355X, 64 sequences, 28 copies in 32 layers of
// 8 heads of 128, E4M3, 125 MB read and written in 25.8 us, 4.9 TB/s; four BF16 sequences with one copy in 36 layers 4.8 us, the launch.
__global__ __launch_bounds__(256) void paged_fork_copy_kernel(const PagedArgs a, const PagedLayers layers, const PagedFork f, int n_copies)
{
    if ((int)blockIdx.x >= n_copies)
    {
        const int per_seq = (a.table_stride + 255) / 256, s = (blockIdx.x - n_copies) / per_seq, i = (blockIdx.x - n_copies) % per_seq * 256 + threadIdx.x;
        const Forked mine(a, f, s);
        const int base = f.base[2 * s], is_new = f.base[2 * s + 1], n_free = *f.n_free;
        if (i >= a.table_stride) { return; }
        int page = -1;
        if (i >= mine.taken ? i < mine.all : i == mine.whole && is_new)
        {
            const int at = base + (i >= mine.taken ? i - mine.taken + is_new : 0);
            page = at < n_free ? f.free_pages[at] : -1;
        }
        else if (i < mine.taken) { page = fork_page(a, mine.old[i]); }
        f.table_out[(size_t)s * a.table_stride + i] = page;
        return;
    }
    const int of = blockIdx.x / f.n_out, s = turned(blockIdx.x, f.n_out), side = of % 2, layer = of / 2;
    const int at = f.base[2 * s];
    if (f.base[2 * s + 1] == 0 || at >= *f.n_free) { return; }
    const Forked mine(a, f, s);
    const int from = mine.old[mine.whole], to = f.free_pages[at], rows = mine.rows - (mine.whole << a.shift);
    uint8_t* const pool = side ? layers.v[layer] : layers.k[layer];
    uint8_t* const scale = side ? layers.v_scale[layer] : layers.k_scale[layer];
    const int per_head = rows * (layers.row / 16), all = per_head * a.n_kv;
    const size_t head = (size_t)layers.row << a.shift;
    const uint8_t* const src = pool + from * a.page_stride;
    uint8_t* const dst = pool + to * a.page_stride;
    for (int i0 = threadIdx.x; i0 < all; i0 += COPY_AT_ONCE * 256)
    {
        u32x4 piece[COPY_AT_ONCE];
        size_t off[COPY_AT_ONCE];
#pragma unroll
        for (int n = 0; n < COPY_AT_ONCE; n++)
        {
            const int i = i0 + 256 * n, h = i / per_head;
            off[n] = h * head + (size_t)(i - h * per_head) * 16;
            if (i < all) { piece[n] = *(const u32x4*)(src + off[n]); }
        }
#pragma unroll
        for (int n = 0; n < COPY_AT_ONCE; n++)
        {
            if (i0 + 256 * n < all) { *(u32x4*)(dst + off[n]) = piece[n]; }
        }
    }
    if (scale)
    {
        for (int i = threadIdx.x; i < rows * a.n_kv; i += 256)
        {
            const size_t byte = ((size_t)(i / rows) << a.shift) + i % rows;
            scale[to * a.scale_stride + byte] = scale[from * a.scale_stride + byte];
        }
    }
}

}    // namespace ccq
