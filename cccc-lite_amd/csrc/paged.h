// A batch of sequences on a paged key / value cache: what the kernels know of it, and the kernels that write and read its rows.
// A row (a position of one kv head) is held as BF16, or as FP8 codes c with one exponent byte b: the value is c 2^(b - 127).
#pragma once
#include "quant_device.h"

namespace ccq
{

struct PagedArgs
{
    const uint8_t* k;               // pages [n_kv][page rows][dim]
    const uint8_t* v;
    const uint8_t* k_scale;         // pages [n_kv][page rows], FP8 only
    const uint8_t* v_scale;
    const int* table;               // [n_seqs][table_stride]
    const int* ctx_len;
    const int* seq_start;           // [n_seqs + 1]
    size_t page_stride, scale_stride;
    int n_pages, n_kv, n_seqs, table_stride;
    int shift;                      // page rows = 1 << shift, 16 or more
    int max_ctx;                    // rows a sequence may have: the table's, and the caller's limit
};

// Rows of a sequence in the cache, of its length as it is stored.
__device__ __forceinline__ int paged_rows(const PagedArgs& a, int ctx_len) { return max(min(ctx_len, a.max_ctx), 0); }

// Where activation rows t0 .. t0 + N - 1 belong: sequence (-1: to none), position, page (-1: none).  Called by whole waves with one t0: a lane per sequence,
// so one trip to memory for the first 64 and for each 256 more, then one each for the N rows' lengths and pages.  Ranges that are not in order name no sequence, or one whose
// range has t: a row index never leaves the range that was looked at.
template <int N>
struct PagedPlaces
{
    int s[N], pos[N], page[N];

    __device__ __forceinline__ PagedPlaces(const PagedArgs& a, int t0)
    {
#pragma unroll
        for (int n = 0; n < N; n++) { s[n] = -1; }
        auto count = [&](int i, int start) {
#pragma unroll
            for (int n = 0; n < N; n++) { s[n] += __builtin_popcountll(__ballot(i <= a.n_seqs && start <= t0 + n)); }
        };
        const int lane = threadIdx.x & 63;
        count(lane, a.seq_start[min(lane, a.n_seqs)]);
        for (int base = 64; base <= a.n_seqs; base += 256)
        {
            int start[4];
#pragma unroll
            for (int b = 0; b < 4; b++) { start[b] = a.seq_start[min(base + 64 * b + lane, a.n_seqs)]; }
#pragma unroll
            for (int b = 0; b < 4; b++) { count(base + 64 * b + lane, start[b]); }
        }
        int at[N], begin[N], end[N], rows[N];
#pragma unroll
        for (int n = 0; n < N; n++)
        {
            at[n] = min(max(s[n], 0), a.n_seqs - 1);
            begin[n] = a.seq_start[at[n]];
            end[n] = a.seq_start[at[n] + 1];
            rows[n] = a.ctx_len[at[n]];
        }
#pragma unroll
        for (int n = 0; n < N; n++)
        {
            if (at[n] != s[n] || begin[n] > t0 + n || end[n] <= t0 + n) { s[n] = -1; }
            pos[n] = paged_rows(a, rows[n]) - (end[n] - (t0 + n));
            page[n] = s[n] < 0 || pos[n] < 0 ? -1 : a.table[(size_t)at[n] * a.table_stride + (pos[n] >> a.shift)];
        }
#pragma unroll
        for (int n = 0; n < N; n++) { page[n] = page[n] < a.n_pages ? max(page[n], -1) : -1; }
    }
};

// Page of position pos >= 0, or -1.
__device__ __forceinline__ int paged_page(const PagedArgs& a, int s, int pos)
{
    const int page = a.table[(size_t)s * a.table_stride + (pos >> a.shift)];
    return page < a.n_pages ? page : -1;
}

// Row of kv head h at position pos of a page, counted from the page's first.
__device__ __forceinline__ int paged_row(const PagedArgs& a, int h, int pos) { return (h << a.shift) + (pos & ((1 << a.shift) - 1)); }

template <int TYPE>
constexpr int CODE_BYTES = TYPE == DT_BF16 ? 2 : 1;

// four codes of one dword -> BF16 times a power of two, exact
template <int TYPE>
__device__ __forceinline__ u32x2 fp8x4_to_bf16(uint32_t w, float scale)
{
    if constexpr (TYPE == DT_E4M3)
    {
        return u32x2{ __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)) };
    }
    else
    {
        return u32x2{ __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, true)) };
    }
}

template <int TYPE>
__device__ __forceinline__ uint32_t f32x4_to_fp8(float x0, float x1, float x2, float x3)
{
    int w = 0;
    if constexpr (TYPE == DT_E4M3)
    {
        w = __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, w, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, w, true);
    }
    else
    {
        w = __builtin_amdgcn_cvt_pk_bf8_f32(x0, x1, w, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(x2, x3, w, true);
    }
}

template <int LANES, class F>
__device__ __forceinline__ float reduce_lanes(float v, F f)
{
    v = f(v, dpp_f32<0xB1>(v));                                 // quad_perm [1,0,3,2]
    v = f(v, dpp_f32<0x4E>(v));                                 // quad_perm [2,3,0,1]
    v = f(v, dpp_f32<0x141>(v));                                // row_half_mirror
    if constexpr (LANES == 16) { v = f(v, dpp_f32<0x140>(v)); } // row_mirror
    return v;
}

struct PagedAppend
{
    const uint16_t *q, *k, *v, *q_norm_w, *k_norm_w, *cos_tab, *sin_tab;
    uint16_t* q_out;
    int n_q, n_tokens, n_positions;
    size_t ldq, ldk, ldv;
    float eps;
    const int* positions;           // given positions: [n_axes] rows of one per token
    const uint8_t* axis;            // of each pair of a head; nullptr: 0
    int n_axes;
    size_t position_stride;
};

__device__ __forceinline__ void unpack4(const u32x2 raw, float* f)
{
#pragma unroll
    for (int d = 0; d < 2; d++)
    {
        f[2 * d] = bits_to_f32(raw[d] << 16);
        f[2 * d + 1] = bits_to_f32(raw[d] & 0xFFFF0000u);
    }
}

__device__ __forceinline__ u32x2 pack4(const float* f)
{
    return u32x2{ f32_to_bf16_bits(f[0]) | f32_to_bf16_bits(f[1]) << 16, f32_to_bf16_bits(f[2]) | f32_to_bf16_bits(f[3]) << 16 };
}

// Norm, rotation and append of a head by DIM / 8 lanes: lane i holds elements 4 i .. + 3 of both halves of the head, so that the rotation needs no
// neighbour.  A lane takes the same head of TOKENS tokens: rows that do not hang on where their token belongs are asked for first, and the trips that tell
// it are shared.  AT: the positions of the rotation are given, on up to four axes; a lane's four pairs may lie on any of them.
// Bound by memory where tokens are many (4 prompts of 1500 to 2600 tokens, 32 / 8 heads, E5M2: 38 us, 4.6 TB/s), by the launch where they are few
// (16 tokens 4.1 us).  Grid: tokens / TOKENS x workgroups of 256 lanes over the n_q + 2 n_kv heads.
template <int TYPE, int DIM, int TOKENS, bool AT>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedArgs a, const PagedAppend p)
{
    constexpr int LANES = DIM / 8, PER_WG = 256 / LANES, TOP = TYPE == DT_E4M3 ? 8 : 15;
    constexpr float LARGEST = TYPE == DT_E4M3 ? 448.0f : 57344.0f;
    const int heads = p.n_q + 2 * a.n_kv, parts = (heads + PER_WG - 1) / PER_WG;
    const int t0 = blockIdx.x / parts * TOKENS, head = min(blockIdx.x % parts * PER_WG + (int)threadIdx.x / LANES, heads - 1), i = threadIdx.x % LANES;
    const bool spare = blockIdx.x % parts * PER_WG + threadIdx.x / LANES >= (unsigned)heads;
    const bool is_q = head < p.n_q, is_v = head >= p.n_q + a.n_kv;
    const int h = is_q ? head : is_v ? head - p.n_q - a.n_kv : head - p.n_q;
    const uint16_t* const src = (is_q ? p.q : is_v ? p.v : p.k) + (size_t)h * DIM + i * 4;
    const size_t ld = is_q ? p.ldq : is_v ? p.ldv : p.ldk;
    u32x2 raw[TOKENS][2];
#pragma unroll
    for (int n = 0; n < TOKENS; n++)
    {
        const uint16_t* const row = src + (size_t)min(t0 + n, p.n_tokens - 1) * ld;
        raw[n][0] = *(const u32x2*)row;
        raw[n][1] = *(const u32x2*)(row + DIM / 2);
    }
    const uint16_t* const nw = is_v ? nullptr : is_q ? p.q_norm_w : p.k_norm_w;
    float w[8] = {};
    if (nw)
    {
        unpack4(*(const u32x2*)(nw + i * 4), w);
        unpack4(*(const u32x2*)(nw + i * 4 + DIM / 2), w + 4);
    }
    u32x2 cs[TOKENS], sn[TOKENS];
    // AT: the tokens' positions, asked for in front of where they belong
    int given[TOKENS][AT ? 4 : 1];
    uint32_t axes = 0;
    if constexpr (AT)
    {
        axes = p.axis ? *(const uint32_t*)(p.axis + i * 4) : 0;             // of the lane's four pairs
#pragma unroll
        for (int n = 0; n < TOKENS; n++)
        {
#pragma unroll
            for (int x = 0; x < 4; x++) { given[n][x] = x < p.n_axes ? p.positions[(size_t)x * p.position_stride + min(t0 + n, p.n_tokens - 1)] : 0; }
        }
    }
    const PagedPlaces<TOKENS> at(a, t0);
    const bool turns = p.cos_tab && !is_v;
    if (AT && turns)
    {
        const bool alike = axes == (axes & 255u) * 0x01010101u;             // all four on one axis: 8 bytes of a row each of cosines and sines, else 2 bytes of four rows
        auto row = [&](int n, uint32_t axis) {
            const int pos = axis == 0 ? given[n][0] : axis == 1 ? given[n][AT ? 1 : 0] : axis == 2 ? given[n][AT ? 2 : 0] : given[n][AT ? 3 : 0];
            return (size_t)min(max(pos, 0), p.n_positions - 1) * (DIM / 2) + i * 4;
        };
#pragma unroll
        for (int n = 0; n < TOKENS; n++)
        {
            if (alike)
            {
                const size_t from = row(n, axes & 255u);
                cs[n] = *(const u32x2*)(p.cos_tab + from);
                sn[n] = *(const u32x2*)(p.sin_tab + from);
                continue;
            }
#pragma unroll
            for (int d = 0; d < 2; d++)
            {
                const size_t lo = row(n, axes >> (16 * d) & 255u) + 2 * d, hi = row(n, axes >> (16 * d + 8) & 255u) + 2 * d + 1;
                cs[n][d] = p.cos_tab[lo] | (uint32_t)p.cos_tab[hi] << 16;
                sn[n][d] = p.sin_tab[lo] | (uint32_t)p.sin_tab[hi] << 16;
            }
        }
    }
    if (turns && !AT)
    {
#pragma unroll
        for (int n = 0; n < TOKENS; n++)
        {
            const size_t from = (size_t)min(max(at.pos[n], 0), p.n_positions - 1) * (DIM / 2) + i * 4;
            cs[n] = *(const u32x2*)(p.cos_tab + from);
            sn[n] = *(const u32x2*)(p.sin_tab + from);
        }
    }
#pragma unroll
    for (int n = 0; n < TOKENS; n++)
    {
        const int t = t0 + n, pos = at.pos[n];
        bool out = !AT && p.cos_tab && pos >= p.n_positions;                // a position that no row of the tables has
        if constexpr (AT)
        {
#pragma unroll
            for (int x = 0; x < 4; x++) { out = out || given[n][x] < 0 || given[n][x] >= p.n_positions; }
        }
        if (at.s[n] < 0 || t >= p.n_tokens || pos < 0 || out || spare) { continue; }
        float x[8];
        unpack4(raw[n][0], x);
        unpack4(raw[n][1], x + 4);
        if (nw)
        {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) { sum += x[e] * x[e]; }
            sum = reduce_lanes<LANES>(sum, [](float u, float v) { return u + v; });
            const float invstd = rsqrtf(sum / (float)DIM + p.eps);
#pragma unroll
            for (int e = 0; e < 8; e++) { x[e] = x[e] * invstd * w[e]; }
        }
        if (turns)
        {
            float c[4], s[4];
            unpack4(cs[n], c);
            unpack4(sn[n], s);
#pragma unroll
            for (int e = 0; e < 4; e++)
            {
                const float lo = x[e], hi = x[e + 4];
                if (AT && (axes >> (8 * e) & 255u) >= (uint32_t)p.n_axes) { continue; }
                x[e] = lo * c[e] - hi * s[e];
                x[e + 4] = hi * c[e] + lo * s[e];
            }
        }
        if (is_q)
        {
            uint16_t* const dst = p.q_out + ((size_t)t * p.n_q + h) * DIM + i * 4;
            *(u32x2*)dst = pack4(x);
            *(u32x2*)(dst + DIM / 2) = pack4(x + 4);
            continue;
        }
        const int page = at.page[n];
        if (page < 0) { continue; }
        const size_t row = paged_row(a, h, pos);
        uint8_t* const dst = const_cast<uint8_t*>(is_v ? a.v : a.k) + page * a.page_stride + row * (DIM * CODE_BYTES<TYPE>);
        if constexpr (TYPE == DT_BF16)
        {
            *(u32x2*)(dst + i * 8) = pack4(x);
            *(u32x2*)(dst + i * 8 + DIM) = pack4(x + 4);
        }
        else
        {
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) { most = fmaxf(most, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.0f); }
            most = reduce_lanes<LANES>(most, [](float u, float v) { return fmaxf(u, v); });
            // most = m 2^k, 1 <= m < 2: both types' largest value is 1.75 2^TOP
            const uint32_t bits = f32_to_bits(most);
            int e2 = (int)(bits >> 23) - 127 - TOP + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
            e2 = min(max(e2, -100), 127 - TOP);
            const float by = bits_to_f32((uint32_t)(127 - e2) << 23);
#pragma unroll
            for (int e = 0; e < 8; e++)
            {
                const float y = x[e] * by;
                x[e] = fabsf(y) < INFINITY ? fminf(fmaxf(y, -LARGEST), LARGEST) : y;      // saturates at the largest exponent only
            }
            *(uint32_t*)(dst + i * 4) = f32x4_to_fp8<TYPE>(x[0], x[1], x[2], x[3]);
            *(uint32_t*)(dst + i * 4 + DIM / 2) = f32x4_to_fp8<TYPE>(x[4], x[5], x[6], x[7]);
            if (i == 0) { const_cast<uint8_t*>(is_v ? a.v_scale : a.k_scale)[page * a.scale_stride + row] = (uint8_t)(e2 + 127); }
        }
    }
}

// Rows back as BF16: DIM / 8 lanes per row of eight values each, the same row of TOKENS tokens per lane.  Bound like the append: 32000 rows E4M3
// 43 us, 4.5 TB/s; 301 rows 3.9 us.  Grid: tokens / TOKENS x workgroups of 256 lanes over the 2 n_kv rows of a token.
template <int TYPE, int DIM, int TOKENS>
__global__ __launch_bounds__(256) void paged_read_kernel(const PagedArgs a, uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out, int n_tokens, long long token_stride, long long head_stride)
{
    constexpr int LANES = DIM / 8, PER_WG = 256 / LANES, BYTES = 8 * CODE_BYTES<TYPE>;
    const int parts = (2 * a.n_kv + PER_WG - 1) / PER_WG;
    const int t0 = blockIdx.x / parts * TOKENS, of = blockIdx.x % parts * PER_WG + threadIdx.x / LANES, i = threadIdx.x % LANES;
    const PagedPlaces<TOKENS> at(a, t0);
    if (of >= 2 * a.n_kv) { return; }
    const bool is_v = of >= a.n_kv;
    const int h = is_v ? of - a.n_kv : of;
    u32x4 codes[TOKENS];
    uint32_t exponent[TOKENS];
#pragma unroll
    for (int n = 0; n < TOKENS; n++)
    {
        // a row without a page: any that is there
        const size_t page = max(at.page[n], 0), row = paged_row(a, h, max(at.pos[n], 0));
        const uint8_t* const src = (is_v ? a.v : a.k) + page * a.page_stride + row * (DIM * CODE_BYTES<TYPE>) + i * BYTES;
        if constexpr (TYPE == DT_BF16) { codes[n] = *(const u32x4*)src; }
        else
        {
            const u32x2 c = *(const u32x2*)src;
            codes[n] = u32x4{ c[0], c[1], 0, 0 };
            exponent[n] = (is_v ? a.v_scale : a.k_scale)[page * a.scale_stride + row];
        }
    }
#pragma unroll
    for (int n = 0; n < TOKENS; n++)
    {
        if (at.s[n] < 0 || t0 + n >= n_tokens) { continue; }
        u32x4 out = codes[n];
        if constexpr (TYPE != DT_BF16)
        {
            const float scale = bits_to_f32(exponent[n] << 23);
            const u32x2 lo = fp8x4_to_bf16<TYPE>(codes[n][0], scale), hi = fp8x4_to_bf16<TYPE>(codes[n][1], scale);
            out = u32x4{ lo[0], lo[1], hi[0], hi[1] };
        }
        if (at.page[n] < 0) { out = u32x4{ 0, 0, 0, 0 }; }
        *(u32x4*)((is_v ? v_out : k_out) + (t0 + n) * token_stride + h * head_stride + i * 8) = out;
    }
}

}    // namespace ccq
