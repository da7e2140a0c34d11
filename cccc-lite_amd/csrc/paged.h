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

// Sequence of activation row t, or -1.  Called by whole waves with one t: a lane per sequence, so one trip to memory per 64 of them.
// Ranges that are not in order name no sequence, or one whose range has t: a row index never leaves the range that was looked at.
__device__ __forceinline__ int paged_sequence(const PagedArgs& a, int t)
{
    int s = -1;
    for (int base = 0; base <= a.n_seqs; base += 64)
    {
        const int i = base + (threadIdx.x & 63);
        s += __builtin_popcountll(__ballot(i <= a.n_seqs && a.seq_start[i] <= t));
    }
    if (s < 0 || s >= a.n_seqs || a.seq_start[s] > t || a.seq_start[s + 1] <= t) { return -1; }
    return s;
}

// Rows of a sequence in the cache.
__device__ __forceinline__ int paged_rows(const PagedArgs& a, int s) { return min(a.ctx_len[s], a.max_ctx); }

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

// Norm, rotation and append of one head of one token by DIM / 8 lanes: lane i holds elements 4 i .. + 3 of both halves of the head, so that the
// rotation needs no neighbour.  Grid: tokens x workgroups of 256 lanes over the n_q + 2 n_kv heads.
template <int TYPE, int DIM>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedArgs a, const PagedAppend p)
{
    constexpr int LANES = DIM / 8, PER_WG = 256 / LANES, TOP = TYPE == DT_E4M3 ? 8 : 15;
    constexpr float LARGEST = TYPE == DT_E4M3 ? 448.0f : 57344.0f;
    const int heads = p.n_q + 2 * a.n_kv, parts = (heads + PER_WG - 1) / PER_WG;
    const int t = blockIdx.x / parts, head = blockIdx.x % parts * PER_WG + threadIdx.x / LANES, i = threadIdx.x % LANES;
    const int s = paged_sequence(a, t);
    if (s < 0) { return; }
    const int pos = paged_rows(a, s) - (a.seq_start[s + 1] - t);
    if (pos < 0 || (p.cos_tab && pos >= p.n_positions) || head >= heads) { return; }
    const bool is_q = head < p.n_q, is_v = head >= p.n_q + a.n_kv;
    const int h = is_q ? head : is_v ? head - p.n_q - a.n_kv : head - p.n_q;
    const uint16_t* const src = (is_q ? p.q + (size_t)t * p.ldq : is_v ? p.v + (size_t)t * p.ldv : p.k + (size_t)t * p.ldk) + (size_t)h * DIM + i * 4;
    float x[8];
    unpack4(*(const u32x2*)src, x);
    unpack4(*(const u32x2*)(src + DIM / 2), x + 4);
    const uint16_t* const nw = is_v ? nullptr : is_q ? p.q_norm_w : p.k_norm_w;
    if (nw)
    {
        float w[8], sum = 0.0f;
        unpack4(*(const u32x2*)(nw + i * 4), w);
        unpack4(*(const u32x2*)(nw + i * 4 + DIM / 2), w + 4);
#pragma unroll
        for (int e = 0; e < 8; e++) { sum += x[e] * x[e]; }
        sum = reduce_lanes<LANES>(sum, [](float u, float v) { return u + v; });
        const float invstd = rsqrtf(sum / (float)DIM + p.eps);
#pragma unroll
        for (int e = 0; e < 8; e++) { x[e] = x[e] * invstd * w[e]; }
    }
    if (p.cos_tab && !is_v)
    {
        float c[4], sn[4];
        unpack4(*(const u32x2*)(p.cos_tab + (size_t)pos * (DIM / 2) + i * 4), c);
        unpack4(*(const u32x2*)(p.sin_tab + (size_t)pos * (DIM / 2) + i * 4), sn);
#pragma unroll
        for (int e = 0; e < 4; e++)
        {
            const float lo = x[e], hi = x[e + 4];
            x[e] = lo * c[e] - hi * sn[e];
            x[e + 4] = hi * c[e] + lo * sn[e];
        }
    }
    if (is_q)
    {
        uint16_t* const dst = p.q_out + ((size_t)t * p.n_q + h) * DIM + i * 4;
        *(u32x2*)dst = pack4(x);
        *(u32x2*)(dst + DIM / 2) = pack4(x + 4);
        return;
    }
    const int page = paged_page(a, s, pos);
    if (page < 0) { return; }
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

// Rows back as BF16: DIM / 8 lanes per row of eight values each.  Grid: tokens x workgroups of 256 lanes over the 2 n_kv rows of a token.
template <int TYPE, int DIM>
__global__ __launch_bounds__(256) void paged_read_kernel(const PagedArgs a, uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out, long long token_stride, long long head_stride)
{
    constexpr int LANES = DIM / 8, PER_WG = 256 / LANES;
    const int parts = (2 * a.n_kv + PER_WG - 1) / PER_WG;
    const int t = blockIdx.x / parts, at = blockIdx.x % parts * PER_WG + threadIdx.x / LANES, i = threadIdx.x % LANES;
    const int s = paged_sequence(a, t);
    if (s < 0 || at >= 2 * a.n_kv) { return; }
    const bool is_v = at >= a.n_kv;
    const int h = is_v ? at - a.n_kv : at;
    const int pos = paged_rows(a, s) - (a.seq_start[s + 1] - t);
    const int page = pos < 0 ? -1 : paged_page(a, s, pos);
    u32x4 out = { 0, 0, 0, 0 };
    if (page >= 0)
    {
        const size_t row = paged_row(a, h, pos);
        const uint8_t* const src = (is_v ? a.v : a.k) + page * a.page_stride + row * (DIM * CODE_BYTES<TYPE>) + i * 8 * CODE_BYTES<TYPE>;
        if constexpr (TYPE == DT_BF16) { out = *(const u32x4*)src; }
        else
        {
            const u32x2 codes = *(const u32x2*)src;
            const float scale = bits_to_f32((uint32_t)(is_v ? a.v_scale : a.k_scale)[page * a.scale_stride + row] << 23);
            const u32x2 lo = fp8x4_to_bf16<TYPE>(codes[0], scale), hi = fp8x4_to_bf16<TYPE>(codes[1], scale);
            out = u32x4{ lo[0], lo[1], hi[0], hi[1] };
        }
    }
    *(u32x4*)((is_v ? v_out : k_out) + t * token_stride + h * head_stride + i * 8) = out;
}

}    // namespace ccq
