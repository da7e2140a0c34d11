// Causal attention of the new tokens of a batch of sequences over their pages.
#pragma once
#include "paged.h"

namespace ccq
{

struct PagedAttention
{
    const uint16_t* q;
    uint16_t* y;
    size_t ldq, ldy;
    int n_q, group, n_tokens, max_new, window, n_sink;
    float scale;
};

// Element d of a cached row, in FP32.
template <int TYPE>
__device__ __forceinline__ float paged_element(const uint8_t* row, int d, float scale)
{
    if constexpr (TYPE == DT_BF16) { return bf16_bits_to_f32(((const uint16_t*)row)[d]); }
    else { return (TYPE == DT_E4M3 ? e4m3_to_f32(row[d]) : e5m2_to_f32(row[d])) * scale; }
}

// One wave per (token, query head), a lane per key for the scores and one or two dims per lane for the products, 64 keys at a time with a running
// maximum and sum.
template <int TYPE, int DIM>
__global__ __launch_bounds__(256) void paged_attention_rows_kernel(const PagedArgs a, const PagedAttention p)
{
    constexpr int ROW = DIM * CODE_BYTES<TYPE>, OUT = DIM / 64;
    __shared__ float q_s[4][DIM];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int parts = (p.n_q + 3) / 4, t = blockIdx.x / parts, head = blockIdx.x % parts * 4 + wave;
    const int s = paged_sequence(a, t);
    if (s < 0 || head >= p.n_q) { return; }
    const int n_new = a.seq_start[s + 1] - a.seq_start[s], ctx = paged_rows(a, s), pos = ctx - (a.seq_start[s + 1] - t);
    if (n_new > p.max_new) { return; }
    const int h = head / p.group;
    for (int d = lane; d < DIM; d += 64) { q_s[wave][d] = bf16_bits_to_f32(p.q[(size_t)t * p.ldq + (size_t)head * DIM + d]); }
    __builtin_amdgcn_wave_barrier();
    float m = -INFINITY, l = 0.0f, out[OUT] = {};
    for (int base = 0; base <= pos; base += 64)
    {
        const int key = base + lane;
        const int page = key <= pos ? paged_page(a, s, key) : -1;
        const bool seen = page >= 0 && (p.window == 0 || key > pos - p.window || key < p.n_sink);
        const size_t row = paged_row(a, h, key);
        float score = -INFINITY;
        if (seen)
        {
            const uint8_t* const k = a.k + page * a.page_stride + row * ROW;
            const float scale = TYPE == DT_BF16 ? 1.0f : bits_to_f32((uint32_t)a.k_scale[page * a.scale_stride + row] << 23);
            float sum = 0.0f;
            for (int d = 0; d < DIM; d++) { sum += q_s[wave][d] * paged_element<TYPE>(k, d, scale); }
            score = sum * p.scale;
        }
        float top = score;
        for (int o = 1; o < 64; o <<= 1) { top = fmaxf(top, __shfl_xor(top, o)); }
        const float next = fmaxf(m, top), shrink = next > -INFINITY ? expf(m - next) : 1.0f;
        const float w = seen && (next > -INFINITY || score != score) ? expf(score - next) : 0.0f;
        m = next;
        l = l * shrink + wave_sum(w);
        for (int o = 0; o < OUT; o++) { out[o] *= shrink; }
        const unsigned long long visible = __ballot(seen);
        for (int j = 0; j < 64; j++)
        {
            if (!(visible >> j & 1)) { continue; }
            const int from = __shfl(page, j);
            const size_t r = paged_row(a, h, base + j);
            const float scale = TYPE == DT_BF16 ? 1.0f : bits_to_f32((uint32_t)a.v_scale[from * a.scale_stride + r] << 23), weight = __shfl(w, j);
            for (int o = 0; o < OUT; o++) { out[o] += weight * paged_element<TYPE>(a.v + from * a.page_stride + r * ROW, lane + 64 * o, scale); }
        }
    }
    for (int o = 0; o < OUT; o++)
    {
        p.y[(size_t)t * p.ldy + (size_t)head * DIM + lane + 64 * o] = (uint16_t)f32_to_bf16_bits(l == 0.0f ? 0.0f : out[o] / l);
    }
}

}    // namespace ccq
