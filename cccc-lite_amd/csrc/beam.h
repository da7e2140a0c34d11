// The best continuations of groups of beams over the vocabulary.
//   total(b, v) = score_b + x_bv - m_b - log sum_v exp(x_bv - m_b),  m_b the largest logit of beam b
// Within a beam a continuation's place follows from its logit alone: 16 bits whose order is that of the numbers, and the token, as one number per continuation that no other
// of its row has.  So a workgroup takes a chunk of a row, keeps the n_out largest of these numbers beside the chunk's maximum and sum, and what is left of all
// chunks of a group's rows is few enough for one workgroup to compare by their totals.
// To keep the largest K of many, each thread's own largest comes first: the K-th largest of those is no larger than the K-th largest of all, and only the K threads that reach it
// can have more.
#pragma once
#include "quant_device.h"

namespace ccq
{

struct BeamSelect
{
    const uint16_t* logits;
    size_t ld;
    const float* score;
    const int* last;
    int eos, n_groups, n_beams, vocab, n_out, chunks;
    int *parent_out, *token_out;
    float* score_out;
    double2* stats;                 // [row][chunk] (largest logit, sum of exp(logit - that))
    uint32_t* found;                // [row][chunk][n_out]: order of the logit and 65535 - place in the chunk; 0: none
};

constexpr int BEAM_THREADS = 256, BEAM_PICK_THREADS = 1024;
constexpr uint32_t BEAM_LEAST = 0x007Fu, BEAM_MOST = 0xFF80u;              // orders of minus and of plus infinity

// BF16 bits -> 16 bits in the order of the numbers; NaN as minus infinity, -0 as 0.
__device__ __forceinline__ uint32_t beam_order(uint32_t b)
{
    b = (b & 0x7FFFu) > 0x7F80u ? 0xFF80u : b == 0x8000u ? 0u : b;
    return b & 0x8000u ? b ^ 0xFFFFu : b | 0x8000u;
}
__device__ __forceinline__ float beam_logit(uint32_t order) { return bits_to_f32((order & 0x8000u ? order ^ 0x8000u : order ^ 0xFFFFu) << 16); }

enum class Beam { ALIVE, ENDED, UNBORN };
__device__ __forceinline__ Beam beam_state(const BeamSelect& p, int row)
{
    if (p.score && !(fabsf(p.score[row]) < INFINITY)) { return Beam::UNBORN; }
    return p.last && p.last[row] == p.eos ? Beam::ENDED : Beam::ALIVE;
}

// e^d for d <= 0 in 64 bits, to 1e-11 of it: 2^n 2^f, |f| <= 1/2, the series of 2^f = e^(f ln 2) to the ninth power.  Scores that are next to each other decide, so
// that the sum's error has to be well below what separates two of them.
__device__ __forceinline__ double beam_exp(double d)
{
    const double t = fmax(d, -700.0) * 1.4426950408889634074, n = rint(t), x = (t - n) * 0.69314718055994530942;
    double r = 1.0 / 362880.0;
    r = fma(r, x, 1.0 / 40320.0);
    r = fma(r, x, 1.0 / 5040.0);
    r = fma(r, x, 1.0 / 720.0);
    r = fma(r, x, 1.0 / 120.0);
    r = fma(r, x, 1.0 / 24.0);
    r = fma(r, x, 1.0 / 6.0);
    r = fma(r, x, 0.5);
    r = fma(r, x, 1.0);
    r = fma(r, x, 1.0);
    return __builtin_bit_cast(double, __builtin_bit_cast(long long, r) + ((long long)(int)n << 52));
}

// The largest number that at least k of the 256 at `of` reach, or one between it and the next smaller of them; 1 if fewer than k are above 0.  Bit by bit, by each wave for itself.
__device__ __forceinline__ uint32_t beam_kth(const uint32_t* of, int k)
{
    const int lane = threadIdx.x & 63;
    const uint32_t v[4] = { of[lane], of[64 + lane], of[128 + lane], of[192 + lane] };
    uint32_t kth = 0;
    for (int bit = 31; bit >= 0; bit--)
    {
        const uint32_t next = kth | 1u << bit;
        int reach = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) { reach += __builtin_popcountll(__ballot(v[i] >= next)); }
        if (reach >= k) { kth = next; }
        if (reach == k) { break; }
    }
    return max(kth, 1u);
}

// A chunk of 256 PER logits of a row, PER of them per thread, eight side by side.  Grid: rows x chunks.  LDS: two lists of numbers.
template <int PER>
__global__ __launch_bounds__(BEAM_THREADS) void beam_chunk_kernel(const BeamSelect p)
{
    constexpr int CHUNK = BEAM_THREADS * PER, VECTORS = PER / 8;
    extern __shared__ __attribute__((aligned(16))) uint32_t lists[];
    __shared__ __attribute__((aligned(16))) uint32_t best[BEAM_THREADS];
    __shared__ double sums[BEAM_THREADS / 64];
    __shared__ int counts[2];
    const int row = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks, first = chunk * CHUNK, left = p.vocab - first;
    const Beam state = beam_state(p, row);
    const uint16_t* const src = p.logits + (size_t)row * p.ld + first;
    u32x4 raw[VECTORS];
#pragma unroll
    for (int v = 0; v < VECTORS; v++)
    {
        const int at = (v * BEAM_THREADS + (int)threadIdx.x) * 8;
        raw[v] = state == Beam::ALIVE && at < left ? *(const u32x4*)(src + at) : u32x4{ 0, 0, 0, 0 };
    }
    // element e of vector v as a number
    auto number = [&](int v, int e) {
        const int at = (v * BEAM_THREADS + (int)threadIdx.x) * 8 + e;
        uint32_t order = beam_order(raw[v][e / 2] >> (16 * (e & 1)) & 0xFFFFu);
        if (state != Beam::ALIVE) { order = state == Beam::ENDED && first + at == p.eos ? BEAM_MOST : BEAM_LEAST; }
        return at < left ? order << 16 | (uint32_t)(0xFFFF - at) : 0u;
    };
    uint32_t mine = 0;
#pragma unroll
    for (int v = 0; v < VECTORS; v++)
#pragma unroll
        for (int e = 0; e < 8; e++) { mine = max(mine, number(v, e)); }
    best[threadIdx.x] = mine;
    if (threadIdx.x < 2) { counts[threadIdx.x] = 0; }
    __syncthreads();
    uint32_t from = beam_kth(best, p.n_out), top = max(max(best[threadIdx.x & 63], best[64 + (threadIdx.x & 63)]), max(best[128 + (threadIdx.x & 63)], best[192 + (threadIdx.x & 63)]));
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) { top = max(top, (uint32_t)__shfl_xor((int)top, d)); }
    // the sum, of rows that go on
    const float m = beam_logit(top >> 16);
    double sum = 0.0;
    if (state == Beam::ALIVE)
    {
#pragma unroll
        for (int v = 0; v < VECTORS; v++)
#pragma unroll
            for (int e = 0; e < 8; e++)
            {
                const uint32_t of = number(v, e);
                const float x = beam_logit(of >> 16);
                if (of != 0 && x > -INFINITY) { sum += x == m ? 1.0 : m == INFINITY ? 0.0 : beam_exp((double)x - (double)m); }
            }
    }
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) { sum += __shfl_xor(sum, d); }
    if ((threadIdx.x & 63) == 0) { sums[threadIdx.x >> 6] = sum; }
    __syncthreads();
    if (threadIdx.x == 0)
    {
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < BEAM_THREADS / 64; w++) { all += sums[w]; }
        p.stats[(size_t)row * p.chunks + chunk] = make_double2(m, all);
    }
    // what reaches the K-th largest of the threads' largest
    uint32_t *list = lists, *next = lists + p.n_out * PER;
    if (mine >= from)
    {
#pragma unroll
        for (int v = 0; v < VECTORS; v++)
#pragma unroll
            for (int e = 0; e < 8; e++)
            {
                const uint32_t of = number(v, e);
                if (of >= from) { list[atomicAdd(counts, 1)] = of; }
            }
    }
    __syncthreads();
    int n = counts[0];
    // the same again while many are left: a thread then has n / 256 of them
    for (int round = 1; n > 2 * BEAM_THREADS; round++)
    {
        mine = 0;
        for (int i = threadIdx.x; i < n; i += BEAM_THREADS) { mine = max(mine, list[i]); }
        best[threadIdx.x] = mine;
        if (threadIdx.x == 0) { counts[round & 1] = 0; }
        __syncthreads();
        from = beam_kth(best, p.n_out);
        for (int i = threadIdx.x; i < n; i += BEAM_THREADS)
        {
            const uint32_t of = list[i];
            if (of >= from) { next[atomicAdd(counts + (round & 1), 1)] = of; }
        }
        __syncthreads();
        n = counts[round & 1];
        uint32_t* const other = list;
        list = next;
        next = other;
    }
    uint32_t* const found = p.found + ((size_t)row * p.chunks + chunk) * p.n_out;
    for (int i = n + threadIdx.x; i < p.n_out; i += BEAM_THREADS) { found[i] = 0; }
    for (int i = threadIdx.x; i < n; i += BEAM_THREADS)
    {
        const uint32_t of = list[i];
        int place = 0;
        for (int j = 0; j < n; j++) { place += list[j] > of; }
        if (place < p.n_out) { found[place] = of; }
    }
}

// A continuation among those of its group: its total in an order of whole numbers, then what decides between equal totals (all 0: none).
struct BeamRank
{
    unsigned long long total, then;
    __device__ __forceinline__ bool operator>(const BeamRank& o) const { return total > o.total || (total == o.total && then > o.then); }
};

// The n_out best of what the chunks of a group's rows left: byte by byte of their ranks, by how many have each value, until just n_out reach the bytes found.  Grid: groups.
template <int PER>
__global__ __launch_bounds__(BEAM_PICK_THREADS) void beam_pick_kernel(const BeamSelect p)
{
    constexpr int CHUNK = BEAM_THREADS * PER, HELD = 4;                     // continuations that a thread keeps the ranks of; with more it works them out for each byte
    __shared__ double largest[64], log_sum[64], scores[64];
    __shared__ Beam states[64];
    __shared__ int bins[256];
    __shared__ int chosen[3];                                               // the byte, how many are above it, and with it
    __shared__ BeamRank picked[128];
    __shared__ int from[128];
    __shared__ int count;
    const int group = blockIdx.x, row0 = group * p.n_beams, per_row = p.chunks * p.n_out, n_all = p.n_beams * per_row;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int b = wave; b < p.n_beams; b += BEAM_PICK_THREADS / 64)
    {
        const double2* const of = p.stats + (size_t)(row0 + b) * p.chunks;
        double m = -INFINITY, sum = 0.0;
        for (int c = lane; c < p.chunks; c += 64) { m = fmax(m, of[c].x); }
#pragma unroll
        for (int d = 32; d >= 1; d /= 2) { m = fmax(m, __shfl_xor(m, d)); }
        for (int c = lane; c < p.chunks; c += 64) { sum += of[c].x == m ? of[c].y : m < INFINITY ? of[c].y * exp(of[c].x - m) : 0.0; }
#pragma unroll
        for (int d = 32; d >= 1; d /= 2) { sum += __shfl_xor(sum, d); }
        if (lane == 0)
        {
            states[b] = beam_state(p, row0 + b);
            scores[b] = p.score ? p.score[row0 + b] : 0.0;
            largest[b] = m;
            log_sum[b] = log(sum);
        }
    }
    if (threadIdx.x == 0) { count = 0; }
    __syncthreads();
    const uint32_t* const found = p.found + (size_t)row0 * per_row;
    auto token_of = [&](int i, uint32_t of) { return i % per_row / p.n_out * CHUNK + (0xFFFF - (int)(of & 0xFFFFu)); };
    auto rank_of = [&](int i) {
        const uint32_t of = i < n_all ? found[i] : 0u;
        if (of == 0) { return BeamRank{ 0, 0 }; }
        const int b = i / per_row;
        const uint32_t order = of >> 16;
        double total = -INFINITY;
        if (states[b] == Beam::ENDED && order == BEAM_MOST) { total = scores[b]; }
        if (states[b] == Beam::ALIVE && order != BEAM_LEAST)
        {
            const double x = beam_logit(order);
            total = scores[b] + ((x == largest[b] ? 0.0 : x - largest[b]) - log_sum[b]);
        }
        const unsigned long long bits = __builtin_bit_cast(unsigned long long, total + 0.0);       // -0 is 0
        return BeamRank{ bits >> 63 ? ~bits : bits | 1ull << 63, (unsigned long long)(0xFFFF - b) << 48 | (unsigned long long)order << 32 | (0xFFFFFFFFu - (uint32_t)token_of(i, of)) };
    };
    BeamRank held[HELD];
    const bool holds = n_all <= HELD * BEAM_PICK_THREADS;
    if (holds)
    {
#pragma unroll
        for (int n = 0; n < HELD; n++) { held[n] = rank_of(n * BEAM_PICK_THREADS + threadIdx.x); }
    }
    auto each = [&](auto f) {
        if (holds)
        {
#pragma unroll
            for (int n = 0; n < HELD; n++) { f(n * BEAM_PICK_THREADS + (int)threadIdx.x, held[n]); }
        }
        else
        {
            for (int i = threadIdx.x; i < n_all; i += BEAM_PICK_THREADS) { f(i, rank_of(i)); }
        }
    };
    // ranks that agree with `least` in the bytes found so far are open, larger ones are in: `need` more
    BeamRank least = { 0, 0 };
    int need = p.n_out;
    for (int byte = 0; byte < 16; byte++)
    {
        const int shift = 56 - byte % 8 * 8;
        if (threadIdx.x < 256) { bins[threadIdx.x] = 0; }
        __syncthreads();
        each([&](int, const BeamRank& r) {
            const unsigned long long word = byte < 8 ? r.total : r.then, known = byte < 8 ? least.total : least.then;
            const bool open = (byte < 8 || r.total == least.total) && (shift == 56 || word >> (shift + 8) == known >> (shift + 8));
            if (open && (r.total | r.then) != 0) { atomicAdd(bins + (word >> shift & 255), 1); }
        });
        __syncthreads();
        if (wave == 0)
        {
            // lane l: bins 255 - 4 l down to 252 - 4 l
            int n[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++)
            {
                n[i] = bins[255 - 4 * lane - i];
                sum += n[i];
            }
            int above = sum;
#pragma unroll
            for (int d = 1; d < 64; d *= 2)
            {
                const int other = __shfl_up(above, d);
                above += lane >= d ? other : 0;
            }
            above -= sum;
#pragma unroll
            for (int i = 0; i < 4; i++)
            {
                if (above < need && above + n[i] >= need)
                {
                    chosen[0] = 255 - 4 * lane - i;
                    chosen[1] = above;
                    chosen[2] = n[i];
                }
                above += n[i];
            }
        }
        __syncthreads();
        (byte < 8 ? least.total : least.then) |= (unsigned long long)chosen[0] << shift;
        need -= chosen[1];
        if (chosen[2] == need) { break; }
    }
    // all from `least` on, n_out of them, each to its place
    each([&](int i, const BeamRank& r) {
        if (!(least > r) && (r.total | r.then) != 0)
        {
            const int at = atomicAdd(&count, 1);
            picked[at] = r;
            from[at] = i;
        }
    });
    __syncthreads();
    if ((int)threadIdx.x < p.n_out)
    {
        const BeamRank mine = picked[threadIdx.x];
        int place = 0;
        for (int j = 0; j < p.n_out; j++) { place += picked[j] > mine; }
        const int i = from[threadIdx.x], to = group * p.n_out + place;
        p.parent_out[to] = row0 + i / per_row;
        p.token_out[to] = token_of(i, found[i]);
        p.score_out[to] = (float)__builtin_bit_cast(double, mine.total >> 63 ? mine.total & ~(1ull << 63) : ~mine.total);
    }
}

}    // namespace ccq
