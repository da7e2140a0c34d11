// The best continuations of groups of beams over the vocabulary.
//   total(b, v) = score_b + x_bv - m_b - log sum_v exp(x_bv - m_b),  m_b the largest logit of beam b
// Within a beam a continuation's place follows from its logit alone: 16 bits whose order is that of the numbers, and the token, as one number per continuation that no other
// of its row has.  So a workgroup takes a chunk of a row, keeps the n_out largest of these numbers beside the chunk's maximum and sum, and what is left of all
// chunks of a group's rows is few enough for one workgroup to compare by their totals.
// To keep the largest K of many, each thread's own largest comes first: the K-th largest of those is no larger than the K-th largest of all, and only the K threads that reach it
// can have more.
#pragma once
#include "quant_device.h"
#include <type_traits>

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

// The order of a logit: 16 bits that compare as the numbers do, -0 as 0 (sign and magnitude as a whole number, from 0x8000 on).
constexpr uint32_t BEAM_LEAST = 0x8000u - 0x7F80u, BEAM_MOST = 0x8000u + 0x7F80u;              // of minus and of plus infinity
__device__ __forceinline__ float beam_logit(uint32_t order) { return bits_to_f32((order >= 0x8000u ? order - 0x8000u : 0x8000u | (0x8000u - order)) << 16); }

// The same of two logits, not yet from 0x8000 on.
typedef short beam_i16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t beam_signed(uint32_t two)
{
    const beam_i16x2 x = __builtin_bit_cast(beam_i16x2, two), sign = x >> 15;
    return __builtin_bit_cast(uint32_t, (beam_i16x2)((x ^ (sign & (short)0x7FFF)) - sign));
}
// Order of a logit's bits, NaN as minus infinity.
__device__ __forceinline__ uint32_t beam_order(uint32_t bits)
{
    const uint32_t size = bits & 0x7FFFu;
    return size > 0x7F80u ? BEAM_LEAST : bits & 0x8000u ? 0x8000u - size : 0x8000u + size;
}

enum class Beam { ALIVE, ENDED, UNBORN };
__device__ __forceinline__ Beam beam_state(const BeamSelect& p, int row)
{
    if (p.score && !(fabsf(p.score[row]) < INFINITY)) { return Beam::UNBORN; }
    return p.last && p.last[row] == p.eos ? Beam::ENDED : Beam::ALIVE;
}

// A value of each lane added up, or its largest, over the wave.
template <int CTRL>
__device__ __forceinline__ double beam_dpp(double v)
{
    const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)bits, CTRL, 0xF, 0xF, true), hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(bits >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double beam_lane(double v, int lane)
{
    const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
    return __builtin_bit_cast(double, (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(bits >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)bits, lane));
}
template <class F>
__device__ __forceinline__ double beam_over_wave(double v, F f)
{
    v = f(v, beam_dpp<0xB1>(v));                                            // quad_perm [1,0,3,2]
    v = f(v, beam_dpp<0x4E>(v));                                            // quad_perm [2,3,0,1]
    v = f(v, beam_dpp<0x141>(v));                                           // row_half_mirror
    v = f(v, beam_dpp<0x140>(v));                                           // row_mirror
    return f(f(beam_lane(v, 0), beam_lane(v, 16)), f(beam_lane(v, 32), beam_lane(v, 48)));
}

// Sum over 16 lanes.
__device__ __forceinline__ int beam_sum16(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);           // quad_perm [1,0,3,2]
    v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);           // quad_perm [2,3,0,1]
    v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true);          // row_half_mirror
    return v + __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, true);    // row_mirror
}

template <class F>
__device__ __forceinline__ uint32_t beam_reduce(uint32_t v, F f)
{
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));          // quad_perm [1,0,3,2]
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));          // quad_perm [2,3,0,1]
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));         // row_half_mirror
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));         // row_mirror
    const uint32_t a = f((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
    return f(a, f((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}

// A number that k of the 256 at `of` reach, or more only if the k-th largest is there several times; the largest of them all in `top`.  Bit by bit behind those that all have in common, by each
// wave for itself.
__device__ __forceinline__ uint32_t beam_kth(const uint32_t* of, int k, uint32_t& top)
{
    const int lane = threadIdx.x & 63;
    const uint32_t v[4] = { of[lane], of[64 + lane], of[128 + lane], of[192 + lane] };
    top = beam_reduce(max(max(v[0], v[1]), max(v[2], v[3])), [](uint32_t a, uint32_t b) { return max(a, b); });
    const uint32_t bottom = beam_reduce(min(min(v[0], v[1]), min(v[2], v[3])), [](uint32_t a, uint32_t b) { return min(a, b); });
    int bit = 31 - __builtin_clz(top ^ bottom | 1u);
    uint32_t kth = top >> bit >> 1 << bit << 1;
    for (; bit >= 0; bit--)
    {
        const uint32_t next = kth | 1u << bit;
        int reach = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) { reach += __builtin_popcountll(__ballot(v[i] >= next)); }
        if (reach >= k) { kth = next; }
        if (reach == k) { break; }
    }
    return kth;
}

// e^d, d <= 0, without the error that log2 e in 24 bits would give all of them alike.
__device__ __forceinline__ float beam_exp(float d) { return __builtin_amdgcn_exp2f(fmaf(d, 1.44269502162933349609f, d * 1.92596299112661746887e-8f)); }

// A chunk of 256 PER logits of a row, PER of them per thread, eight side by side; PER <= 64.  Each logit is seen once, as it arrives: the thread's largest number, and its sum
// beside its largest logit so far (FP32 exponentials of exact differences, errors of both signs: the logarithm of a row's sum is off by 2e-9 to 6e-8 on average, over rows of five distributions).  The few threads that reach the
// bound have their logits read once more, from the L2.  MI355X, 128 rows of 128256 logits 17.6 us (33 MB: 1.9 TB/s): all workgroups run at once, so that loads (6 us by their bytes), the arithmetic
// and the search for the best come one after the other: 17.6 vector instructions per logit, counted over the launch, 7 us of their issue.  Grid: rows x chunks.  LDS: two lists of numbers.
template <int PER>
__global__ __launch_bounds__(BEAM_THREADS) void beam_chunk_kernel(const BeamSelect p)
{
    constexpr int CHUNK = BEAM_THREADS * PER, VECTORS = PER / 8;
    constexpr uint32_t BARRED = 0xFF80FF80u;                                // minus infinity, twice
    extern __shared__ __attribute__((aligned(16))) uint32_t lists[];
    __shared__ uint32_t best[BEAM_THREADS];
    __shared__ double sums[BEAM_THREADS / 64];
    __shared__ int winners[128];
    __shared__ int counts[3];
    const int row = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks, first = chunk * CHUNK, left = p.vocab - first, lane = threadIdx.x & 63;
    const uint16_t* const src = p.logits + (size_t)row * p.ld + first;
    auto place = [&](int thread, int n) { return (n / 8 * BEAM_THREADS + thread) * 8 + n % 8; };                   // of a thread's n-th
    int largest = -0x7FFFFFFF - 1;                                          // order, then 63 - n
    float m = -3.402823466e38f, sum = 0.0f;
    auto take = [&](auto partial) {
        // a last chunk: behind the vocabulary barred, and left out at the end
        u32x4 raw[VECTORS];
#pragma unroll
        for (int v = 0; v < VECTORS; v++)
        {
            const int at = place(threadIdx.x, 8 * v);
            raw[v] = *(const u32x4*)(src + (partial && at >= left ? 0 : at));
        }
#pragma unroll
        for (int v = 0; v < VECTORS; v++)
        {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e += 2)
            {
                const int n = 8 * v + e;
                uint32_t two = raw[v][e / 2];
                if constexpr (partial)
                {
                    two = place(threadIdx.x, n) < left ? two : BARRED;
                    two = place(threadIdx.x, n + 1) < left ? two : (two & 0xFFFFu) | (BARRED & 0xFFFF0000u);
                }
                const uint32_t order = beam_signed(two);
                largest = max(largest, max((int)(order << 16 | (uint32_t)(63 - n)), (int)((order & 0xFFFF0000u) | (uint32_t)(62 - n))));
                x[e] = bits_to_f32(two << 16);
                x[e + 1] = bits_to_f32(two & 0xFFFF0000u);
            }
            const float next = fmaxf(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))), m);
            float part[2] = { sum * beam_exp(m - next), 0.0f };
#pragma unroll
            for (int e = 0; e < 8; e++) { part[e & 1] += beam_exp(x[e] - next); }
            sum = part[0] + part[1];
            m = next;
        }
    };
    if (left >= CHUNK) { take(std::false_type()); }
    else { take(std::true_type()); }
    const Beam state = beam_state(p, row);
    const int eos = state == Beam::ENDED && p.eos >= first && p.eos - first < left ? p.eos - first : -1;       // (a place behind the vocabulary would count for the bound)
    auto number = [](uint32_t order, int at) { return order << 16 | (uint32_t)(0xFFFF - at); };
    auto number_of = [&](uint32_t bits, int at) { return number(state == Beam::ALIVE ? beam_order(bits) : at == eos ? BEAM_MOST : BEAM_LEAST, at); };
    uint32_t mine = number((uint32_t)((largest >> 16) + 0x8000), place(threadIdx.x, 63 - (largest & 0xFFFF)));
    if (state != Beam::ALIVE)
    {
        const bool owns = eos >= 0 && eos < CHUNK && eos / 8 % BEAM_THREADS == (int)threadIdx.x;
        mine = number_of(0, owns ? eos : place(threadIdx.x, 0));
        sum = 0.0f;
    }
    else if (!(sum == sum))
    {
        // NaN or plus infinity among them: one by one
        mine = 0;
        for (int n = 0; n < PER; n++)
        {
            const int at = place(threadIdx.x, n);
            mine = max(mine, number_of(at < left ? src[at] : 0xFF80u, at));
        }
        m = beam_logit(mine >> 16);
        sum = 0.0f;
        for (int n = 0; n < PER && m > -INFINITY; n++)
        {
            const int at = place(threadIdx.x, n);
            const float x = beam_logit(number_of(at < left ? src[at] : 0xFF80u, at) >> 16);
            sum += x == m ? 1.0f : m < INFINITY ? beam_exp(x - m) : 0.0f;
        }
    }
    best[threadIdx.x] = mine;
    if (threadIdx.x < 3) { counts[threadIdx.x] = 0; }
    __syncthreads();
    uint32_t top;
    uint32_t from = beam_kth(best, p.n_out, top);
    const float all_m = beam_logit(top >> 16);
    double all = m == all_m ? (double)sum : all_m < INFINITY && sum > 0.0f ? (double)(sum * beam_exp(m - all_m)) : 0.0;
    all = beam_over_wave(all, [](double a, double b) { return a + b; });
    if (lane == 0) { sums[threadIdx.x >> 6] = all; }
    if (mine >= from) { winners[atomicAdd(counts + 2, 1)] = threadIdx.x; }
    __syncthreads();
    if (threadIdx.x == 0) { p.stats[(size_t)row * p.chunks + chunk] = make_double2(all_m, (sums[0] + sums[1]) + (sums[2] + sums[3])); }
    // what reaches the K-th largest of the threads' largest
    uint32_t *list = lists, *next = lists + p.n_out * PER;
    const int n_winners = counts[2];
    for (int i = threadIdx.x; i < n_winners * VECTORS; i += BEAM_THREADS)
    {
        const int at = place(winners[i / VECTORS], i % VECTORS * 8);
        if (at >= left) { continue; }
        const u32x4 eight = *(const u32x4*)(src + at);
#pragma unroll
        for (int e = 0; e < 8; e++)
        {
            const uint32_t of = number_of(eight[e / 2] >> (16 * (e & 1)) & 0xFFFFu, at + e);
            if (of >= from && at + e < left) { list[atomicAdd(counts, 1)] = of; }
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
        from = beam_kth(best, p.n_out, top);
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
    // places by counting, 16 lanes for each
    for (int i0 = 0; i0 < n; i0 += BEAM_THREADS / 16)
    {
        const int i = i0 + threadIdx.x / 16;
        const uint32_t of = i < n ? list[i] : 0u;
        int rank = 0;
        for (int j = threadIdx.x % 16; j < n; j += 16) { rank += list[j] > of; }
        rank = beam_sum16(rank);
        if (i < n && threadIdx.x % 16 == 0 && rank < p.n_out) { found[rank] = of; }
    }
}

// A continuation among those of its group: its total in an order of whole numbers, then what decides between equal totals (all 0: none).
struct BeamRank
{
    unsigned long long total, then;
    __device__ __forceinline__ bool operator>(const BeamRank& o) const { return total > o.total || (total == o.total && then > o.then); }
};

// The n_out best of what the chunks of a group's rows left, whose lists are in order.  The n_out-th largest of the lists' first entries, 256 in all, is a bound
// that n_out continuations reach, and few more do: those are ranked by counting.  Where more reach it than there is room for (equal totals, such as minus infinity), the ranks are gone
// through byte by byte, by how many have each value, until just n_out reach the bytes found.  Grid: groups.
constexpr int BEAM_ROOM = 512;

// i / d for 0 <= i < 2^24, `by` next to 1 / d.
__device__ __forceinline__ int beam_divided(int i, int d, float by)
{
    const int q = (int)((float)i * by), left = i - q * d;
    return q + (left >= d ? 1 : 0) - (left < 0 ? 1 : 0);
}

template <int PER>
__global__ __launch_bounds__(BEAM_PICK_THREADS) void beam_pick_kernel(const BeamSelect p)
{
    constexpr int CHUNK = BEAM_THREADS * PER, HELD = 4;                     // continuations that a thread keeps the ranks of; with more it works them out for each byte
    __shared__ double largest[64], log_sum[64], scores[64];
    __shared__ Beam states[64];
    __shared__ int bins[256];
    __shared__ int chosen[3];                                               // the byte, how many are above it, and with it
    __shared__ BeamRank picked[BEAM_ROOM];
    __shared__ uint32_t heads[256];
    __shared__ int count;
    const int group = blockIdx.x, row0 = group * p.n_beams, per_row = p.chunks * p.n_out, n_all = p.n_beams * per_row;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // asked for beside the statistics: what the thread keeps, and an entry for the bound, of the first 256 lists as many of each as make 256
    const uint32_t* const found = p.found + (size_t)row0 * per_row;
    const int n_lists = min(p.n_beams * p.chunks, 256), deep = min(256 / n_lists, p.n_out), head = (int)threadIdx.x / deep * p.n_out + (int)threadIdx.x % deep;
    const bool holds = n_all <= HELD * BEAM_PICK_THREADS;
    uint32_t words[HELD], head_word = (int)threadIdx.x < n_lists * deep ? found[head] : 0u;
#pragma unroll
    for (int n = 0; n < HELD; n++)
    {
        const int i = n * BEAM_PICK_THREADS + threadIdx.x;
        words[n] = holds && i < n_all ? found[i] : 0u;
    }
    for (int b = wave; b < p.n_beams; b += BEAM_PICK_THREADS / 64)
    {
        const double2* const of = p.stats + (size_t)(row0 + b) * p.chunks;
        double m, sum;
        const double2 mine = lane < p.chunks ? of[lane] : make_double2(-INFINITY, 0.0);
        m = mine.x;
        for (int c = lane + 64; c < p.chunks; c += 64) { m = fmax(m, of[c].x); }
        m = beam_over_wave(m, [](double a, double b) { return fmax(a, b); });
        auto part = [&](const double2& c) { return c.x == m ? c.y : m < INFINITY && c.y > 0.0 ? c.y * exp(c.x - m) : 0.0; };
        sum = part(mine);
        for (int c = lane + 64; c < p.chunks; c += 64) { sum += part(of[c]); }
        sum = beam_over_wave(sum, [](double a, double b) { return a + b; });
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
    const float by_row = 1.0f / (float)per_row, by_out = 1.0f / (float)p.n_out;
    auto beam_of = [&](int i) { return beam_divided(i, per_row, by_row); };
    auto token_of = [&](int i, int b, uint32_t of) { return beam_divided(i - b * per_row, p.n_out, by_out) * CHUNK + (0xFFFF - (int)(of & 0xFFFFu)); };
    auto rank_of = [&](int i, uint32_t of) {
        if (of == 0) { return BeamRank{ 0, 0 }; }
        const int b = beam_of(i);
        const uint32_t order = of >> 16;
        double total = -INFINITY;
        if (states[b] == Beam::ENDED && order == BEAM_MOST) { total = scores[b]; }
        if (states[b] == Beam::ALIVE && order != BEAM_LEAST)
        {
            const double x = beam_logit(order);
            total = scores[b] + ((x == largest[b] ? 0.0 : x - largest[b]) - log_sum[b]);
        }
        const unsigned long long bits = __builtin_bit_cast(unsigned long long, total + 0.0);       // -0 is 0
        return BeamRank{ bits >> 63 ? ~bits : bits | 1ull << 63, (unsigned long long)(0xFFFF - b) << 48 | (unsigned long long)order << 32 | (0xFFFFFFFFu - (uint32_t)token_of(i, b, of)) };
    };
    BeamRank held[HELD];
#pragma unroll
    for (int n = 0; n < HELD; n++) { held[n] = rank_of(n * BEAM_PICK_THREADS + threadIdx.x, words[n]); }
    auto each = [&](auto f) {
        if (holds)
        {
#pragma unroll
            for (int n = 0; n < HELD; n++) { f(held[n]); }
        }
        else
        {
            for (int i = threadIdx.x; i < n_all; i += BEAM_PICK_THREADS) { f(rank_of(i, found[i])); }
        }
    };
    // the bound, of the totals' upper halves
    if (threadIdx.x < 256) { heads[threadIdx.x] = (uint32_t)(rank_of(head, head_word).total >> 32); }
    __syncthreads();
    uint32_t top;
    const uint32_t bound = beam_kth(heads, p.n_out, top);
    each([&](const BeamRank& r) {
        if ((uint32_t)(r.total >> 32) >= bound && (r.total | r.then) != 0)
        {
            const int at = atomicAdd(&count, 1);
            if (at < BEAM_ROOM) { picked[at] = r; }
        }
    });
    __syncthreads();
    int n_picked = count;
    if (n_picked > BEAM_ROOM)
    {
        __syncthreads();
        if (threadIdx.x == 0) { count = 0; }
        // ranks that agree with `least` in the bytes found so far are open, larger ones are in: `need` more
        BeamRank least = { 0, 0 };
        int need = p.n_out;
        for (int byte = 0; byte < 16; byte++)
        {
            const int shift = 56 - byte % 8 * 8;
            if (threadIdx.x < 256) { bins[threadIdx.x] = 0; }
            __syncthreads();
            each([&](const BeamRank& r) {
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
        // all from `least` on, n_out of them
        each([&](const BeamRank& r) {
            if (!(least > r) && (r.total | r.then) != 0)
            {
                const int at = atomicAdd(&count, 1);
                picked[at] = r;
            }
        });
        __syncthreads();
        n_picked = p.n_out;
    }
    for (int i0 = 0; i0 < n_picked; i0 += BEAM_PICK_THREADS / 16)
    {
        const int n = i0 + threadIdx.x / 16;
        const BeamRank mine = picked[min(n, n_picked - 1)];
        int place = 0;
        for (int j = threadIdx.x % 16; j < n_picked; j += 16) { place += picked[j] > mine; }
        place = beam_sum16(place);
        if (n < n_picked && threadIdx.x % 16 == 0 && place < p.n_out)
        {
            const int to = group * p.n_out + place;
            p.parent_out[to] = row0 + 0xFFFF - (int)(mine.then >> 48);
            p.token_out[to] = (int)(0xFFFFFFFFu - (uint32_t)mine.then);
            p.score_out[to] = (float)__builtin_bit_cast(double, mine.total >> 63 ? mine.total & ~(1ull << 63) : ~mine.total);
        }
    }
}

}    // namespace ccq
