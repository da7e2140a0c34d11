// Attention of the new tokens of a batch of sequences over their pages, causal or (TREE) with bits that say which new tokens each sees.
//   y = sum_k p_k v_k / sum_k p_k,  p_k = exp(scale q k - m),  over the keys that the token sees, m a running maximum.
// The rows of a kv head are those of the sequence's new tokens and of the query heads that share it: row r is token r / group, head r % group.
// One kernel with two forms: sequences of up to 16 rows per kv head (RowsForm), their keys in parts that the last workgroup of a sequence adds up, and tiles of
// 128 rows of longer ones (TileForm), with ranges of keys where tiles are few, which a second launch adds.  The same sequences in tiles alone, MI355X us, 32 / 8 heads: 64 of
// one token on 1000 to 8000 E4M3 rows 216 for 108, 16 with a window of 4096 46 for 31, one on 4096 BF16 rows 16.0 for 13.4, 8 of four tokens on 500 to 3000 E4M3 rows 22 for 15.
#pragma once
#include "paged.h"

namespace ccq
{

struct PagedAttention
{
    const uint16_t* q;
    uint16_t* y;
    float* partial;                 // of tiles with ranges: [range][token][head][dim] sums, then [range][token][head] (max, sum)
    size_t ldq, ldy;
    int n_q, group, n_tokens, max_new, window, n_sink;
    int tiles, tile_split;          // tiles of 128 rows (at most) and the most ranges of each
    int row_slots;                  // workgroups per kv head that the GPU runs at once
    int row_parts;                  // workgroups per kv head for the parts of all sequences of at most 16 rows per kv head; 0: one for each sequence
    float* row_partial;             // [part][kv head][16][dim] sums, then (max, sum) likewise
    unsigned long long* there;      // [part][kv head]: the name of the call whose part is there
    unsigned long long call;        // of this call alone, 48 bits
    int min_rows;                   // sequences of at most so many rows per kv head are not cut into tiles
    int snake;                      // the second half of the tiles in the other order
    float scale;                    // log2 e / sqrt(dim)
    const unsigned long long* seen; // trees: bits of the new tokens that a token sees, seen_stride words each
    size_t seen_stride;
    int piece_slots;                // trees: `tiles` counts pieces of tiles (find_piece), about so many of them per kv head besides one for each tile; 0: whole tiles

    __device__ __forceinline__ float* row_sums(int slot, int kvh, int n_kv, int row, int dim) const { return row_partial + (((size_t)slot * n_kv + kvh) * 16 + row) * dim; }
    __device__ __forceinline__ float* row_stats(int slot, int kvh, int n_kv, int row, int dim) const
    {
        return row_partial + (size_t)row_parts * n_kv * 16 * dim + (((size_t)slot * n_kv + kvh) * 16 + row) * 2;
    }
    // of a piece of a tile that is in several, 2 piece_slots of them at most, by its row in the tile
    __device__ __forceinline__ float* piece_sums(int piece, int kvh, int n_kv, int row, int dim) const { return partial + (((size_t)piece * n_kv + kvh) * 128 + row) * dim; }
    __device__ __forceinline__ float2* piece_stats(int piece, int kvh, int n_kv, int row, int dim) const
    {
        return (float2*)(partial + (size_t)2 * piece_slots * n_kv * 128 * dim) + ((size_t)piece * n_kv + kvh) * 128 + row;
    }
    __device__ __forceinline__ float* piece_length() const { return partial - 4; }       // 1 / blocks of a range
    __device__ __forceinline__ size_t outputs() const { return (size_t)n_tokens * n_q; }
    __device__ __forceinline__ float* sums(int range, size_t row, int dim) const { return partial + ((size_t)range * outputs() + row) * dim; }
    __device__ __forceinline__ float2* stats(int range, size_t row, int dim) const { return (float2*)(partial + (size_t)tile_split * outputs() * dim) + (size_t)range * outputs() + row; }
};

// a value that all lanes have, in a scalar register
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// the sum of a value over the lanes up to this one
__device__ __forceinline__ int add_up_lanes(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);         // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);         // row_bcast 15 to rows 1 and 3
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast 31 to rows 2 and 3
}

// The new tokens of a sequence that a call computes: tokens first .. first + n - 1 of the activations, the first of them at position pos.
struct NewTokens
{
    int first, n, pos;
};

// What a lane has to read for them of sequence s (any from 0 on; beyond the last: none): asked for first where several are, in one trip.
struct SeqWords
{
    int begin = 0, end = 0, rows = 0;

    __device__ __forceinline__ SeqWords() {}
    __device__ __forceinline__ SeqWords(const PagedArgs& a, int s)
    {
        const int at = min(s, a.n_seqs - 1);
        begin = a.seq_start[at];
        end = a.seq_start[at + 1];
        rows = a.ctx_len[at];
    }
    __device__ __forceinline__ NewTokens tokens(const PagedArgs& a, const PagedAttention& p, int s) const
    {
        const int first = max(begin, 0), last = min(end, p.n_tokens);
        // (compared and not subtracted: ranges may hold anything)
        if (s >= a.n_seqs || last <= first || (long long)end - begin > p.max_new) { return { 0, 0, 0 }; }
        return { first, last - first, paged_rows(a, rows) - (end - first) };
    }
};

// The blocks of SIZE keys that tokens at positions lo .. hi see: the first `sinks` ones, then from block sinks + skip on; n in all.
template <int SIZE>
struct KeyBlocks
{
    int n = 0, sinks = 0, skip = 0;

    __device__ __forceinline__ KeyBlocks() {}
    __device__ __forceinline__ KeyBlocks(const PagedAttention& p, int lo, int hi)
    {
        const int blocks = max(hi + SIZE, 0) / SIZE;
        const int from = p.window == 0 ? 0 : max(lo - p.window + 1, 0) / SIZE;
        sinks = min((int)min(((long long)p.n_sink + SIZE - 1) / SIZE, (long long)blocks), from);
        skip = from - sinks;
        n = blocks - skip;
    }
    __device__ __forceinline__ int block(int i) const { return i < sinks ? i : i + skip; }
};

__device__ __forceinline__ bool sees(const PagedAttention& p, int pos, int key) { return key <= pos && (p.window == 0 || key > pos - p.window || key < p.n_sink); }

// Trees: a token sees the rows in front of its sequence's new tokens (within its window) and the new tokens whose bits are set.
// Which of keys key0 .. + 63 that is: `first` is the position of the first new token, pos the one that the token's window counts from, word(i) bits 64 i .. + 63 of
// the new tokens (any i from 0 on).
template <class Word>
__device__ __forceinline__ unsigned long long named_keys(const PagedAttention& p, int first, int pos, int key0, Word word)
{
    const int from = key0 - first;                                          // of the new tokens
    unsigned long long r = ~0ull;
    if (from >= 0)
    {
        r = word(from >> 6) >> (from & 63);
        if (from & 63) { r |= word((from >> 6) + 1) << (64 - (from & 63)); }
    }
    else if (from > -64) { r = word(0) << -from | ((1ull << -from) - 1); }
    if (p.window != 0)
    {
        // hidden: rows in front, from n_sink to pos - window
        const int lo = max(p.n_sink - key0, 0), hi = min(min(pos - p.window, first - 1) - key0, 63);
        if (lo <= hi) { r &= ~(~0ull >> (63 - hi) & ~0ull << lo); }
    }
    return r;
}

// Bits 64 i .. + 63 of a row of bits for n new tokens.
__device__ __forceinline__ unsigned long long seen_word(const unsigned long long* row, int n, int i)
{
    const int left = n - 64 * i;
    return left <= 0 ? 0ull : row[i] & (left >= 64 ? ~0ull : (1ull << left) - 1);
}

constexpr int PA_ROWS = 16, PA_TILE = 128, PA_TILE_KEYS = 64;

// Sequences of up to 16 rows per kv head: the keys of each in shares of four blocks (a block per wave), cut into parts of about the same number of shares, a
// workgroup each.  How many shares a part has follows from those of all sequences, so that long and short ones leave no workgroup with much more than
// another: about two workgroups' worth of an even split, since a part costs some 5 us besides its keys, but of that not over PA_PART, which evens out what is
// left over at the end.  At least what three rounds of parts leave, and what fits the parts that there is room for: with very many keys a part has more than PA_PART shares.
// (MI355X, 32 / 8 heads, E4M3, us.  Parts of a sequence 1 / 2 / 4, this rule: 16 of 4100 keys 34.9 / 30.2 / 31.2, 30.1; 8 of 4000 31.4 / 22.8 / 18.7, 18.7; 64 of 1000 to 8000
// with 1 / 3 / 6 on average 110.0 / 108.9 / 108.9, 107.2.  PA_PART 9 / 14 / 20 / 32: 64 of 1000 to 8000 110.2 / 106.8 / 107.4 / 112.4, 64 of 4500 103.2 / 103.0 / 94.8 / 94.9,
// 32 of 2000 to 4000 40.7 / 42.8 / 42.5 / 42.6, 16 of 500 to 16000 45.3 / 52.9 / 52.7 / 52.7, 4 of 32000 BF16 94.7 / 97.0 / 89.2 / 83.7, 64 BF16 190.7 / 188.3 / 191.4 / 194.3.
// 20 is right for a full batch; a few sequences of uneven lengths would like 9, a few of long ones 32: up to 16 % that one number does not give.)
constexpr int PA_PART = 20;

// The most sequences whose keys are cut into parts: more are a workgroup each, enough of them to fill the GPU, and nobody has to look at all of them.
// MI355X, 32 / 8 heads E4M3 us, cut / one each: 64 of 100 to 8000 103 / 105, 256 352 / 358, 256 of 200 to 2000 107 / 103; 8 / 1 heads, 100
// to 8000: 64 24 / 51, 128 35 / 52, 256 64 / 61.  Beyond, with a trip to memory for each 64 sequences: 512 of 200 to 2000 257 / 199, 1024 606 / 381.  A sequence much longer
// than the rest sets the time beyond: by itself 8000 / 32000 / 100000 rows take 48 / 180 / 545 us as a workgroup per kv head, 15 / 22 / 43 cut.
constexpr int PA_CUT_SEQS = 256;

template <int KEYS>
struct Parts
{
    int s = -1, part = 0, parts = 1, shares = 0;                            // part `part` of the `parts` that the shares of sequence s are in; s < 0: none
    NewTokens mine = { 0, 0, 0 };

    __device__ __forceinline__ static KeyBlocks<KEYS> keys(const PagedAttention& p, const NewTokens& n) { return KeyBlocks<KEYS>(p, n.pos, n.pos + n.n - 1); }
    __device__ __forceinline__ static int shares_of(const PagedAttention& p, const NewTokens& n)
    {
        const int rows = n.n * p.group;
        return rows == 0 || rows > PA_ROWS ? 0 : max((keys(p, n).n + 3) / 4, 1);
    }
    // Part c of all.  Whole waves, four sequences per lane.
    __device__ __forceinline__ Parts(const PagedArgs& a, const PagedAttention& p, int c)
    {
        constexpr int BATCHES = PA_CUT_SEQS / 64;
        const int lane = threadIdx.x & 63;
        SeqWords words[BATCHES];
        NewTokens tokens[BATCHES];
        int have[BATCHES], total = 0;
        words[0] = SeqWords(a, lane);
        if (a.n_seqs > 64)
        {
#pragma unroll
            for (int b = 1; b < BATCHES; b++) { words[b] = SeqWords(a, 64 * b + lane); }
        }
#pragma unroll
        for (int b = 0; b < BATCHES; b++)
        {
            if (b != 0 && a.n_seqs <= 64 * b) { break; }
            tokens[b] = words[b].tokens(a, p, 64 * b + lane);
            have[b] = shares_of(p, tokens[b]);
            total += __builtin_amdgcn_readlane(add_up_lanes(have[b]), 63);
        }
        auto split = [&](int n) { return (total + n - 1) / n; };
        int per = max(max(split(3 * p.row_slots), min(PA_PART, split((p.row_slots + 1) / 2))), KEYS == 32 ? 2 : 1);
        per = max(per, split(max(p.row_parts - a.n_seqs, 1)));              // no more parts than workgroups
        int before = 0;
#pragma unroll
        for (int b = 0; b < BATCHES; b++)
        {
            if (b != 0 && a.n_seqs <= 64 * b) { break; }
            const int n = (have[b] + per - 1) / per, upto = before + add_up_lanes(n);
            const unsigned long long past = __ballot(upto > c);
            if (past != 0)
            {
                const int of = __builtin_ctzll(past);
                s = 64 * b + of;
                parts = __builtin_amdgcn_readlane(n, of);
                part = c - (__builtin_amdgcn_readlane(upto, of) - parts);
                shares = __builtin_amdgcn_readlane(have[b], of);
                mine = { __builtin_amdgcn_readlane(tokens[b].first, of), __builtin_amdgcn_readlane(tokens[b].n, of), __builtin_amdgcn_readlane(tokens[b].pos, of) };
                break;
            }
            before = __builtin_amdgcn_readlane(upto, 63);
        }
    }
};

// A tile: rows row0 .. + 127 of sequence s (< 0: none), the positions of their tokens and the keys they see, in n_ranges ranges of `per` blocks.
// Of trees: the range that workgroup `tile` has of it, and where the sums of its first range go.
struct Tile
{
    int s = -1, row0 = 0, n_rows = 0, lo = 0, hi = 0, per = 1, n_ranges = 1, range = 0, piece0 = 0;
    NewTokens mine = { 0, 0, 0 };
    KeyBlocks<PA_TILE_KEYS> blocks;
};

// Tile `tile` of those of all sequences, a sequence's last ones first: they see the most keys.  Where a CU gets two workgroups in all, the second half of
// the tiles comes in the other order, so that a long one has a short one beside it (MI355X, 512 tiles of 2048 tokens behind 6000: 249 us for 256; with more
// tiles than that a CU takes the next one when it is done, and the order from long to short is the better one: 2000 tiles of four prompts 142 us for 146).  Called by whole waves: a lane per
// sequence, 256 of them per trip to memory, their tiles added up.
__device__ __forceinline__ Tile find_tile(const PagedArgs& a, const PagedAttention& p, int tile)
{
    Tile r;
    const int lane = threadIdx.x & 63;
    if (p.snake && tile >= (p.tiles + 1) / 2) { tile = p.tiles - 1 - (tile - (p.tiles + 1) / 2); }
    for (int base = 0; base < a.n_seqs; base += 256)
    {
        SeqWords words[4];                                                  // of 256 sequences, in one trip
        words[0] = SeqWords(a, base + lane);
        if (base + 64 < a.n_seqs)
        {
#pragma unroll
            for (int b = 1; b < 4; b++) { words[b] = SeqWords(a, base + 64 * b + lane); }
        }
#pragma unroll
        for (int b = 0; b < 4; b++)
        {
            if (base + 64 * b >= a.n_seqs) { break; }
            const NewTokens mine = words[b].tokens(a, p, base + 64 * b + lane);
            const int rows = mine.n * p.group, tiles = rows > p.min_rows ? (rows + PA_TILE - 1) / PA_TILE : 0;
            const int upto = add_up_lanes(tiles);
            const unsigned long long past = __ballot(upto > tile);
            if (past != 0)
            {
                const int at = __builtin_ctzll(past);
                r.s = uniform(base + 64 * b + at);
                r.mine = { __builtin_amdgcn_readlane(mine.first, at), __builtin_amdgcn_readlane(mine.n, at), __builtin_amdgcn_readlane(mine.pos, at) };
                r.row0 = uniform(__builtin_amdgcn_readlane(upto, at) - 1 - tile) * PA_TILE;
                break;
            }
            tile -= __builtin_amdgcn_readlane(upto, 63);
        }
        if (r.s >= 0) { break; }
    }
    if (r.s < 0) { return r; }
    r.n_rows = uniform(r.mine.n * p.group);
    r.lo = uniform(r.mine.pos + r.row0 / p.group);
    r.hi = uniform(r.mine.pos + min(r.row0 + PA_TILE - 1, r.n_rows - 1) / p.group);
    r.blocks = KeyBlocks<PA_TILE_KEYS>(p, r.lo, r.hi);
    r.blocks.n = uniform(r.blocks.n);
    r.blocks.sinks = uniform(r.blocks.sinks);
    r.blocks.skip = uniform(r.blocks.skip);
    r.per = max((r.blocks.n + p.tile_split - 1) / p.tile_split, 4);
    r.n_ranges = max((r.blocks.n + r.per - 1) / r.per, 1);
    return r;
}

// Trees: piece `piece` of all tiles' ranges of keys.  All of a sequence's tiles see the same blocks, so that lengths alone say how many pieces there are.  Every range is of about the same length, which follows from
// all sequences: the shortest, from an even split over the workgroups that run at once, with which there are no more pieces than those (a piece costs 5 us besides its 2.15 per block, and its sums are written and read), but
// at least PIECE_LEAST blocks.  With more than 256 sequences, or tiles enough, it is the even split.  MI355X us, attention + the launch that adds, 32 / 8 heads of 128 E4M3, 32 sequences of 17 to 33 tokens on 1000 to 8000
// rows: as many ranges for short ones as for long ones 150 + 10, these 120 + 11.
// ADDED: tile `piece` of those in several ranges, with the length that the attention's first workgroup left.
constexpr int PIECE_LEAST = 4;

template <bool ADDED>
__device__ __forceinline__ Tile find_piece(const PagedArgs& a, const PagedAttention& p, int piece)
{
    Tile r;
    const int lane = threadIdx.x & 63;
    SeqWords words[4];
    NewTokens mine[4];
    int tiles[4], blocks[4];
    auto read = [&](int base) {                                             // 256 sequences
        words[0] = SeqWords(a, base + lane);
        if (base + 64 < a.n_seqs)
        {
#pragma unroll
            for (int b = 1; b < 4; b++) { words[b] = SeqWords(a, base + 64 * b + lane); }
        }
#pragma unroll
        for (int b = 0; b < 4; b++)
        {
            if (b != 0 && base + 64 * b >= a.n_seqs)
            {
                tiles[b] = blocks[b] = 0;
                continue;
            }
            mine[b] = words[b].tokens(a, p, base + 64 * b + lane);
            const int rows = mine[b].n * p.group;
            tiles[b] = rows > p.min_rows ? (rows + PA_TILE - 1) / PA_TILE : 0;
            blocks[b] = tiles[b] > 0 ? KeyBlocks<PA_TILE_KEYS>(p, mine[b].pos, mine[b].pos + mine[b].n - 1).n : 0;
        }
    };
    // ranges of `per` blocks, or so (the same for whoever asks)
    auto ranges_of = [](int n, float by) { return max((int)ceilf(fmaf((float)n, by, -0.001f)), 1); };
    float by = 0.0f;                                                        // 1 / per
    const float left = ADDED ? *p.piece_length() : 0.0f;
    read(0);
    if (ADDED) { by = left; }
    else if (p.piece_slots > 0)
    {
        float all = 0.0f;
        int n_tiles = 0;
        for (int base = 0; base < a.n_seqs; base += 256)
        {
            if (base != 0) { read(base); }
#pragma unroll
            for (int b = 0; b < 4; b++)
            {
                all += (float)tiles[b] * (float)blocks[b];
                n_tiles += tiles[b];
            }
        }
        if (a.n_seqs > 256) { read(0); }
        all = reduce_lanes<16>(all, [](float u, float v) { return u + v; });
        all = (__shfl(all, 0) + __shfl(all, 16)) + (__shfl(all, 32) + __shfl(all, 48));
        n_tiles = __builtin_amdgcn_readlane(add_up_lanes(n_tiles), 63);
        // (the sum's rounding counts upwards)
        float per = fmaxf(all * 1.001f / (float)p.piece_slots, (float)PIECE_LEAST);
        if (a.n_seqs <= 256 && n_tiles <= p.piece_slots)
        {
            auto fits = [&](float per) {
                int pieces = 0;
#pragma unroll
                for (int b = 0; b < 4; b++) { pieces += tiles[b] * ranges_of(blocks[b], __builtin_amdgcn_rcpf(per)); }
                return __builtin_amdgcn_readlane(add_up_lanes(pieces), 63) <= p.piece_slots;
            };
            for (int n = 0; n < 40 && !fits(per); n++) { per *= n < 10 ? 1.06f : 1.3f; }
        }
        by = __builtin_amdgcn_rcpf(per);
        if (blockIdx.x == 0 && threadIdx.x == 0) { *p.piece_length() = by; }
    }
    int before = 0, split_before = 0;
    for (int base = 0; base < a.n_seqs; base += 256)
    {
        if (base != 0) { read(base); }
#pragma unroll
        for (int b = 0; b < 4; b++)
        {
            if (base + 64 * b >= a.n_seqs) { break; }
            const int ranges = ranges_of(blocks[b], by), split_upto = split_before + add_up_lanes(ranges > 1 ? tiles[b] * ranges : 0);
            const int upto = before + add_up_lanes(!ADDED ? tiles[b] * ranges : ranges > 1 ? tiles[b] : 0);
            const unsigned long long past = __ballot(upto > piece);
            if (past != 0)
            {
                const int at = __builtin_ctzll(past);
                r.s = uniform(base + 64 * b + at);
                r.mine = { __builtin_amdgcn_readlane(mine[b].first, at), __builtin_amdgcn_readlane(mine[b].n, at), __builtin_amdgcn_readlane(mine[b].pos, at) };
                r.n_ranges = __builtin_amdgcn_readlane(ranges, at);
                const int back = __builtin_amdgcn_readlane(upto, at) - 1 - piece, tile = ADDED ? back : back / r.n_ranges;
                r.range = ADDED ? 0 : r.n_ranges - 1 - back % r.n_ranges;
                r.piece0 = uniform(__builtin_amdgcn_readlane(split_upto, at) - (tile + 1) * r.n_ranges);
                r.row0 = uniform(tile) * PA_TILE;
                break;
            }
            before = __builtin_amdgcn_readlane(upto, 63);
            split_before = __builtin_amdgcn_readlane(split_upto, 63);
        }
        if (r.s >= 0) { break; }
    }
    if (r.s < 0) { return r; }
    r.n_rows = uniform(r.mine.n * p.group);
    r.lo = uniform(r.mine.pos);
    r.hi = uniform(r.mine.pos + r.mine.n - 1);
    r.blocks = KeyBlocks<PA_TILE_KEYS>(p, r.lo, r.hi);
    r.blocks.n = uniform(r.blocks.n);
    r.blocks.sinks = uniform(r.blocks.sinks);
    r.blocks.skip = uniform(r.blocks.skip);
    r.n_ranges = uniform(r.n_ranges);
    r.range = uniform(r.range);
    r.per = (r.blocks.n + r.n_ranges - 1) / r.n_ranges;
    return r;
}

// The weights' running maximum moves only when a score exceeds it by more than this (in log2): until then they are at most 2^8, which FP32 sums
// and BF16's exponent do not notice, and the sums are left alone.
constexpr float PA_LAG = 8.0f;

// Workgroup barrier that orders LDS traffic only: __syncthreads() waits for the loads in flight too.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

typedef short pa_b16x4 __attribute__((ext_vector_type(4)));
typedef int pa_b32x2 __attribute__((ext_vector_type(2)));

// Transposing reads of LDS, by 16 lanes each.  16 bits: lane i points at 4 elements of row i / 4, piece i % 4, and receives element i of the 4 rows.
__device__ __forceinline__ u32x2 lds_transposed16(const uint8_t* at)
{
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_b16x4*)at));
}

// 8 bits: lane i points at 8 elements of row i / 2, piece i % 2, and receives element i of the 8 rows.
__device__ __forceinline__ u32x2 lds_transposed8(const uint8_t* at)
{
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) pa_b32x2*)at));
}

__device__ __forceinline__ uint32_t lds_offset(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p; }

// Loads from memory into LDS; whoever reads waits for them.  Unless `wanted` is 0, a KiB from base + off:
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void kib_to_lds(uint32_t wanted, uint32_t lds, const uint8_t* base, uint32_t off)
{
    asm volatile("s_cmp_eq_u32 %0, 0\n\ts_cbranch_scc1 .Lkib_to_lds%=\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n.Lkib_to_lds%=:"
                 : : "s"(wanted), "s"(lds), "v"(off), "s"(base) : "memory", "m0", "scc");
}
// N KiB in a row, lane l's 16 bytes of the n-th at off[n] (the instruction's own offset counts on both sides).
template <int N>
__device__ __forceinline__ void kibs_to_lds(uint32_t lds, const uint8_t* base, const uint32_t (&off)[N])
{
    static_assert(N == 1 || N == 2 || N == 4, "16 rows");
    if constexpr (N == 1) { asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" : : "s"(lds), "v"(off[0]), "s"(base) : "memory", "m0"); }
    else if constexpr (N == 2)
    {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3 nt\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024 nt"
                     : : "s"(lds), "v"(off[0]), "v"(off[1]), "s"(base) : "memory", "m0");
    }
    else
    {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5 nt\n\tglobal_load_lds_dwordx4 %2, %5 offset:1024 nt\n\t"
                     "global_load_lds_dwordx4 %3, %5 offset:2048 nt\n\tglobal_load_lds_dwordx4 %4, %5 offset:3072 nt"
                     : : "s"(lds), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base) : "memory", "m0");
    }
}
// a byte per lane to a dword per lane:
__device__ __forceinline__ void bytes_to_lds(uint32_t lds, const uint8_t* at)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" : : "s"(lds), "v"(at) : "memory", "m0");
}
#pragma clang diagnostic pop

// Bits of a dword's two BF16 values that are infinite or NaN, as a mask over both; and whether there are any in four dwords.
__device__ __forceinline__ uint32_t not_finite(uint32_t w)
{
    return (((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u);
}
__device__ __forceinline__ uint32_t not_finite(const u32x4& v) { return not_finite(v[0]) | not_finite(v[1]) | not_finite(v[2]) | not_finite(v[3]); }

// The same with zeros there.
__device__ __forceinline__ u32x4 finite_part(const u32x4& v)
{
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) { r[i] = v[i] & ~((not_finite(v[i]) >> 15) * 0xFFFFu); }
    return r;
}

// Bit 7 of each byte of a dword that is an infinite or NaN code.
template <int TYPE>
__device__ __forceinline__ uint32_t codes_not_finite(uint32_t w)
{
    if constexpr (TYPE == DT_E4M3) { return (w & 0x7F7F7F7Fu) + 0x01010101u & 0x80808080u; }
    else { return (w & 0x7C7C7C7Cu) + 0x04040404u & 0x80808080u; }
}

// Parts pass between workgroups of different XCDs, whose L2s do not know of each other: they are written through and read past them by relaxed atomics of the
// device's scope.  (Plain stores between fences, which write back and drop a whole L2, cost 15 us and more a call.)
__device__ __forceinline__ void store_part(float* to, float x, float y)
{
    __hip_atomic_store((unsigned long long*)to, (unsigned long long)f32_to_bits(y) << 32 | f32_to_bits(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_part(const float* from)
{
    const unsigned long long v = __hip_atomic_load((const unsigned long long*)from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(bits_to_f32((uint32_t)v), bits_to_f32((uint32_t)(v >> 32)));
}

// Whether the n parts that belong together are all there, this workgroup's own, just stored, among them.  A part is there when its word holds the name of this
// call, whatever lay there before; flag(i) is the i-th one's word, `own` this workgroup's.  Each workgroup sets its word and then looks at all of them, so at least the
// last one finds them set; where several do, all write the same result.  (A counter instead, with a compare and swap per workgroup, took 0.8 us for each.)
template <class Flag>
__device__ __forceinline__ bool all_there(unsigned long long* own, unsigned long long call, int n, uint32_t* lds_result, Flag flag)
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                        // the wave's stores are there
    __syncthreads();
    if (threadIdx.x < 64)
    {
        if (threadIdx.x == 0) { __hip_atomic_store(own, call, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        bool all = true;
        for (int i = threadIdx.x; i < n; i += 64) { all = all && __hip_atomic_load(flag(i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == call; }
        all = __all(all);
        if (threadIdx.x == 0) { *lds_result = all; }
    }
    __syncthreads();
    return *lds_result != 0;
}

// DIM / 16 dims of a row from its n parts: rescaled to the largest maximum, added in order, divided by the sum of the weights, one rounding.
// part(i, sums, stat) tells where the i-th one's sums and (max, sum) are.  PLAIN: parts of an earlier launch.
template <int DIM, bool PLAIN = false, class Part>
__device__ __forceinline__ void add_parts(int n, uint16_t* y, Part part)
{
    constexpr int PER = DIM / 16, AT_ONCE = PLAIN ? 4 : 8;
    float sum[PER] = {};
    float m = -INFINITY, l = 0.0f;
    for (int r0 = 0; r0 < n; r0 += AT_ONCE)
    {
        float2 v[AT_ONCE][PER / 2], stat[AT_ONCE];                          // parts requested at once
#pragma unroll
        for (int r = 0; r < AT_ONCE; r++)
        {
            const float *from, *at;
            part(min(r0 + r, n - 1), from, at);
            stat[r] = PLAIN ? *(const float2*)at : load_part(at);
#pragma unroll
            for (int d = 0; d < PER / 2; d += 2)
            {
                if (PLAIN)
                {
                    const f32x4 four = *(const f32x4*)(from + 2 * d);
                    v[r][d] = make_float2(four[0], four[1]);
                    v[r][d + 1] = make_float2(four[2], four[3]);
                }
                else
                {
                    v[r][d] = load_part(from + 2 * d);
                    v[r][d + 1] = load_part(from + 2 * d + 2);
                }
            }
        }
        float top = m;
#pragma unroll
        for (int r = 0; r < AT_ONCE; r++) { top = fmaxf(top, stat[r].x); }
        const float base = top > -INFINITY ? top : 0.0f, shrink = __builtin_amdgcn_exp2f(m - base);
        m = top;
        l *= shrink;
#pragma unroll
        for (int d = 0; d < PER; d++) { sum[d] *= shrink; }
#pragma unroll
        for (int r = 0; r < AT_ONCE; r++)
        {
            const float w = __builtin_amdgcn_exp2f(stat[r].x - base);
            if (r0 + r < n)                                                 // also with weight 0: a part without a key has sums of 0, one with infinities or NaN makes them NaN
            {
                l += w * stat[r].y;                                         // NaN where a score is, also if all are: the maximum is then minus infinity, the weight 0
#pragma unroll
                for (int d = 0; d < PER; d++) { sum[d] += w * (d % 2 ? v[r][d / 2].y : v[r][d / 2].x); }
            }
        }
    }
#pragma unroll
    for (int d = 0; d < PER; d++) { sum[d] = l == 0.0f ? 0.0f : sum[d] / l; }
#pragma unroll
    for (int d = 0; d < PER; d += 4) { *(u32x2*)(y + d) = pack4(sum + d); }
}

// Up to 16 rows of a kv head: single tokens, or a few.  Bound by the cached rows' way from memory: 64 sequences of 1000 to 8000 E4M3 rows 108 us, 5.4 TB/s (a large
// copy: 5.1); few or short ones by the chain of launch, place, page, row, flags and parts: one sequence of 4096 BF16 rows 13 us, of which the rows' way takes 3.
//   A workgroup of four waves takes a range of the sequence's blocks of KEYS keys, a wave every fourth block, each with a pipeline of its own: rows go by
// direct loads to the wave's part of LDS, keys and values STAGES blocks ahead each, and nothing but the wave's own count of loads in flight is waited for.
//   scores: v_mfma_f32_16x16x32_bf16, key rows as row operand, the 16 queries as columns: D lane (row j = lane % 16, g = lane / 16) holds keys 4 g .. + 3
//           of 16.  FP8 keys become BF16 in registers, times their power of two (a lane's operand is one key's): exact.
//   V p:    the eight weights of a lane in 32 keys (4 g .. + 3 and 16 + 4 g .. + 3) are its column operand as they are; the row operand (dim, the same
//           keys) comes from transposing reads.  FP8 values' powers of two go to the weights.
// Weights are rounded to BF16 for that product, their sum is of the FP32 ones: the matrix cores' FP32 product has a sixteenth of BF16's rate.  At most half a step, 2^-8 of a weight, errors of both signs: trees of 4
// to 60 tokens differ from 64 bits by 2.2e-3 - 2.3e-3 of the results' size, where FP32 weights leave the 1.7e-3 of the results' own rounding.
// Rows are read once per kv head and kept out of the way of what is read again (nt): 64 sequences 114 us for 124 without.
// LDS: chunk c (16 bytes) of row r lies at c ^ swizzle(r), so that the operand reads hit all banks.
template <int TYPE, int DIM>
struct RowsForm
{
    static constexpr int ROW = DIM * CODE_BYTES<TYPE>, KEYS = ROW == 256 ? 32 : 64, STAGES = ROW == 64 ? 2 : 1;
    static constexpr int SIDE = KEYS * ROW, EXPONENTS = TYPE == DT_BF16 ? 0 : 2 * KEYS * 4, WAVE = STAGES * (2 * SIDE + EXPONENTS);
    static constexpr int SUM = DIM + 4;                                     // floats per row of the sums
    static constexpr int STAT = 4 * (WAVE > PA_ROWS * SUM * 4 ? WAVE : PA_ROWS * SUM * 4), LDS = STAT + 4 * PA_ROWS * 8;
};

template <int TYPE, int DIM, bool TREE>
__device__ __forceinline__ void attend_rows(const PagedArgs& a, const PagedAttention& p, uint8_t* lds, int s, const NewTokens& mine, int kvh, int from_share, int to_share, int slot, int part, int n_parts)
{
    typedef RowsForm<TYPE, DIM> F;
    constexpr int KEYS = F::KEYS, STAGES = F::STAGES, ROW = F::ROW, SIDE = F::SIDE, SUM = F::SUM, CHUNKS = ROW / 16;
    constexpr int TILES = KEYS / 16, LOADS = SIDE / 1024, PART_LOADS = LOADS / TILES, KEY_LOADS = LOADS + (TYPE == DT_BF16 ? 0 : 2);
    float2* const stat = (float2*)(lds + F::STAT);                          // [wave][row] (max, sum)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int j = lane & 15, g = lane >> 4;
    const auto blocks = Parts<KEYS>::keys(p, mine);
    const int n_rows = uniform(mine.n * p.group), lo = uniform(mine.pos), hi = uniform(mine.pos + mine.n - 1);
    const int begin = from_share * 4, end = uniform(min(blocks.n, to_share * 4));

    const int row = min(j, n_rows - 1), token = row / p.group, head = kvh * p.group + row % p.group;
    const int my_pos = mine.pos + token;
    // trees: what the row's token sees of the new ones, 16 at most; asked for here, there with the first pages, before the counted loads
    int seen_pos = 0;
    uint32_t new_seen = 0;
    if constexpr (TREE) { new_seen = (uint32_t)p.seen[(size_t)(mine.first + token) * p.seen_stride] & ((1u << mine.n) - 1); }
    u32x4 qf[DIM / 32];                                                     // elements 32 c + 8 g .. + 7
#pragma unroll
    for (int c = 0; c < DIM / 32; c++) { qf[c] = *(const u32x4*)(p.q + (size_t)(mine.first + token) * p.ldq + (size_t)head * DIM + c * 32 + g * 8); }

    auto key_swizzle = [](int r) { return r / (256 / ROW) % CHUNKS; };
    auto value_swizzle = [](int r) {
        if constexpr (TYPE == DT_BF16) { return DIM == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); }
        else { return DIM == 128 ? ((r >> 1) & 3) | ((r >> 4) & 1) << 2 : ((r >> 2) & 1) | ((r >> 4) & 1) << 1; }
    };
    // the wave's LDS: key blocks, value blocks, exponents (keys', then values')
    uint8_t* const my_lds = lds + wave * F::WAVE;
    const uint32_t my_lds0 = __builtin_amdgcn_readfirstlane(lds_offset(my_lds));
    constexpr int VALUES = STAGES * SIDE, EXPONENTS = 2 * VALUES;
    // the wave's n-th block of the range is list entry begin + wave + 4 n
    const int n_mine = begin + wave < end ? (end - begin - wave + 3) / 4 : 0;
    // lane l: where rows 16 (l % TILES) .. + 15 of the wave's block k 64 / TILES + l / TILES begin in the pool (and their exponents); bit 63: they have no page
    constexpr int BATCH = 64 / TILES;
    size_t rows_from = 0, exponents_from = 0;
    auto look_up = [&](int n0) {
        const int i = begin + wave + 4 * (n0 + lane / TILES);
        const int pos = blocks.block(i) * KEYS + 16 * (lane % TILES);
        const int page = i >= end || pos > hi ? 0 : paged_page(a, s, pos);
        const size_t r0 = paged_row(a, kvh, pos);
        rows_from = max(page, 0) * a.page_stride + r0 * ROW | (page < 0 ? (size_t)1 << 63 : 0);
        exponents_from = max(page, 0) * a.scale_stride + r0;
    };
    auto of_part = [&](size_t v, int n, int part) {
        const int at = n % BATCH * TILES + part;
        return (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), at) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, at);
    };
    const uint32_t key_off = lane * 16 ^ key_swizzle(lane / CHUNKS) * 16, value_off = lane * 16 ^ value_swizzle(lane / CHUNKS) * 16;
    auto stage = [&](int n, bool values) {
#pragma unroll
        for (int part = 0; part < TILES; part++)
        {
            const size_t from = of_part(rows_from, n, part) & ~((size_t)1 << 63);
            uint32_t off[PART_LOADS];
#pragma unroll
            for (int i = 0; i < PART_LOADS; i++)
            {
                // row 16 part + i 1024 / ROW + lane / CHUNKS: the first two terms change bits of the swizzle that the lane's row does not reach
                const int r = 16 * part + i * (1024 / ROW);
                off[i] = values ? value_off ^ (uint32_t)(value_swizzle(r) * 16) : key_off ^ (uint32_t)(key_swizzle(r) * 16);
            }
            kibs_to_lds(my_lds0 + (values ? VALUES : 0) + n % STAGES * SIDE + part * 16 * ROW, (values ? a.v : a.k) + from, off);
        }
        if constexpr (TYPE != DT_BF16)
        {
            if (!values)
            {
                // lane l: the exponent of row l
                const int at = n % BATCH * TILES + g;
                const size_t from = (size_t)(uint32_t)__shfl((int)(exponents_from >> 32), at) << 32 | (uint32_t)__shfl((int)exponents_from, at);
                bytes_to_lds(my_lds0 + EXPONENTS + n % STAGES * F::EXPONENTS, a.k_scale + from + j);
                bytes_to_lds(my_lds0 + EXPONENTS + n % STAGES * F::EXPONENTS + KEYS * 4, a.v_scale + from + j);
            }
        }
    };
    // list entries plain_from .. plain_to - 1: every row sees every key
    int plain_from = 0, plain_to = (TREE ? max(lo, 0) : lo + 1) / KEYS;
    if (p.window != 0) { plain_from = (hi - p.window + KEYS) / KEYS; }
    plain_from = uniform(max(plain_from - blocks.skip, hi < p.window || p.window == 0 ? 0 : blocks.sinks));
    plain_to = uniform(plain_to - blocks.skip);

    float m = -INFINITY, l = 0.0f;
    f32x4 out[DIM / 16];
#pragma unroll
    for (int d = 0; d < DIM / 16; d++) { out[d] = f32x4{ 0.0f, 0.0f, 0.0f, 0.0f }; }

    // which 16 rows of block n have no page
    auto lacks_of = [&](int n) {
        int lacks = 0;
#pragma unroll
        for (int part = 0; part < TILES; part++) { lacks |= (int)((uint32_t)__builtin_amdgcn_readlane((int)(rows_from >> 32), n % BATCH * TILES + part) >> 31) << part; }
        return lacks;
    };
    int kept = 0;
    // trees: which keys of a block the row sees
    auto keys_seen = [&](int key0) { return named_keys(p, mine.pos, seen_pos, key0, [&](int i) { return i == 0 ? (unsigned long long)new_seen : 0ull; }); };

    auto block = [&](int n) {
        const uint8_t* const kb = my_lds + n % STAGES * SIDE;
        const uint8_t* const vb = my_lds + VALUES + n % STAGES * SIDE;
        const uint8_t* const exponents = my_lds + EXPONENTS + n % STAGES * F::EXPONENTS;
        const int entry = begin + wave + 4 * n;
        const int lacks = STAGES == 2 && n % BATCH == BATCH - 1 && n + 1 < n_mine ? kept : lacks_of(n);
        // what was asked for behind the keys of n may still be on its way
        if (STAGES == 2 && n + 1 < n_mine) { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * LOADS + KEY_LOADS) : "memory"); }
        else { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LOADS) : "memory"); }
        f32x4 acc[TILES];
        u32x4 value_exponents[TILES];
#pragma unroll
        for (int kt = 0; kt < TILES; kt++)
        {
            acc[kt] = f32x4{ 0.0f, 0.0f, 0.0f, 0.0f };
            const int r = 16 * kt + j;
            float kscale = 1.0f;
            if constexpr (TYPE != DT_BF16)
            {
                kscale = bits_to_f32(*(const uint32_t*)(exponents + r * 4) << 23);
                value_exponents[kt] = *(const u32x4*)(exponents + KEYS * 4 + (16 * kt + 4 * g) * 4);
            }
#pragma unroll
            for (int c = 0; c < DIM / 32; c++)
            {
                u32x4 kf;
                if constexpr (TYPE == DT_BF16) { kf = *(const u32x4*)(kb + r * ROW + ((4 * c + g) ^ key_swizzle(r)) * 16); }
                else
                {
                    const u32x2 codes = *(const u32x2*)(kb + r * ROW + ((2 * c + (g >> 1)) ^ key_swizzle(r)) * 16 + (g & 1) * 8);
                    const u32x2 lo = fp8x4_to_bf16<TYPE>(codes[0], kscale), hi = fp8x4_to_bf16<TYPE>(codes[1], kscale);
                    kf = u32x4{ lo[0], lo[1], hi[0], hi[1] };
                }
                acc[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf), __builtin_bit_cast(bf16x8, qf[c]), acc[kt], 0, 0, 0);
            }
        }
        if (n + STAGES < n_mine)
        {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");           // the keys have been read
            if ((n + STAGES) % BATCH == 0)
            {
                if (STAGES == 2) { kept = lacks_of(n + 1); }               // the one block whose place in the list is overwritten before its turn
                look_up(n + STAGES);
            }
            stage(n + STAGES, false);
        }
        if (STAGES == 2 && n + 2 < n_mine) { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LOADS + 2 * KEY_LOADS) : "memory"); }
        else if (STAGES == 2 && n + 1 < n_mine) { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LOADS + KEY_LOADS) : "memory"); }
        else if (STAGES == 1 && n + 1 < n_mine) { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(KEY_LOADS) : "memory"); }
        else { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }
        // values as they lie there: eight of a dim, BF16 or codes
        constexpr int WORDS = TYPE == DT_BF16 ? 4 : 2, STEPS = TILES / 2;
        uint32_t raw[STEPS][DIM / 16][WORDS];
#pragma unroll
        for (int u = 0; u < STEPS; u++)
#pragma unroll
            for (int d = 0; d < DIM / 16; d++)
            {
                if constexpr (TYPE == DT_BF16)
                {
                    const int r = 32 * u + 4 * g + (j >> 2);
                    const uint8_t* const at0 = vb + r * ROW + (((2 * d + ((j & 3) >> 1)) ^ value_swizzle(r)) << 4) + ((j & 1) << 3);
                    const u32x2 lo = lds_transposed16(at0), hi = lds_transposed16(at0 + 16 * ROW);      // the swizzle of row r + 16 is that of r
                    raw[u][d][0] = lo[0], raw[u][d][1] = lo[1], raw[u][d][2] = hi[0], raw[u][d][3] = hi[1];
                }
                else
                {
                    const int r = 32 * u + 4 * g + ((j >> 1) & 3) + (j >> 3) * 16;
                    const u32x2 codes = lds_transposed8(vb + r * ROW + ((d ^ value_swizzle(r)) << 4) + ((j & 1) << 3));
                    raw[u][d][0] = codes[0], raw[u][d][1] = codes[1];
                }
            }
        auto values = [&](int u, int d) {
            if constexpr (TYPE == DT_BF16) { return u32x4{ raw[u][d][0], raw[u][d][1], raw[u][d][2], raw[u][d][3] }; }
            else
            {
                const u32x2 lo = fp8x4_to_bf16<TYPE>(raw[u][d][0], 1.0f), hi = fp8x4_to_bf16<TYPE>(raw[u][d][1], 1.0f);
                return u32x4{ lo[0], lo[1], hi[0], hi[1] };
            }
        };
        const bool plain = entry >= plain_from && entry < plain_to && lacks == 0;
        if (!plain)
        {
            const int b = blocks.block(entry);
            unsigned long long bits = 0;
            if constexpr (TREE) { bits = keys_seen(b * KEYS); }
#pragma unroll
            for (int e = 0; e < 4 * TILES; e++)
            {
                const int at = 16 * (e >> 2) + 4 * g + (e & 3);
                const bool see = (TREE ? (bits >> at & 1) != 0 : sees(p, my_pos, b * KEYS + at)) && !(lacks >> (e >> 2) & 1);
                acc[e >> 2][e & 3] = see ? acc[e >> 2][e & 3] : -INFINITY;
                if constexpr (TYPE != DT_BF16) { value_exponents[e >> 2][e & 3] = see ? value_exponents[e >> 2][e & 3] : 0; }     // one that nobody wrote may be an infinity's
            }
            // Weight 0 times an infinity is NaN: what is infinite or NaN is added to the sums of the rows that see it and cleared in front of the products.
            uint32_t odd = 0;
#pragma unroll
            for (int u = 0; u < STEPS; u++)
#pragma unroll
                for (int d = 0; d < DIM / 16; d++)
#pragma unroll
                    for (int i = 0; i < WORDS; i++) { odd |= TYPE == DT_BF16 ? not_finite(raw[u][d][i]) : codes_not_finite<TYPE>(raw[u][d][i]); }
            if (__any(odd != 0))
            {
#pragma unroll 1
                for (int key = 0; key < KEYS; key++)
                {
                    const bool see = (TREE ? (bits >> key & 1) != 0 : sees(p, my_pos, b * KEYS + key)) && !(lacks >> (key / 16) & 1);
#pragma unroll
                    for (int d = 0; d < DIM / 16; d++)
                    {
                        // dims 16 d + 4 g .. + 3
                        const int byte = (16 * d + 4 * g) * CODE_BYTES<TYPE>;
                        const uint8_t* const from = vb + key * ROW + ((byte / 16 ^ value_swizzle(key)) << 4) + byte % 16;
                        u32x2 w;
                        if constexpr (TYPE == DT_BF16) { w = *(const u32x2*)from; }
                        else { w = fp8x4_to_bf16<TYPE>(*(const uint32_t*)from, 1.0f); }
                        float v[4];
                        unpack4(w, v);
#pragma unroll
                        for (int e = 0; e < 4; e++) { out[d][e] += see && !(fabsf(v[e]) < INFINITY) ? v[e] : 0.0f; }
                    }
                }
#pragma unroll
                for (int u = 0; u < STEPS; u++)
#pragma unroll
                    for (int d = 0; d < DIM / 16; d++)
#pragma unroll
                        for (int i = 0; i < WORDS; i++)
                        {
                            const uint32_t w = raw[u][d][i];
                            raw[u][d][i] = w & ~(TYPE == DT_BF16 ? (not_finite(w) >> 15) * 0xFFFFu : (codes_not_finite<TYPE>(w) >> 7) * 0xFFu);
                        }
            }
        }
        if (n + STAGES < n_mine)
        {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");           // the values have been read
            stage(n + STAGES, true);
        }
        float top = acc[0][0];
#pragma unroll
        for (int e = 1; e < 4 * TILES; e++) { top = fmaxf(top, acc[e >> 2][e & 3]); }
        top *= p.scale;
        if (__any(top > m + PA_LAG))
        {
            top = fmaxf(top, __shfl_xor(top, 16));
            const float next = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
            const float shrink = m > -INFINITY ? __builtin_amdgcn_exp2f(m - next) : 1.0f;         // sums of nothing: 0, or what is not finite
            m = next;
            l *= shrink;
#pragma unroll
            for (int d = 0; d < DIM / 16; d++) { out[d] *= shrink; }
        }
        const float off = m > -INFINITY ? -m : 0.0f;                        // no key seen yet: every weight is 2^-inf = 0
        float sum[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
        bf16x8 pb[STEPS];
#pragma unroll
        for (int e = 0; e < 4 * TILES; e++)
        {
            float w = __builtin_amdgcn_exp2f(fmaf(acc[e >> 2][e & 3], p.scale, off));
            sum[e & 3] += w;
            if constexpr (TYPE != DT_BF16) { w *= bits_to_f32(value_exponents[e >> 2][e & 3] << 23); }
            pb[e >> 3][e & 7] = (__bf16)w;
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int u = 0; u < STEPS; u++)
#pragma unroll
            for (int d = 0; d < DIM / 16; d++) { out[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, values(u, d)), pb[u], out[d], 0, 0, 0); }
    };

    if (n_mine > 0)
    {
        look_up(0);
        if constexpr (TREE)
        {
            asm volatile("" : "+v"(new_seen));
            seen_pos = mine.pos + max(__builtin_popcount(new_seen) - 1, 0);
        }
        stage(0, false);
        stage(0, true);
    }
    if (STAGES == 2 && n_mine > 1)
    {
        stage(1, false);
        stage(1, true);
    }
    for (int n = 0; n < n_mine; n++) { block(n); }

    // the four waves' sums of a row meet in LDS
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) { stat[wave * 16 + j] = make_float2(m, l); }
    __syncthreads();
    float* const sums = (float*)lds;
#pragma unroll
    for (int d = 0; d < DIM / 16; d++) { *(f32x4*)(sums + (wave * 16 + j) * SUM + 16 * d + 4 * g) = out[d]; }
    __syncthreads();
    const int r = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (DIM / 16);
    if (r < n_rows)
    {
        float top = -INFINITY, total = 0.0f, weight[4];
#pragma unroll
        for (int w = 0; w < 4; w++) { top = fmaxf(top, stat[w * 16 + r].x); }
        const float base = top > -INFINITY ? top : 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++)
        {
            weight[w] = __builtin_amdgcn_exp2f(stat[w * 16 + r].x - base);  // 2^-inf = 0 for a wave without a key
            total += weight[w] * stat[w * 16 + r].y;
        }
        float sum[DIM / 16];
#pragma unroll
        for (int d = 0; d < DIM / 16; d++)
        {
            sum[d] = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) { sum[d] += weight[w] * sums[(w * 16 + r) * SUM + d0 + d]; }      // also with weight 0, as in add_parts
        }
        if (n_parts > 1)
        {
            float* const dst = p.row_sums(slot, kvh, a.n_kv, r, DIM) + d0;
#pragma unroll
            for (int d = 0; d < DIM / 16; d += 2) { store_part(dst + d, sum[d], sum[d + 1]); }
            if (d0 == 0) { store_part(p.row_stats(slot, kvh, a.n_kv, r, DIM), top, total); }
        }
        else
        {
            const float by = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int d = 0; d < DIM / 16; d++) { sum[d] = total == 0.0f ? 0.0f : sum[d] * by; }
            uint16_t* const dst = p.y + (size_t)(mine.first + r / p.group) * p.ldy + (size_t)(kvh * p.group + r % p.group) * DIM + d0;
#pragma unroll
            for (int d = 0; d < DIM / 16; d += 4) { *(u32x2*)(dst + d) = pack4(sum + d); }
        }
    }
    if (n_parts > 1)
    {
        auto slot_of = [&](int i) { return slot - part + i; };
        auto flag = [&](int i) { return p.there + (size_t)slot_of(i) * a.n_kv + kvh; };
        if (all_there(p.there + (size_t)slot * a.n_kv + kvh, p.call, n_parts, (uint32_t*)stat, flag))
        {
            if (r < n_rows)
            {
                add_parts<DIM>(n_parts, p.y + (size_t)(mine.first + r / p.group) * p.ldy + (size_t)(kvh * p.group + r % p.group) * DIM + d0, [&](int i, const float*& from, const float*& at) {
                    from = p.row_sums(slot_of(i), kvh, a.n_kv, r, DIM) + d0;
                    at = p.row_stats(slot_of(i), kvh, a.n_kv, r, DIM);
                });
            }
            // a captured call may be replayed under its name
            for (int i = threadIdx.x; i < n_parts; i += 256) { __hip_atomic_store(flag(i), 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
        }
    }
}

// Part c of a kv head's, or with row_parts 0 all of sequence c.
template <int TYPE, int DIM, bool TREE>
__device__ __forceinline__ void attend_part(const PagedArgs& a, const PagedAttention& p, uint8_t* lds, int c, int kvh)
{
    typedef Parts<RowsForm<TYPE, DIM>::KEYS> P;
    if (p.row_parts == 0)
    {
        const NewTokens mine = SeqWords(a, c).tokens(a, p, c);
        const int shares = uniform(P::shares_of(p, mine));
        if (shares > 0) { attend_rows<TYPE, DIM, TREE>(a, p, lds, c, mine, kvh, 0, shares, 0, 0, 1); }
        return;
    }
    const P of(a, p, c);
    if (of.s >= 0) { attend_rows<TYPE, DIM, TREE>(a, p, lds, of.s, of.mine, kvh, (int)((long long)of.shares * of.part / of.parts), (int)((long long)of.shares * (of.part + 1) / of.parts), c, of.part, of.parts); }
}

// 128 rows of a kv head: chunks and prompts.  Bound by the matrix cores and what a wave issues between their instructions: for a block of 64 keys of 128 dims a wave
// has 1024 cycles of products, about as many of weights, masks' tests and addresses, and 4 x 254 on the way from LDS that its workgroup shares.  Two workgroups on a
// CU fill each other's gaps (a block of both 2.15 us, a lone one 1.35): 2048 tokens behind 6000 E4M3 rows 226 to 244 us by the card, 965 to 1040 TFLOP/s of the 1413 that a
// large product reaches.  (64 rows per wave, half the way from LDS, do not fit a wave's registers: three times as long.)
//   A workgroup of four waves takes 128 rows, a wave 32 of them and every key of each block of 64; keys and values reach LDS as BF16, shared by
// the waves: from a BF16 cache by direct loads, from FP8 through registers, times their powers of two (exact, once per workgroup).
//   scores: v_mfma_f32_32x32x16_bf16, key rows as row operand, queries as columns: D lane (row j = lane % 32, h = lane / 32), register i holds key
//           8 (i / 4) + 4 h + i % 4 of 32.
//   V p:    registers 8 u .. + 7 of a lane are its column operand of the u-th 16 keys as they are; the row operand (dim, the same keys) comes from
//           two transposing reads.
// Weights are rounded to BF16 for that product as in the form above, and for its reason.
// A row's statistics and sums stay in the two lanes that have it.
template <int TYPE, int DIM>
struct TileForm
{
    static constexpr int BLOCK = PA_TILE_KEYS * DIM * 2;
    static constexpr int ODD = 4 * BLOCK, LDS = ODD + 32;                   // two blocks of keys, two of values
};

template <int TYPE, int DIM, bool TREE>
__device__ __forceinline__ void attend_tile(const PagedArgs& a, const PagedAttention& p, uint8_t* lds, int tile, int kvh, int range)
{
    typedef TileForm<TYPE, DIM> F;
    constexpr int KEYS = PA_TILE_KEYS, ROW = DIM * 2, CHUNKS = ROW / 16, BLOCK = F::BLOCK;
    constexpr int CODES = DIM * CODE_BYTES<TYPE>;                           // bytes of a cached row
    uint32_t* const odd_rows = (uint32_t*)(lds + F::ODD);                   // per buffer of values and wave that staged: something infinite or NaN
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int j = lane & 31, h = lane >> 5;
    Tile rows;
    if constexpr (TREE)
    {
        rows = find_piece<false>(a, p, tile);
        range = rows.range;
    }
    else { rows = find_tile(a, p, tile); }
    if (rows.s < 0 || range >= rows.n_ranges) { return; }
    const NewTokens mine = rows.mine;
    const auto& blocks = rows.blocks;
    const int s = rows.s, n_rows = rows.n_rows, row0 = rows.row0, tile_lo = rows.lo, tile_hi = rows.hi;
    const int begin = range * rows.per, end = min(blocks.n, begin + rows.per);

    // the wave's rows
    const int r = row0 + wave * 32 + j, row = min(r, n_rows - 1);
    const bool real = r < n_rows;
    const int token = mine.first + row / p.group, head = kvh * p.group + row % p.group, my_pos = mine.pos + row / p.group;
    // trees: the bits of the row's token, and as many positions behind the first new token as it descends from tokens
    const unsigned long long* const seen_row = p.seen + (TREE ? (size_t)token * p.seen_stride : 0);
    int seen_pos = 0;
    if (TREE && p.window != 0)
    {
        for (int i = 0; 64 * i < mine.n; i++) { seen_pos += __builtin_popcountll(seen_word(seen_row, mine.n, i)); }
        seen_pos = mine.pos + max(seen_pos - 1, 0);
    }
    auto keys_seen = [&](int key0) { return named_keys(p, mine.pos, seen_pos, key0, [&](int i) { return seen_word(seen_row, mine.n, i); }); };
    u32x4 qf[DIM / 16];
#pragma unroll
    for (int c = 0; c < DIM / 16; c++) { qf[c] = *(const u32x4*)(p.q + (size_t)token * p.ldq + (size_t)head * DIM + c * 16 + h * 8); }

    auto key_swizzle = [](int r) { return r / (256 / ROW) % CHUNKS; };
    auto value_swizzle = [](int r) { return DIM == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); };
    // lane l, entry 64 n + l of the range: where the 16 rows that this wave stages begin in the pool (and their exponents), and above bit 60 which
    // quarters of the entry have no page
    size_t rows_from = 0, exponents_from = 0;
    auto look_up = [&](int i0) {
        const int i = i0 + lane, key0 = blocks.block(i) * KEYS;
        size_t lacks = 0;
        int mine_page = 0, page[4];
        const int last = max(tile_hi, 0);
#pragma unroll
        for (int quarter = 0; quarter < 4; quarter++) { page[quarter] = paged_page(a, s, min(key0 + 16 * quarter, last)); }      // four loads, one trip
        if (i < end)
        {
#pragma unroll
            for (int quarter = 0; quarter < 4; quarter++)
            {
                lacks |= page[quarter] < 0 && key0 + 16 * quarter <= tile_hi ? (size_t)1 << (60 + quarter) : 0;
                mine_page = quarter == wave ? max(page[quarter], 0) : mine_page;
            }
        }
        const size_t r0 = paged_row(a, kvh, key0 + 16 * wave);
        rows_from = mine_page * a.page_stride + r0 * CODES | lacks;
        exponents_from = mine_page * a.scale_stride + r0;
    };
    auto of_entry = [&](size_t v, int i) {
        const int at = (i - begin) & 63;
        return (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), at) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, at);
    };
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_offset(lds));
    // FP8: lane group q (DIM / 8 lanes, eight codes each) takes rows PIECES q .. of the wave's 16
    constexpr int LANES = DIM / 8, PIECES = DIM / 32;
    struct Staged
    {
        u32x2 codes[PIECES];
        uint32_t exponents;
    };
    const uint32_t key_from = lane * 16 ^ key_swizzle(lane / CHUNKS) * 16, value_from = lane * 16 ^ value_swizzle(lane / CHUNKS) * 16;
    const uint32_t code_from = lane / LANES * PIECES * CODES + lane % LANES * 8;
    const int code_row = lane / LANES * PIECES;
    const uint32_t key_to = code_row * ROW + (lane % LANES ^ key_swizzle(code_row)) * 16, value_to = code_row * ROW + (lane % LANES ^ value_swizzle(code_row)) * 16;
    // The wave's 16 rows of an entry in PIECES parts: on their way to LDS (BF16) or to registers, and from there to LDS as BF16 (FP8).
    struct Source
    {
        const uint8_t* rows;
        const uint8_t* exponents;
    };
    auto source = [&](bool values, size_t from, size_t exponents) {
        return Source{ (values ? a.v : a.k) + (from & ((size_t)1 << 60) - 1), (values ? a.v_scale : a.k_scale) + exponents };
    };
    auto load = [&](bool values, int n, uint32_t wanted, const Source& of, uint32_t to, Staged& raw) {
        if constexpr (TYPE == DT_BF16)
        {
            // rows n (1024 / ROW) + lane / CHUNKS: with n the keys' swizzle changes by 4 n, the values' not at all
            uint32_t at = values ? value_from : key_from ^ 64 * n;
            asm volatile("" : "+v"(at));                                    // worked out anew: registers are short
            kib_to_lds(uniform((int)wanted), lds0 + to + n * 1024, of.rows + n * 1024, at);
        }
        else
        {
            uint32_t at = code_from;
            asm volatile("" : "+v"(at));
            raw.codes[n] = *(const u32x2*)(of.rows + at + n * CODES);
            if (n == 0)
            {
                if constexpr (DIM == 128) { raw.exponents = *(const uint32_t*)(of.exponents + lane / LANES * 4); }
                else { raw.exponents = *(const uint16_t*)(of.exponents + lane / LANES * 2); }
            }
        }
    };
    auto store = [&](bool values, int n, uint32_t to, const Staged& raw) {
        if constexpr (TYPE != DT_BF16)
        {
            uint32_t at = values ? value_to : key_to;
            asm volatile("" : "+v"(at));
            const float by = bits_to_f32((raw.exponents >> (8 * n) & 255u) << 23);
            const u32x2 lo = fp8x4_to_bf16<TYPE>(raw.codes[n][0], by), hi = fp8x4_to_bf16<TYPE>(raw.codes[n][1], by);
            // row PIECES q + n: n is in the row's low bits, which the swizzles take as they are
            *(u32x4*)(lds + to + (at ^ (values ? value_swizzle(n) : key_swizzle(n)) * 16) + n * ROW) = u32x4{ lo[0], lo[1], hi[0], hi[1] };
        }
    };
    auto keys_at = [&](int i) { return (uint32_t)((i - begin) & 1) * BLOCK; };
    auto values_at = [&](int i) { return (uint32_t)(2 + ((i - begin) & 1)) * BLOCK; };
    const uint32_t part = wave * (BLOCK / 4);                               // the wave's rows of a block
    // entries plain_from .. plain_to - 1: every row of the tile sees every key
    int plain_from = 0, plain_to = (TREE ? max(tile_lo, 0) : tile_lo + 1) / KEYS;
    if (p.window != 0) { plain_from = (tile_hi - p.window + KEYS) / KEYS; }
    plain_from = max(plain_from - blocks.skip, tile_hi < p.window || p.window == 0 ? 0 : blocks.sinks);
    plain_to -= blocks.skip;
    auto masked = [&](int i, size_t from) { return i < plain_from || i >= plain_to || from >> 60 != 0; };
    // in front of the barrier behind which the values of entry i are read: whether any of this wave's rows is infinite or NaN, where that matters
    auto note_odd = [&](int i) {
        uint32_t odd = 0;
#pragma unroll
        for (int n = 0; n < PIECES; n++) { odd |= not_finite(*(const u32x4*)(lds + values_at(i) + part + n * 1024 + lane * 16)); }
        const bool any = __any(odd != 0);
        if (lane == 0) { odd_rows[(i & 1) * 4 + wave] = any; }
    };

    const uint32_t k_at = j * ROW + (h ^ key_swizzle(j)) * 16;             // of chunk h of key row j; chunk 2 c + h at k_at ^ 32 c
    auto score_products = [&](int i, f32x16 (&acc)[2]) {
        uint32_t at = k_at + keys_at(i);
        asm volatile("" : "+v"(at));
        const f32x16 zero = {};
#pragma unroll
        for (int c = 0; c < DIM / 16; c++)
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
            {
                const bf16x8 kf = *(const bf16x8*)(lds + (at ^ (32 * c)) + kt * 32 * ROW);       // the swizzle of row j + 32 is that of j
                acc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, __builtin_bit_cast(bf16x8, qf[c]), c == 0 ? zero : acc[kt], 0, 0, 0);
            }
    };

    float m = -INFINITY, l = 0.0f;
    f32x16 out[DIM / 32];
#pragma unroll
    for (int d = 0; d < DIM / 32; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) { out[d][e] = 0.0f; }
    // dims 32 d + 16 (lane / 16 % 2) + 4 (lane % 4) .. + 3 of key row 4 h + lane % 16 / 4 (and of rows 8 further, and of the next 16)
    const int v_row = 4 * h + ((lane & 15) >> 2), v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const uint32_t v_at = v_row * ROW + ((v_chunk ^ value_swizzle(v_row)) << 4) + ((lane & 1) << 3);     // dims 32 d on at v_at ^ 64 d

    // scores of keys that a row does not see
    auto mask = [&](f32x16 (&acc)[2], int b, int lacks) {
        if constexpr (TREE)
        {
            const unsigned long long bits = keys_seen(b * KEYS) >> (4 * h);
#pragma unroll
            for (int e = 0; e < 32; e++)
            {
                const bool see = (bits >> (8 * (e / 4) + e % 4) & 1) != 0 && !(lacks >> (e / 8) & 1);
                acc[e / 16][e % 16] = see ? acc[e / 16][e % 16] : -INFINITY;
            }
            return;
        }
        // element e: key 8 (e / 4) + 4 h + e % 4 of the block
        const int last = my_pos - b * KEYS - 4 * h, from = p.window == 0 ? -0x40000000 : last - p.window, sinks = p.n_sink - b * KEYS - 4 * h;
#pragma unroll
        for (int e = 0; e < 32; e++)
        {
            const int key = 8 * (e / 4) + e % 4;
            const bool see = key <= last && (key > from || key < sinks) && !(lacks >> (e / 8) & 1);
            acc[e / 16][e % 16] = see ? acc[e / 16][e % 16] : -INFINITY;
        }
    };
    // largest raw score of a row
    float top;
    auto find_top = [&](const f32x16 (&acc)[2]) {
        top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 32; e++) { top = fmaxf(top, acc[e / 16][e % 16]); }
    };
    // the running maximum; sums rescaled where it moves
    float off;
    auto raise = [&]() {
        const float least = top * p.scale;
        if (__any(least > m + PA_LAG))
        {
            const float next = fmaxf(m, fmaxf(least, __shfl_xor(least, 32)));
            const float shrink = m > -INFINITY ? __builtin_amdgcn_exp2f(m - next) : 1.0f;       // sums of nothing: 0, or what is not finite
            m = next;
            l *= shrink;
#pragma unroll
            for (int d = 0; d < DIM / 32; d++) { out[d] *= shrink; }
        }
        off = m > -INFINITY ? -m : 0.0f;                       // no key seen yet: every weight is 2^-inf = 0
    };
    // The weights of entry i under the products of entry i + 1, then the products of the weights under the largest scores of i + 1: in each step the
    // vector unit has work for as long as the matrix core has.  A wave goes before its SIMD's other one from the scores until half of the values' products, so
    // that the two fall into different halves (MI355X, 2048 tokens behind 6000 E4M3 rows 241 -> 236 us, windowed prompts 144 -> 141; before it in the values'
    // products instead 247).
    auto advance = [&](int i, const f32x16 (&cur)[2], f32x16 (&next)[2], auto loads, auto stores) {
        constexpr int STEPS = DIM / 16, WEIGHTS = 32 / STEPS, PAIRS = DIM / 64;
        uint32_t key_at = k_at + keys_at(i + 1), value_at = v_at + values_at(i);
        asm volatile("" : "+v"(key_at), "+v"(value_at));
        auto keys = [&](int c, int kt) { return *(const bf16x8*)(lds + (key_at ^ (32 * c)) + kt * 32 * ROW); };      // the swizzle of row j + 32 is that of j
        auto values = [&](int u, int d) {
            const u32x2 lo = lds_transposed16(lds + (value_at ^ (64 * d)) + u * 16 * ROW), hi = lds_transposed16(lds + (value_at ^ (64 * d)) + (u * 16 + 8) * ROW);
            return __builtin_bit_cast(bf16x8, u32x4{ lo[0], lo[1], hi[0], hi[1] });
        };
        const f32x16 zero = {};
        constexpr int AHEAD = 2, N_VALUES = 4 * PAIRS;    // steps that operands are read ahead
        bf16x8 pb[4], kf[STEPS][2], vf[N_VALUES][2];
        float sum[2] = {};
        auto read = [&](int step) {                                         // operands of a step, counted through
#pragma unroll
            for (int n = 0; n < 2; n++)
            {
                if (step < STEPS) { kf[step][n] = keys(step, n); }
                else if (step < STEPS + N_VALUES) { vf[step - STEPS][n] = values((step - STEPS) / PAIRS, (step - STEPS) % PAIRS * 2 + n); }
            }
        };
#pragma unroll
        for (int c = 0; c < AHEAD; c++) { read(c); }
        __builtin_amdgcn_sched_barrier(0);
        raise();                                                            // while they are on their way
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < STEPS; c++)
        {
            read(c + AHEAD);
            loads(c);
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
                { next[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[c][kt], __builtin_bit_cast(bf16x8, qf[c]), c == 0 ? zero : next[kt], 0, 0, 0); }
#pragma unroll
            for (int e = c * WEIGHTS; e < (c + 1) * WEIGHTS; e++)
            {
                const float w = __builtin_amdgcn_exp2f(fmaf(cur[e / 16][e % 16], p.scale, off));
                sum[e & 1] += w;
                pb[e / 8][e % 8] = (__bf16)w;
            }
            asm volatile("" : "+v"(sum[0]), "+v"(sum[1]));        // added here, not when somebody asks
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < N_VALUES; n++)
        {
            const int u = n / PAIRS, d = n % PAIRS * 2;
            read(STEPS + n + AHEAD);
            stores(n);
#pragma unroll
            for (int k = 0; k < 2; k++)
                { out[d + k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[n][k], pb[u], out[d + k], 0, 0, 0); }
            if (n == 0) { top = -INFINITY; }
            if (n == N_VALUES / 2) { __builtin_amdgcn_s_setprio(0); }
#pragma unroll
            for (int e = n * (8 / PAIRS); e < (n + 1) * (8 / PAIRS); e++) { top = fmaxf(top, next[e / 16][e % 16]); }
            asm volatile("" : "+v"(top));
            __builtin_amdgcn_sched_barrier(0);
        }
        l += sum[0] + sum[1];
    };
    // Weight 0 times an infinity is NaN: where some rows do not see every key of entry i, what is infinite or NaN among its values is added to the sums of
    // the rows that see it and cleared in front of the products.
    auto set_apart = [&](int i, int lacks) {
        const u32x4 odd = *(const u32x4*)(odd_rows + (i & 1) * 4);
        if (__builtin_amdgcn_readfirstlane(odd[0] | odd[1] | odd[2] | odd[3]) == 0) { return; }
        uint8_t* const vb = lds + values_at(i);
        const int b = blocks.block(i);
        const unsigned long long bits = TREE ? keys_seen(b * KEYS) : 0;
#pragma unroll 1
        for (int key = 0; key < KEYS; key++)
        {
            if (lacks >> (key / 16) & 1) { continue; }
            const bool see = TREE ? (bits >> key & 1) != 0 : sees(p, my_pos, b * KEYS + key);
#pragma unroll
            for (int n = 0; n < DIM / 8; n++)
            {
                const int dim = 8 * n + 4 * h;
                const u32x2 raw = *(const u32x2*)(vb + key * ROW + (((dim / 8) ^ value_swizzle(key)) << 4) + (dim & 4) * 2);
                float v[4];
                unpack4(raw, v);
#pragma unroll
                for (int e = 0; e < 4; e++) { out[n / 4][n % 4 * 4 + e] += see && !(fabsf(v[e]) < INFINITY) ? v[e] : 0.0f; }
            }
        }
        lds_barrier();
#pragma unroll
        for (int n = 0; n < ROW * 16 / 1024; n++)
        {
            u32x4* const at = (u32x4*)(vb + part + n * 1024 + lane * 16);
            *at = finite_part(*at);
        }
        lds_barrier();
    };
    // loads of this wave into LDS have arrived and its accesses of LDS are done; the same, then the workgroup's barrier
    auto arrived = []() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); };
    auto barrier = []() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    if (begin < end)
    {
        Staged raw_k, raw_v;
        f32x16 cur[2], next[2];
        look_up(begin);
        // where the values of the next entry begin, and whether this one and the next are masked (for what they lack)
        size_t from = of_entry(rows_from, begin), exponents = TYPE == DT_BF16 ? 0 : of_entry(exponents_from, begin);
        bool is_masked = masked(begin, from), next_masked = false;
        int lacks = (int)(from >> 60), next_lacks = 0;
        // the first entry and the keys of the second, all asked for at once
        Staged raw_next;
        auto fetch = [&](bool values, uint32_t to, Staged& raw) {
            const Source of = source(values, from, exponents);
#pragma unroll
            for (int n = 0; n < PIECES; n++) { load(values, n, 1, of, to, raw); }
        };
        fetch(false, keys_at(begin) + part, raw_k);
        fetch(true, values_at(begin) + part, raw_v);
        if (begin + 1 < end)
        {
            from = of_entry(rows_from, begin + 1);
            if constexpr (TYPE != DT_BF16) { exponents = of_entry(exponents_from, begin + 1); }
            next_masked = masked(begin + 1, from);
            next_lacks = (int)(from >> 60);
        }
        fetch(false, keys_at(begin + 1) + part, raw_next);
#pragma unroll
        for (int n = 0; n < PIECES; n++)
        {
            store(false, n, keys_at(begin) + part, raw_k);
            store(true, n, values_at(begin) + part, raw_v);
            store(false, n, keys_at(begin + 1) + part, raw_next);
        }
        arrived();
        if (is_masked) { note_odd(begin); }
        barrier();
        score_products(begin, cur);
        find_top(cur);
        // entry i: its values and the keys of i + 1 are in LDS, `cur` holds its raw scores
        auto entry = [&](int i, f32x16 (&cur)[2], f32x16 (&next)[2]) {
            // behind the last entry: its rows again (FP8) or none (BF16), and scores of what lies there, for nobody
            const int ahead = min(i + 2, end - 1);
            if (((i + 2 - begin) & 63) == 0 && i + 2 < end) { look_up(i + 2); }
            const size_t from_ahead = of_entry(rows_from, ahead), exponents_ahead = TYPE == DT_BF16 ? 0 : of_entry(exponents_from, ahead);
            const Source key_rows = source(false, from_ahead, exponents_ahead), value_rows = source(true, from, exponents);
            const uint32_t keys_to = keys_at(i) + part, values_to = values_at(i + 1) + part;       // keys of i + 2: those of i were read before the last barrier
            if (is_masked)
            {
                set_apart(i, lacks);
                mask(cur, blocks.block(i), lacks);
                find_top(cur);
            }
            // a workgroup's loads all at once would hold up its waves: one or two with every step
            constexpr int STEPS = DIM / 16, PER = 2 * PIECES * 2 / STEPS;
            auto loads = [&](int step) {
#pragma unroll
                for (int n = step * PER; n < (step + 1) * PER; n++)
                {
                    if (n < PIECES) { load(false, n, i + 2 < end, key_rows, keys_to, raw_k); }
                    else if (n < 2 * PIECES) { load(true, n - PIECES, i + 1 < end, value_rows, values_to, raw_v); }
                }
            };
            auto stores = [&](int step) {
                constexpr int FROM = 4 * (DIM / 64) - 2 * PIECES;
                const int n = step - FROM;
                if (n < 0) { return; }
                if (n < PIECES) { store(false, n, keys_to, raw_k); }
                else { store(true, n - PIECES, values_to, raw_v); }
            };
            advance(i, cur, next, loads, stores);
            arrived();
            if (next_masked && i + 1 < end) { note_odd(i + 1); }
            barrier();
            is_masked = next_masked;
            lacks = next_lacks;
            from = from_ahead;
            exponents = exponents_ahead;
            next_masked = masked(i + 2, from);
            next_lacks = (int)(from >> 60);
        };
        for (int i = begin; i < end; i += 2)
        {
            entry(i, cur, next);
            if (i + 1 < end) { entry(i + 1, next, cur); }
        }
    }

    const float total = l + __shfl_xor(l, 32);
    if (!real) { return; }
    const size_t at_row = (size_t)token * p.n_q + head;
    if (rows.n_ranges > 1)
    {
        float* const dst = (TREE ? p.piece_sums(rows.piece0 + range, kvh, a.n_kv, wave * 32 + j, DIM) : p.sums(range, at_row, DIM)) + 4 * h;
#pragma unroll
        for (int d = 0; d < DIM / 32; d++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) { *(f32x4*)(dst + 32 * d + 2 * e) = f32x4{ out[d][e], out[d][e + 1], out[d][e + 2], out[d][e + 3] }; }
        if (h == 0) { *(TREE ? p.piece_stats(rows.piece0 + range, kvh, a.n_kv, wave * 32 + j, DIM) : p.stats(range, at_row, DIM)) = make_float2(m, total); }
        return;
    }
    uint16_t* const dst = p.y + (size_t)token * p.ldy + (size_t)head * DIM + 4 * h;
    const float by = 1.0f / total;
#pragma unroll
    for (int d = 0; d < DIM / 32; d++)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
        {
            float v[4];
#pragma unroll
            for (int n = 0; n < 4; n++) { v[n] = total == 0.0f ? 0.0f : out[d][e + n] * by; }
            *(u32x2*)(dst + 32 * d + 2 * e) = pack4(v);
        }
}

// Both forms in one launch, tiles first: single tokens beside a chunk run beside it.  Grid: ranges x tiles x kv heads, then parts x kv heads.
template <int TYPE, int DIM, bool TREE>
__global__ __launch_bounds__(256, 2) void paged_attention_kernel(const PagedArgs a, const PagedAttention p)
{
    typedef RowsForm<TYPE, DIM> R;
    typedef TileForm<TYPE, DIM> T;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[R::LDS > T::LDS ? R::LDS : T::LDS];
    static_assert(sizeof(lds) <= 80 * 1024, "two workgroups on a CU");
    const int tiles = p.tiles * a.n_kv, n_tiles = tiles * p.tile_split;
    if ((int)blockIdx.x < n_tiles) { attend_tile<TYPE, DIM, TREE>(a, p, lds, blockIdx.x % tiles / a.n_kv, blockIdx.x % a.n_kv, blockIdx.x / tiles); }
    else { attend_part<TYPE, DIM, TREE>(a, p, lds, (blockIdx.x - n_tiles) / a.n_kv, (blockIdx.x - n_tiles) % a.n_kv); }
}

// The tiles' ranges added, 16 rows per workgroup and DIM / 16 dims of a row per thread.  Rows in one piece are written already.  Grid: eighths of tiles x kv heads.
template <int DIM, bool TREE>
__global__ __launch_bounds__(256) void paged_attention_combine_kernel(const PagedArgs a, const PagedAttention p)
{
    const int kvh = blockIdx.x % a.n_kv, at = blockIdx.x / a.n_kv;
    const Tile rows = TREE ? find_piece<true>(a, p, at / 8) : find_tile(a, p, at / 8);
    const int row = rows.row0 + at % 8 * 16 + (threadIdx.x >> 4);
    if (rows.s < 0 || row >= rows.n_rows || rows.n_ranges <= 1) { return; }
    const size_t token = rows.mine.first + row / p.group, head = kvh * p.group + row % p.group, at_row = token * p.n_q + head;
    const int d0 = (threadIdx.x & 15) * (DIM / 16);
    add_parts<DIM, true>(rows.n_ranges, p.y + token * p.ldy + head * DIM + d0, [&](int i, const float*& from, const float*& stat) {
        from = (TREE ? p.piece_sums(rows.piece0 + i, kvh, a.n_kv, row - rows.row0, DIM) : p.sums(i, at_row, DIM)) + d0;
        stat = (const float*)(TREE ? p.piece_stats(rows.piece0 + i, kvh, a.n_kv, row - rows.row0, DIM) : p.stats(i, at_row, DIM));
    });
}

}    // namespace ccq
