// C-ABI entry point of beam selection (kernels in beam.h).
#include "../../include/cccc_hip_quant.h"
#include "beam.h"
#include "runtime.h"
#include <algorithm>

using namespace ccq;

namespace
{
inline bool aligned(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Logits per thread: 64, and fewer where that leaves the GPU with less than two workgroups per CU.  MI355X us, both launches: 128 rows of 128256 logits, n_out 16, with 64 / 16 29.6 / 34.4 (26.9 with 64 since the groups' launch became
// faster); 4 rows of 151936, n_out 4, with 8 (300 workgroups) 13.8.
int logits_per_thread(int rows, int vocab)
{
    int per = 64;
    while (per > 8 && (long long)rows * ((vocab + BEAM_THREADS * per - 1) / (BEAM_THREADS * per)) < 2LL * cu_count()) { per /= 2; }
    return per;
}

int chunks_of(int vocab, int per) { return (vocab + BEAM_THREADS * per - 1) / (BEAM_THREADS * per); }

bool beam_sizes(int n_groups, int n_beams, int vocab, int n_out)
{
    if (n_groups < 0 || n_beams <= 0 || n_beams > 64 || vocab <= 0 || vocab > 1 << 20 || n_out <= 0 || n_out > 128 || n_out > (long long)n_beams * vocab) { return false; }
    // grids of fewer than 2^32 lanes: of 256 for each chunk, of 1024 for each group
    return (long long)n_groups * n_beams * chunks_of(vocab, 8) <= 0xFFFFFF && (long long)n_groups * BEAM_PICK_THREADS <= 0xFFFFFFFFLL;
}

template <int PER>
void launch(const BeamSelect& p)
{
    const int room = p.n_out * PER, lists = room + p.n_out * ((room + BEAM_THREADS - 1) / BEAM_THREADS);
    beam_chunk_kernel<PER><<<p.n_groups * p.n_beams * p.chunks, BEAM_THREADS, lists * 4, stream()>>>(p);
    beam_pick_kernel<PER><<<p.n_groups, BEAM_PICK_THREADS, 0, stream()>>>(p);
}
}    // namespace

unsigned long long hip_beam_select_workspace_bytes(int n_groups, int n_beams, int vocab, int n_out)
{
    if (!beam_sizes(n_groups, n_beams, vocab, n_out)) { return 0; }
    return (unsigned long long)n_groups * n_beams * chunks_of(vocab, logits_per_thread(n_groups * n_beams, vocab)) * (16 + 4ull * ((n_out + 3) & ~3));
}

int hip_beam_select_bf16(const void* logits, long long ld, const void* score, const void* last, int eos, int n_groups, int n_beams, int vocab, int n_out, void* parent_out, void* token_out,
                         void* score_out, void* workspace, unsigned long long workspace_bytes)
{
    if (!beam_sizes(n_groups, n_beams, vocab, n_out)) { return -1; }
    if (n_groups == 0) { return 0; }
    if (!logits || !parent_out || !token_out || !score_out || !workspace || ld < vocab || ld % 8 != 0) { return -1; }
    if (!aligned(logits, 16) || !aligned(workspace, 16) || !aligned(score, 4) || !aligned(last, 4) || !aligned(parent_out, 4) || !aligned(token_out, 4) || !aligned(score_out, 4)) { return -1; }
    if (n_out != n_beams && (score_out == score || token_out == last)) { return -1; }
    if (workspace_bytes < hip_beam_select_workspace_bytes(n_groups, n_beams, vocab, n_out)) { return -1; }
    const int rows = n_groups * n_beams, per = logits_per_thread(rows, vocab), chunks = chunks_of(vocab, per);
    double2* const stats = (double2*)workspace;
    const BeamSelect p = { (const uint16_t*)logits, (size_t)ld, (const float*)score, (const int*)last, eos, n_groups, n_beams, vocab, n_out, chunks, (int*)parent_out, (int*)token_out,
                           (float*)score_out, stats, (uint32_t*)(stats + (size_t)rows * chunks) };
    switch (per)
    {
    case 8: launch<8>(p); break;
    case 16: launch<16>(p); break;
    case 32: launch<32>(p); break;
    default: launch<64>(p); break;
    }
    return finish("beam_select");
}
