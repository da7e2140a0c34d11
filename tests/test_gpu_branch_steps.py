"""Sequences that branch over some steps as they would be served, calls one behind the other without waiting: drafted trees checked and kept, and beams over quantized logits."""
import numpy as np
import pytest
from oracle import synth

from branch_util import Layers, beam, bits, fork, tree_attend, trees
from gpu_util import check_rows, to_dev
from paged_util import BF16, E4M3, E5M2, Batch, attend, from_bf16, to_bf16
from test_gpu_paged import ptr, put

pytestmark = pytest.mark.gpu

N_Q, N_KV, DIM, PAGE, LAYERS = 8, 2, 64, 16, 2
HEADS = N_Q + 2 * N_KV


def tables(n):
    angle = np.arange(n)[:, None] * 1e4 ** (-np.arange(DIM // 2) / (DIM // 2))
    return to_bf16(np.cos(angle)), to_bf16(np.sin(angle))


class Server:
    """Two layers' caches with a table and lengths that forks replace."""

    def __init__(self, gpu, pkg, b):
        self.torch, self.dev, self.lib = gpu
        self.pkg, self.b, self.layers = pkg, b, Layers(b, LAYERS, *gpu[:2])
        cos, sin = tables(400)
        self.cos, self.sin = put(self.torch, self.dev, cos), put(self.torch, self.dev, sin)
        self.int32 = lambda v: self.torch.from_numpy(np.ascontiguousarray(v, dtype=np.int32)).to(self.dev)  # noqa: E731

    def at_layers(self, table, ctx, start, n):
        """The caches with these tables, and this module's batches in step for the formulas."""
        for x in self.layers.batches:
            x.dev["table"], x.dev["ctx_len"], x.dev["seq_start"], x.n_seqs = table, ctx, start, n
        return self.layers.caches(self.pkg)

    def fork(self, caches, n_out, parent, rows, grow):
        torch, lib = self.torch, self.lib
        table, ctx, missing = (torch.full(shape, -9, dtype=torch.int32, device=self.dev) for shape in ((n_out, self.b.table_stride), (n_out,), (1,)))
        need = lib.kv_paged_fork_workspace_bytes(caches, LAYERS, n_out)
        ws = torch.empty(need, dtype=torch.uint8, device=self.dev)
        assert lib.kv_paged_fork(caches, LAYERS, n_out, ptr(parent), ptr(rows), ptr(grow), None, ptr(table), ptr(ctx), ptr(missing), ptr(ws), need) == 0
        self.kept = (ws, parent, rows, grow)
        return table, ctx, missing

    def read_back(self, table, ctx, start, new):
        """What lies in memory, for the formulas."""
        for x in self.layers.batches:
            x.table, x.ctx, x.new = table.cpu().numpy(), [int(v) for v in ctx.cpu()], list(new)
            x.ctx_len, x.seq_start, x.tokens = np.array(x.ctx), start.cpu().numpy(), sum(new)
            for name in ("k", "v"):
                x.pool[name] = x.download(name)
                if x.kind != BF16: x.scale[name] = x.download(name + "_scale")


@pytest.mark.parametrize("kind", [BF16, E4M3, E5M2])
def test_drafted_trees(gpu, pkg, kind):
    """Room for a tree, its keys at their depths, attention by layer, the path that is kept: the caches hold what the same tokens give that are appended one behind the other, byte for byte, attention is the formula's."""
    torch, dev, lib = gpu
    n, rng = 3, np.random.default_rng(kind)
    behind = [70, 15, 33]
    b = Batch(kind, kind, DIM, N_KV, PAGE, [1] * n, behind, spare=40, table_extra=12)
    line = Batch(kind, kind, DIM, N_KV, PAGE, [1] * n, behind, spare=40, table_extra=12)       # the same, without trees
    s, plain = Server(gpu, pkg, b), Server(gpu, pkg, line)
    for x, y in zip(s.layers.batches, plain.layers.batches):
        for name in ("k", "v", "k_scale", "v_scale"):
            if x.dev[name] is not None: y.dev[name].copy_(x.dev[name])
    table, ctx, start = b.dev["table"], b.dev["ctx_len"], b.dev["seq_start"]
    far, far_ctx = line.dev["table"], line.dev["ctx_len"]
    lib.set_sync(False)
    try:
        for step, new in enumerate(([7, 1, 20], [12, 30, 4], [1, 9, 16])):
            T, seen = sum(new), trees(rng, new)
            kept = []                           # a path from the root on
            for one in seen:
                leaf = int(rng.integers(0, len(one)))
                kept.append(np.flatnonzero(one[leaf]))
            keep = np.concatenate([np.concatenate([k, np.zeros(m - len(k), dtype=int)]) for k, m in zip(kept, new)])
            n_keep = [len(k) for k in kept]
            start = s.int32(np.concatenate([[0], np.cumsum(new)]))
            caches = s.at_layers(table, ctx, start, n)
            table, ctx, missing = s.fork(caches, n, s.int32(range(n)), None, s.int32(new))
            caches = s.at_layers(table, ctx, start, n)
            x = [to_bf16(rng.standard_normal((T, HEADS * DIM))) for _ in range(LAYERS)]
            xd, words = [put(torch, dev, a) for a in x], torch.from_numpy(bits(seen, 1)).to(dev)
            depth = torch.from_numpy(np.concatenate([one.sum(1) - 1 for one in seen]).astype(np.int32)).to(dev)
            seq = torch.repeat_interleave(torch.arange(n, device=dev), torch.tensor(new, device=dev))
            positions = ((ctx - s.int32(new))[seq] + depth).contiguous()
            q, y = ([torch.zeros(T, N_Q * DIM, dtype=torch.int16, device=dev) for _ in range(LAYERS)] for _ in range(2))
            need = lib.attention_paged_tree_workspace_bytes(caches[0], N_Q, T, 30, 400)
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
            for i in range(LAYERS):
                at = xd[i].data_ptr()
                assert lib.qk_norm_rope_kv_paged_at(caches[i], at, at + 2 * N_Q * DIM, at + 2 * (N_Q + N_KV) * DIM, None, None, ptr(s.cos), ptr(s.sin), 400, ptr(positions), 1, T, None, ptr(q[i]), N_Q, T,
                                                    HEADS * DIM, HEADS * DIM, HEADS * DIM) == 0
                assert lib.attention_paged_tree(caches[i], ptr(q[i]), ptr(y[i]), ptr(words), 1, ptr(ws), need, N_Q, T, 30, 400, 0, 0, N_Q * DIM, N_Q * DIM) == 0
            torch.cuda.synchronize()
            s.read_back(table, ctx, start, new)
            assert int(missing) == 0
            for i, batch in enumerate(s.layers.batches):
                want, bound = tree_attend(batch, from_bf16(q[i].cpu().numpy().view(np.uint16)).reshape(T, N_Q, DIM), N_Q, seen)
                assert (np.abs(from_bf16(y[i].cpu().numpy().view(np.uint16)).reshape(T, N_Q, DIM) - want) <= bound).all(), (step, i)
            ctx_kept = torch.zeros(n, dtype=torch.int32, device=dev)
            assert lib.kv_paged_keep(caches, LAYERS, ptr(s.int32(keep)), ptr(s.int32(n_keep)), T, 30, ptr(ctx_kept)) == 0
            torch.cuda.synchronize()
            ctx = ctx_kept
            # the kept tokens alone, as any new ones
            rows = np.concatenate([k + sum(new[:j]) for j, k in enumerate(kept)])
            far_start = s.int32(np.concatenate([[0], np.cumsum(n_keep)]))
            far, far_ctx, _ = plain.fork(plain.at_layers(far, far_ctx, far_start, n), n, s.int32(range(n)), None, s.int32(n_keep))
            far_caches = plain.at_layers(far, far_ctx, far_start, n)
            for i in range(LAYERS):
                part = put(torch, dev, x[i][rows])
                at = part.data_ptr()
                assert lib.qk_norm_rope_kv_paged(far_caches[i], None, at + 2 * N_Q * DIM, at + 2 * (N_Q + N_KV) * DIM, None, None, ptr(s.cos), ptr(s.sin), 400, None, 0, len(rows), 0, HEADS * DIM, HEADS * DIM) == 0
                torch.cuda.synchronize()
            assert torch.equal(ctx, far_ctx)
            s.read_back(table, ctx, far_start, n_keep)
            plain.read_back(far, far_ctx, far_start, n_keep)
            for u, v in zip(s.layers.batches, plain.layers.batches):
                for j in range(n):
                    for name in ("k", "v"): assert np.array_equal(u.rows(name, j), v.rows(name, j)), (step, j, name)
    finally:
        lib.set_sync(True)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_beams(gpu, pkg, oracle, kind):
    """Two prompts become two groups of three beams; steps of append, attention, quantized logits, selection and fork: each against 64 bits from what lies in memory."""
    torch, dev, lib = gpu
    groups, beams, vocab, eos = 2, 3, 1003, 5
    n, rng, ld = groups * beams, np.random.default_rng(kind), 1008
    b = Batch(kind, kind, DIM, N_KV, PAGE, [1] * groups, [37, 64], spare=60, table_extra=4)
    s = Server(gpu, pkg, b)
    W = synth.weights_e5m2(synth.seed_for(8, 1), ld, N_Q * DIM)
    dense = oracle.dequant_weight(W, oracle.E5M2, ld, N_Q * DIM, 1.0)
    wd = to_dev(torch, dev, W)
    embed = torch.from_numpy(to_bf16(rng.standard_normal((vocab, HEADS * DIM))).view(np.int16)).to(dev)
    start = s.int32(range(n + 1))
    score = torch.tensor([0.0, -np.inf, -np.inf] * groups, device=dev)
    last = torch.full((n,), 9, dtype=torch.int32, device=dev)
    caches = s.at_layers(b.dev["table"], b.dev["ctx_len"], start, groups)
    parent = s.int32([0] * beams + [1] * beams)
    lib.set_sync(False)
    try:
        held = (b.dev["table"], b.dev["ctx_len"])
        for step in range(6):
            table, ctx, missing = s.fork(caches, n, parent, None, s.int32([1] * n))
            torch.cuda.synchronize()
            want = fork(held[0].cpu().numpy(), held[1].cpu().numpy(), PAGE, b.n_pages, parent.cpu().numpy(), None, [1] * n, None)
            assert np.array_equal(table.cpu().numpy(), want[0]) and np.array_equal(ctx.cpu().numpy(), want[1]) and int(missing) == want[2] == 0
            held, caches = (table, ctx), s.at_layers(table, ctx, start, n)
            x = embed[last.long()].contiguous()
            q, y = (torch.zeros(n, N_Q * DIM, dtype=torch.int16, device=dev) for _ in range(2))
            need = lib.attention_paged_workspace_bytes(caches[0], N_Q, n, 1, 400)
            ws, logits = torch.empty(max(need, 16), dtype=torch.uint8, device=dev), torch.zeros(n, ld, dtype=torch.int16, device=dev)
            at = x.data_ptr()
            for i in range(LAYERS):
                assert lib.qk_norm_rope_kv_paged(caches[i], at, at + 2 * N_Q * DIM, at + 2 * (N_Q + N_KV) * DIM, None, None, ptr(s.cos), ptr(s.sin), 400, ptr(q), N_Q, n, HEADS * DIM, HEADS * DIM, HEADS * DIM) == 0
                assert lib.attention_paged(caches[i], ptr(q), ptr(y), ptr(ws), need, N_Q, n, 1, 400, 0, 0, N_Q * DIM, N_Q * DIM) == 0
            assert lib.linear(ptr(wd), 5, ptr(y), ptr(logits), ld, n, N_Q * DIM) == 0
            parent, token, next_score = torch.zeros(n, dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev), torch.zeros(n, device=dev)
            room = lib.beam_select_workspace_bytes(groups, beams, vocab, beams)
            space = torch.empty(room, dtype=torch.uint8, device=dev)
            assert lib.beam_select(ptr(logits), ld, ptr(score), ptr(last), eos, groups, beams, vocab, beams, ptr(parent), ptr(token), ptr(next_score), ptr(space), room) == 0
            torch.cuda.synchronize()
            s.read_back(table, ctx, start, [1] * n)
            attended, bound = attend(s.layers.batches[-1], from_bf16(q.cpu().numpy().view(np.uint16)).reshape(n, N_Q, DIM), N_Q)
            got = from_bf16(y.cpu().numpy().view(np.uint16)).reshape(n, N_Q, DIM)
            assert (np.abs(got - attended) <= bound).all()
            seen = from_bf16(logits.cpu().numpy().view(np.uint16))
            check_rows(seen, oracle.linear_exact(dense, y.cpu().numpy().view(np.uint16)), f"logits {step}")
            rows, tokens, totals = beam(seen[:, :vocab], score.cpu().numpy().astype(np.float64), last.cpu().numpy() == eos, eos, groups, beams, beams)
            assert np.array_equal(parent.cpu().numpy(), rows.ravel()) and np.array_equal(token.cpu().numpy(), tokens.ravel())
            assert (np.abs(next_score.cpu().numpy() - totals.ravel()) <= 2.0 ** -24 * np.abs(totals.ravel()) + 112 * 2.0 ** -24).all()
            score, last = next_score, token
            if step == 2: last = torch.where(torch.arange(n, device=dev) == 1, eos, last).int()           # one has ended
    finally:
        lib.set_sync(True)
