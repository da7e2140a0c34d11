"""Rows kept of a tree and batches that fork on a paged cache, in all layers: against lists worked out one entry after the other, every byte of the pools."""
import numpy as np
import pytest

from branch_util import Layers, fork
from paged_util import BF16, E4M3, E5M2, Batch
from test_gpu_paged import KINDS, ptr

pytestmark = pytest.mark.gpu


def ints(torch, dev, v):
    return torch.from_numpy(np.ascontiguousarray(v, dtype=np.int32)).to(dev)


def lists(rng, new, kept=None):
    """Ascending ones, and how many of each are kept; what lies behind them is anything."""
    keep, n_keep = [], []
    for s, n in enumerate(new):
        k = int(rng.integers(0, n + 1)) if kept is None else min(kept[s], n)
        keep += sorted(rng.choice(n, k, replace=False).tolist()) + rng.integers(-5, 2 * n + 5, n - k).tolist()
        n_keep.append(k)
    return np.array(keep, dtype=np.int32), np.array(n_keep, dtype=np.int32)


def check_keep(gpu, pkg, b, n_layers, keep, n_keep, ctx=None, max_new=None, ctx_out=True, skip=(), table=None):
    """keep, n_keep as handed over; skip: sequences that are left as they are."""
    torch, dev, lib = gpu
    layers = Layers(b, n_layers, torch, dev)
    before = layers.pools()
    kd, nd, out = ints(torch, dev, keep), ints(torch, dev, n_keep), torch.full((b.n_seqs + 1,), -7, dtype=torch.int32, device=dev)
    assert lib.kv_paged_keep(layers.caches(pkg), n_layers, ptr(kd), ptr(nd), b.tokens, max_new or max(b.new), ptr(out) if ctx_out else None) == 0
    torch.cuda.synchronize()
    want_ctx, page, anything = [], b.page, np.zeros((b.n_pages, b.page), dtype=bool)
    want = [{name: a.copy() for name, a in pools.items()} for pools in before]
    for s in range(b.n_seqs):
        n, c, t0 = b.new[s], b.ctx[s], int(b.seq_start[s])
        if s in skip or not n:
            want_ctx.append(c)
            continue
        first, k = c - n, int(min(max(n_keep[s], 0), n))
        want_ctx.append(max(first + k, 0))
        for i in range(k):
            j = int(keep[t0 + i])
            if not i < j < n or first + i < 0: continue
            src, dst = b.table[s, (first + j) // page], b.table[s, (first + i) // page]
            if not (0 <= src < b.n_pages and 0 <= dst < b.n_pages): continue
            for w, old in zip(want, before):
                for name in w: w[name][dst, :, (first + i) % page] = old[name][src, :, (first + j) % page]
        for i in range(k, n):
            if first + i >= 0 and 0 <= b.table[s, (first + i) // page] < b.n_pages: anything[b.table[s, (first + i) // page], (first + i) % page] = True
    for got, w in zip(layers.pools(), want):
        for name in w: assert np.array_equal(got[name].swapaxes(1, 2)[~anything], w[name].swapaxes(1, 2)[~anything]), name
    if ctx_out: assert out.cpu().tolist() == want_ctx + [-7]
    else: assert (out == -7).all()


KEEP = [  # dim, n_kv, page, new, ctx, layers
    (128, 1, 16, [1], [1], 1), (128, 2, 16, [13], [4108], 2), (64, 8, 32, [5, 0, 26, 1], [5, 9, 700, 60], 3), (128, 8, 64, [60, 16, 17, 33], [64, 90, 100, 1000], 2), (64, 3, 16, [100, 64], [130, 64], 2),
    (128, 40, 16, [20, 7], [37, 7], 1), (64, 100, 16, [35], [35], 1), (128, 2, 4096, [40], [5000], 1)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_kv,page,new,ctx,n_layers", KEEP)
@pytest.mark.parametrize("kept", ["some", "all", "none", "last"])
def test_keep(gpu, pkg, kind, dim, n_kv, page, new, ctx, n_layers, kept):
    b = Batch(dim + n_kv + sum(new) + kind, kind, dim, n_kv, page, new, ctx)
    keep, n_keep = lists(b.rng, new, {"all": new, "none": [0] * len(new)}.get(kept))
    if kept == "last":                          # the last ones, each source the place of a later one
        n_keep = np.array([max(n - 1, 0) for n in new], dtype=np.int32)
        keep = np.concatenate([np.concatenate([np.arange(1, n), [0]])[:n] for n in new if n]).astype(np.int32)
    check_keep(gpu, pkg, b, n_layers, keep, n_keep, ctx_out=kept != "none")


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_keep_of_lists_and_lengths_that_are_not_right(gpu, pkg, kind):
    """Indices below their place or past the new tokens move nothing, counts are cut; more new tokens than rows; pages outside the pool; a sequence with more new tokens than max_new stays."""
    b = Batch(kind, kind, 64, 2, 16, [10, 20, 6], [40, 15, 30])
    b.table[2, 1] = -1
    keep = np.array([0, 0, 4, 2 ** 31 - 1, -2 ** 31, 5, 7, 9, 10, 11] + list(range(4, 20)) + [0] * 4 + [2, 4, 5, 0, 0, 0], dtype=np.int32)
    check_keep(gpu, pkg, b, 2, keep, np.array([2 ** 31 - 1, 16, 3]))
    b = Batch(kind, kind, 64, 2, 16, [10, 20, 6], [40, 35, 30])
    check_keep(gpu, pkg, b, 1, keep, np.array([-3, 16, 3]), max_new=19, skip=[1])


@pytest.mark.parametrize("n_layers", [63, 64, 65, 130])
def test_many_layers(gpu, pkg, n_layers):
    """As many as one launch takes, and more: kept rows and copied pages of each."""
    b = Batch(n_layers, E5M2, 64, 1, 16, [6, 3], [20, 9])
    keep, n_keep = lists(b.rng, b.new)
    check_keep(gpu, pkg, b, n_layers, keep, n_keep)
    check_fork(gpu, pkg, Batch(n_layers, E5M2, 64, 1, 16, [1, 1], [20, 9], spare=4), n_layers, [0, 0, 1], None, [1, 1, 0])


def check_fork(gpu, pkg, b, n_layers, parent, rows, grow, reserved=None, ctx=None, fill=0x7F):
    """The tables, lengths and pools after a fork; returns the table.  ctx: the lengths in memory."""
    torch, dev, lib = gpu
    layers = Layers(b, n_layers, torch, dev)
    if ctx is not None: b.dev["ctx_len"].copy_(torch.from_numpy(np.array(ctx, dtype=np.int32)))
    b.dev["seq_start"].fill_(-1)                # not looked at
    before, caches, n = layers.pools(), layers.caches(pkg), len(parent)
    want, lengths, missing, copies = fork(b.table, b.ctx if ctx is None else ctx, b.page, b.n_pages, parent, rows, grow, reserved)
    table, ctx_out, lost = (torch.full((k,), -9, dtype=torch.int32, device=dev) for k in (n * b.table_stride + 1, n + 1, 2))
    need = lib.kv_paged_fork_workspace_bytes(caches, n_layers, n)
    ws = torch.full((need + 16,), fill, dtype=torch.uint8, device=dev)
    pd, rd, gd = ints(torch, dev, parent), None if rows is None else ints(torch, dev, rows), ints(torch, dev, grow)
    res = None if reserved is None else torch.from_numpy(np.asarray(reserved, dtype=np.uint8)).to(dev)
    for _ in range(2):                          # the same again: what it reads stays
        assert lib.kv_paged_fork(caches, n_layers, n, ptr(pd), ptr(rd), ptr(gd), ptr(res), ptr(table), ptr(ctx_out), ptr(lost), ptr(ws), need) == 0
        torch.cuda.synchronize()
        got = table.cpu().numpy()
        assert np.array_equal(got[:-1].reshape(n, -1), want) and got[-1] == -9
        assert ctx_out.cpu().tolist() == lengths.tolist() + [-9] and lost.cpu().tolist() == [missing, -9]
        assert (ws[need:] == fill).all()
    for pools, old in zip(layers.pools(), before):
        for name in pools:
            new = old[name].copy()
            for src, dst, r in copies: new[dst, :, :r] = old[name][src, :, :r]
            assert np.array_equal(pools[name], new), name
    return want


def shared(b, rng, groups, prefix):
    """Sequences g, g + groups, ... share `prefix` pages of the first of them."""
    for s in range(groups, b.n_seqs): b.table[s, :prefix] = b.table[s % groups, :prefix]
    return b


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_kv,page,ctx,n_layers", [(128, 1, 16, [1], 1), (64, 2, 16, [37, 33, 48, 64], 2), (128, 8, 32, [200, 200, 200, 200, 31, 32], 2), (64, 16, 64, [1000, 70, 5, 0, 64, 128, 129], 2), (64, 1, 4096, [5000, 4096], 1)])
@pytest.mark.parametrize("case", ["beams", "same", "all of one", "parts", "fresh", "fewer", "more"])
def test_fork(gpu, pkg, kind, dim, n_kv, page, ctx, n_layers, case):
    n = len(ctx)
    b = Batch(dim + sum(ctx) + kind, kind, dim, n_kv, page, [1] * n, ctx, spare=3 * n + 9, table_extra=3)
    if n > 2: shared(b, b.rng, 2, min(c // page for c in ctx[:4]))
    n_out = {"fewer": max(n // 2, 1), "more": 3 * n + 1}.get(case, n)
    parent = {"same": np.arange(n), "all of one": np.full(n, n - 1)}.get(case, b.rng.integers(0, n, n_out))
    rows = np.array([b.rng.integers(0, ctx[p] + 3) for p in parent]) if case in ("parts", "more") else None
    grow = b.rng.integers(0, 2 * page, n_out) if case in ("fresh", "fewer", "parts") else np.ones(n_out, dtype=int)
    if case == "fresh": parent = np.where(b.rng.random(n) < 0.5, -1, parent)
    reserved = b.rng.random(b.n_pages) < 0.2 if case in ("parts", "beams") else None
    check_fork(gpu, pkg, b, n_layers, parent, rows, grow, reserved)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_fork_where_something_is_not_right(gpu, pkg, kind):
    """Pages outside the pool, parents that are none, lengths and growth beyond the table or negative; no pages left, for copies or for rows to come; everything reserved."""
    b = Batch(kind, kind, 64, 2, 16, [1] * 4, [40, 20, 64, 7], spare=3)
    b.table[0, 1], b.table[2, 3], b.table[1, 1] = -1, 10 ** 9, -2 ** 31
    check_fork(gpu, pkg, b, 2, [0, 2, 0, 1, 1, 3, 3], None, [1, 0, 30, 1, 1, 1, 1])
    b = Batch(kind, kind, 64, 2, 16, [1] * 4, [40, 20, 64, 7], spare=2)
    check_fork(gpu, pkg, b, 2, [-1, 4, 2 ** 31 - 1, -2 ** 31], None, [3, 70, 0, 5])
    b = Batch(kind, kind, 64, 2, 16, [1] * 4, [40, 20, 64, 7], spare=2)
    check_fork(gpu, pkg, b, 2, [0, 1, 2, 3], [-1, 2 ** 31 - 1, -2 ** 31, 3], [2 ** 31 - 1, -5, -2 ** 31, 2 ** 31 - 1])
    b = Batch(kind, kind, 64, 2, 16, [1] * 4, [40, 20, 64, 7], spare=2)
    check_fork(gpu, pkg, b, 2, [0, 0, 1, 1, 1, 3, 3, 2], None, [0, 40, 0, 1, 20, 0, 0, 1])
    b = Batch(kind, kind, 64, 2, 16, [1] * 4, [40, 20, 64, 7], spare=2)
    check_fork(gpu, pkg, b, 2, [0, 1, 2, 3], None, [1, 1, 1, 1], reserved=np.ones(b.n_pages))
    b = Batch(kind, kind, 64, 2, 16, [1] * 3, [40, 20, 64], spare=20, table_extra=0)
    check_fork(gpu, pkg, b, 2, [0, 1, 2, 1], None, [1, 1, 1, 0], ctx=[2 ** 31 - 1, -4, 70])


def test_a_page_that_is_whole_for_one_and_last_for_another(gpu, pkg):
    """A part of a longer sequence's rows ends within a page that the longer one keeps; one sequence takes over its own beginning."""
    b = Batch(1, BF16, 64, 1, 16, [1, 1], [50, 30], spare=6)
    want = check_fork(gpu, pkg, b, 1, [0, 0, 0, 1, 1], [50, 20, 20, 3, 30], [1, 1, 1, 1, 1])
    # the first keeps its pages, two get their own second one; of the last two the longer has the first page whole
    assert want[0, 1] == b.table[0, 1] and len(set(want[:3, 1])) == 3 and want[3, 0] != b.table[1, 0] == want[4, 0]


@pytest.mark.parametrize("n_seqs,n_out,ctx,page", [(1000, 3000, 70, 16), (65536, 65536, 17, 16), (3, 1500, 4000, 16), (40, 40, 60000, 16)])
def test_many_sequences_and_pages(gpu, pkg, n_seqs, n_out, ctx, page):
    """Tables alone (one head of 64, one layer), more sequences and pages than threads: tables, lengths and a sample of the copied rows."""
    torch, dev, lib = gpu
    rng = np.random.default_rng(n_seqs)
    per = -(-ctx // page)
    stride, n_pages = per + 2, n_seqs * per + 2 * n_out + 5
    table = rng.permutation(n_pages)[:n_seqs * per].reshape(n_seqs, per)
    table = np.concatenate([table, np.full((n_seqs, 2), -1)], 1).astype(np.int32)
    lengths = rng.integers(0, ctx + 1, n_seqs).astype(np.int32)
    parent, grow = rng.integers(0, n_seqs, n_out).astype(np.int32), rng.integers(0, 2, n_out).astype(np.int32)
    want, want_ctx, missing, copies = fork(table, lengths, page, n_pages, parent, None, grow, None)
    assert missing == 0
    pool = torch.arange(n_pages, device=dev).to(torch.int16)[:, None].expand(-1, page * 64).contiguous()
    td, ld = torch.from_numpy(table).to(dev), torch.from_numpy(lengths).to(dev)
    cache = pkg.capi.paged_layers([pkg.capi.make_paged_kv(BF16, 64, 1, page, n_pages, ptr(pool), ptr(pool), ptr(td), stride, ptr(ld), ptr(ld), n_seqs)])
    other = pool.clone()
    cache[0].v = ptr(other)
    out, ctx_out, lost = torch.zeros(n_out, stride, dtype=torch.int32, device=dev), torch.zeros(n_out, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    need = lib.kv_paged_fork_workspace_bytes(cache, 1, n_out)
    ws, pd, gd = torch.zeros(need, dtype=torch.uint8, device=dev), torch.from_numpy(parent).to(dev), torch.from_numpy(grow).to(dev)
    assert lib.kv_paged_fork(cache, 1, n_out, ptr(pd), None, ptr(gd), None, ptr(out), ptr(ctx_out), ptr(lost), ptr(ws), need) == 0
    assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(ctx_out.cpu().numpy(), want_ctx) and int(lost) == 0
    rows = np.arange(page)
    expect = np.repeat(np.arange(n_pages).astype(np.int16)[:, None], page, 1)
    for src, dst, r in copies: expect[dst, rows < r] = np.array(src, dtype=np.int64).astype(np.int16)
    for p in (pool, other): assert np.array_equal(p.view(n_pages, page, 64)[:, :, 5].cpu().numpy(), expect)


@pytest.mark.parametrize("kind", [BF16, E5M2])
def test_captured_moves(gpu, pkg, kind):
    """Keep and fork captured once, replayed on a stream of their own with other lists and lengths: every replay as the eager calls."""
    torch, dev, lib = gpu
    n, tokens = 3, 30
    b = Batch(kind, kind, 64, 2, 16, [10, 10, 10], [100, 50, 20], spare=12)
    layers = Layers(b, 2, torch, dev)
    caches = layers.caches(pkg)
    keep, n_keep, parent, grow = (torch.zeros(k, dtype=torch.int32, device=dev) for k in (tokens, n, n, n))
    table, ctx_out, ctx_kept, lost = torch.zeros(n, b.table_stride, dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    need = lib.kv_paged_fork_workspace_bytes(caches, 2, n)
    ws = torch.zeros(need, dtype=torch.uint8, device=dev)

    def step():
        assert lib.kv_paged_keep(caches, 2, ptr(keep), ptr(n_keep), tokens, 10, ptr(ctx_kept)) == 0
        assert lib.kv_paged_fork(caches, 2, n, ptr(parent), ptr(ctx_kept), ptr(grow), None, ptr(table), ptr(ctx_out), ptr(lost), ptr(ws), need) == 0

    names = ("k", "v") if kind == BF16 else ("k", "v", "k_scale", "v_scale")
    held = [x.dev[name] for x in layers.batches for name in names]
    start = [t.clone() for t in held]
    stream = torch.cuda.Stream(device=dev)
    lib.set_sync(False)
    try:
        lib.set_stream(stream.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream): step()
        for i in range(4):
            k, m = lists(b.rng, b.new)
            keep.copy_(torch.from_numpy(k)); n_keep.copy_(torch.from_numpy(m))
            parent.copy_(torch.from_numpy(b.rng.integers(0, n, n).astype(np.int32))); grow.copy_(torch.from_numpy(b.rng.integers(0, 12, n).astype(np.int32)))
            b.dev["ctx_len"].copy_(torch.tensor([100 - i, 50 - 9 * i, 20 + i], dtype=torch.int32))
            results = []
            for how in ("eager", "graph", "graph"):
                for t, o in zip(held, start): t.copy_(o)
                for t in (table, ctx_out, ctx_kept, lost): t.fill_(-3)
                torch.cuda.synchronize()
                if how == "eager": step()
                else:
                    with torch.cuda.stream(stream): graph.replay()
                torch.cuda.synchronize()
                results.append([t.clone() for t in held + [table, ctx_out, ctx_kept, lost]])
            for other in results[1:]: assert all(torch.equal(u, v) for u, v in zip(results[0], other)), i
    finally:
        lib.set_stream(None)
        lib.set_sync(True)
