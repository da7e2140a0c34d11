"""Attention of trees of new tokens on a paged cache against its formula in 64 bits: shapes, windows, bits that name nobody, what is not seen, pages and lengths that are not right, graphs."""
import numpy as np
import pytest

from branch_util import bits, tree_attend, tree_keys, trees
from paged_util import BF16, E4M3, E5M2, Batch, code_values, from_bf16, to_bf16
from test_gpu_paged import KINDS, ptr, put, run_attend
from test_gpu_paged_edges import odd_codes

pytestmark = pytest.mark.gpu


def run_tree(gpu, pkg, b, q, n_q, seen, window=0, n_sink=0, workspace=1.0, max_new=None, max_ctx=None, pad=0, extra=1, more=0, **other):
    """Rows of y (one more than there are tokens, ending as they began).  seen: per sequence [n][n], or the words; bits behind hold anything, rows are `more` words longer."""
    torch, dev, lib = gpu
    tokens, dim = b.tokens, b.dim
    max_new, max_ctx = max_new or max(b.new), max_ctx or max(b.ctx)
    stride = -(-max_new // 64) + more
    words = np.zeros((tokens + extra, stride), dtype=np.int64)
    words[:tokens] = bits(seen, stride, np.random.default_rng(1)) if isinstance(seen, list) else seen
    wd = torch.from_numpy(words).to(dev)
    ld = n_q * dim + pad
    qd = torch.zeros(tokens + extra, ld, dtype=torch.int16, device=dev)
    qd[:tokens, :n_q * dim] = put(torch, dev, to_bf16(q).reshape(tokens, -1))
    y = torch.full((tokens + extra, ld), 0x1234, dtype=torch.int16, device=dev)
    cache = b.descriptor(pkg, **other)
    need = lib.attention_paged_tree_workspace_bytes(cache, n_q, tokens + extra, max_new, max_ctx, window, n_sink)
    need = int(need * workspace) & ~15
    ws = torch.full((need + 16,), 0x7F, dtype=torch.uint8, device=dev) if need else None
    assert lib.attention_paged_tree(cache, ptr(qd), ptr(y), ptr(wd), stride, ptr(ws), need if ws is not None else 0, n_q, tokens + extra, max_new, max_ctx, window, n_sink, ld, ld) == 0
    torch.cuda.synchronize()
    if ws is not None: assert (ws[need:] == 0x7F).all()
    out = y.cpu().numpy().view(np.uint16)
    assert (out[tokens:] == 0x1234).all() and (out[:, n_q * dim:] == 0x1234).all()
    return out[:tokens, :n_q * dim].reshape(tokens, n_q, dim)


def check_tree(gpu, pkg, b, n_q, seen, window=0, n_sink=0, q=None, rows=None, lost=None, **kw):
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, b.dim)) * 1.3)) if q is None else q
    got = from_bf16(run_tree(gpu, pkg, b, q, n_q, seen, window, n_sink, **kw))
    want, bound = tree_attend(b, q, n_q, seen, window, n_sink, rows, lost)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want)[bad][:5], bound[bad][:5])
    return got


SHAPES = [  # dim, n_q, n_kv, page, new, ctx
    (128, 4, 1, 16, [1], [1]), (128, 4, 1, 16, [4], [4]), (64, 8, 1, 16, [2, 1, 0, 2], [64, 300, 20, 7]), (128, 8, 8, 32, [16, 3], [127, 513]), (128, 3, 1, 64, [5, 2], [33, 129]), (64, 10, 2, 16, [3, 1, 3], [3, 200, 70]),
    (128, 8, 2, 16, [13], [4108]), (128, 4, 1, 32, [129], [129]), (64, 4, 2, 64, [65, 1, 30], [465, 400, 90]), (128, 16, 1, 128, [9, 70], [500, 71]), (128, 2, 2, 16, [64, 3], [700, 64]), (64, 64, 1, 16, [1, 5], [90, 1030]),
    (128, 4, 1, 16, [4, 60, 4], [64, 1500, 68]), (64, 8, 2, 16, [33, 5, 70, 17], [2100, 1300, 70, 3000]), (128, 16, 4, 32, [26] * 5, [1700, 26, 130, 900, 2500])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,page,new,ctx", SHAPES)
@pytest.mark.parametrize("window,n_sink", [(0, 0), (1, 0), (37, 0), (64, 4), (100, 70)])
def test_trees(gpu, pkg, kind, dim, n_q, n_kv, page, new, ctx, window, n_sink):
    b = Batch(dim + n_q + sum(ctx) + kind, kind, dim, n_kv, page, new, ctx).upload(*gpu[:2])
    check_tree(gpu, pkg, b, n_q, trees(b.rng, new), window, n_sink, pad=8, more=dim // 128)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,new,ctx", [(128, 4, 1, [4, 3], [4, 67]), (64, 4, 2, [8], [200]), (128, 4, 2, [100, 30], [100, 300]), (64, 8, 1, [140], [333])])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (20, 3)])
def test_any_bits(gpu, pkg, kind, dim, n_q, n_kv, new, ctx, window, n_sink):
    """Bits that form no tree: later tokens, not itself, none at all -- a token that sees nothing, with no rows in front, gives 0."""
    b = Batch(dim + sum(ctx) + kind, kind, dim, n_kv, 16, new, ctx).upload(*gpu[:2])
    seen = [b.rng.random((n, n)) < 0.4 for n in new]
    for s in seen:
        s[1] = False
        s[2] = True
    got = check_tree(gpu, pkg, b, n_q, seen, window, n_sink)
    if new[0] == ctx[0]: assert not got[1].any()


# single tokens, a few, tiles, in one piece and in parts
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,new,ctx,window,n_sink", [(64, 4, 2, [3, 5], [50, 300], 0, 0), (128, 4, 1, [4, 4], [64, 3000], 70, 3), (128, 4, 1, [40, 1], [90, 70], 0, 0), (64, 8, 1, [130], [200], 0, 0),
                                                                (128, 2, 1, [70, 20], [300, 500], 50, 5), (64, 2, 2, [200], [1400], 0, 0)])
def test_what_is_not_seen_does_not_reach_a_token(gpu, pkg, kind, dim, n_q, n_kv, new, ctx, window, n_sink):
    """Every row that no new token sees, and rows of the pool that hold nothing, are infinite or NaN, keys and values; among the new tokens one is infinite or NaN in both, and one more in a
    few dims of its values: tokens that do not see them are as without them, tokens that see the first are NaN, those that see the second not finite there."""
    b = Batch(dim + sum(ctx) + kind, kind, dim, n_kv, 16, new, ctx)
    seen = trees(b.rng, new)
    keep = np.zeros((b.n_pages, 16), dtype=bool)
    for s in range(b.n_seqs):
        any_see = np.any([tree_keys(ctx[s], ctx[s] - new[s], one, window, n_sink) for one in seen[s]], axis=0)
        for pos in np.flatnonzero(any_see): keep[b.table[s, pos // 16], pos % 16] = True
    rows = {name: [b.rows(name, s) for s in range(b.n_seqs)] for name in ("k", "v")}
    bad = odd_codes(kind)
    for name in ("k", "v"):
        wild = b.rng.choice(bad, size=b.pool[name].shape).astype(b.pool[name].dtype)
        b.pool[name] = np.where(keep[:, None, :, None], b.pool[name], wild)
        if kind != BF16: b.scale[name] = np.where(keep[:, None, :], b.scale[name], np.uint8(255))
    both, few = np.zeros(b.tokens, dtype=bool), np.zeros(b.tokens, dtype=bool)
    for s in range(b.n_seqs):
        if new[s] < 3: continue
        first, t0 = ctx[s] - new[s], int(b.seq_start[s])
        i, j = new[s] - 1, new[s] // 2
        for name in ("k", "v"): b.pool[name][b.table[s, (first + i) // 16], :, (first + i) % 16] = bad[-1]
        b.pool["v"][b.table[s, (first + j) // 16], :, (first + j) % 16, 3::17] = bad[0]
        rows["v"][s][:, first + j, 3::17] = 0.0
        both[t0:t0 + new[s]], few[t0:t0 + new[s]] = seen[s][:, i], seen[s][:, j]
    b.upload(*gpu[:2])
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim))))
    got = from_bf16(run_tree(gpu, pkg, b, q, n_q, seen, window, n_sink))
    want, bound = tree_attend(b, q, n_q, seen, window, n_sink, rows=rows)
    assert np.isnan(got[both]).all()
    assert not np.isfinite(got[few & ~both][..., 3::17]).any()
    reached = np.zeros(got.shape, dtype=bool)
    reached[both] = True
    reached[few, :, 3::17] = True
    assert (np.abs(got - want) <= bound)[~reached].all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,ctx", [([3, 4], [100, 90]), ([70], [300]), ([4], [2500])])
@pytest.mark.parametrize("wrong", [-1, 10 ** 9, -2 ** 31])
def test_pages_outside_the_pool(gpu, pkg, kind, new, ctx, wrong):
    b = Batch(sum(ctx) + kind, kind, 64, 2, 16, new, ctx)
    rows = {name: [b.rows(name, s) for s in range(b.n_seqs)] for name in ("k", "v")}
    lost = [np.zeros(c, dtype=bool) for c in ctx]
    for s in range(b.n_seqs):
        pages = -(-ctx[s] // 16)
        b.table[s, pages:] = wrong
        for page in {1, pages // 2, pages - 1}:
            b.table[s, page] = wrong
            lost[s][16 * page:16 * page + 16] = True
    b.upload(*gpu[:2])
    check_tree(gpu, pkg, b, 4, trees(b.rng, new), rows=rows, lost=lost)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_lengths_that_are_not_right(gpu, pkg, kind):
    """More new tokens than rows: those at negative positions are seen by nobody.  A sequence with more new tokens than max_new is left out, ranges that are not in order stay within
    the activations."""
    torch, dev, lib = gpu
    b = Batch(7, kind, 64, 1, 16, [4, 30, 2, 1], [2, 20, 64, 5]).upload(torch, dev)
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, 4, 64))))
    seen = trees(b.rng, b.new)
    got = from_bf16(run_tree(gpu, pkg, b, q, 4, seen))
    want, bound = tree_attend(b, q, 4, seen)
    there = np.array([any(t == x for x, _, _ in b.slots()) for t in range(b.tokens)])
    assert (np.abs(got - want) <= bound)[there].all() and np.isfinite(got).all()
    b = Batch(8, kind, 64, 1, 16, [1, 20], [90, 100]).upload(torch, dev)
    q, seen = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, 4, 64)))), trees(b.rng, b.new)
    want = run_tree(gpu, pkg, b, q, 4, seen)
    got = run_tree(gpu, pkg, b, q, 4, seen, max_new=19)
    assert np.array_equal(got[0], want[0]) and (got[1:] == 0x1234).all()
    for starts in ([5, 1, 0], [-7, 3, 2], [21, 21, 21], [2 ** 31 - 1, -2 ** 31, 4], [0, 2 ** 31 - 1, 2 ** 31 - 1]):
        b.dev["seq_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        run_tree(gpu, pkg, b, q, 4, seen, max_new=64, max_ctx=100)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,ctx", [([1, 1], [700, 64]), ([4], [3000]), ([100], [500]), ([2, 60], [30, 2000])])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (90, 5)])
def test_a_line_is_causal_attention(gpu, pkg, kind, new, ctx, window, n_sink):
    """Tokens that see all in front of them: as hip_attention_paged_bf16, up to the order of FP32 sums and a weight's rounding (two bounds of the formula)."""
    b = Batch(sum(ctx) + kind, kind, 128, 1, 16, new, ctx).upload(*gpu[:2])
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, 4, 128))))
    line = [np.tril(np.ones((n, n), dtype=bool)) for n in new]
    got = from_bf16(run_tree(gpu, pkg, b, q, 4, line, window, n_sink))
    causal = from_bf16(run_attend(gpu, pkg, b, q, 4, window, n_sink))
    _, bound = tree_attend(b, q, 4, line, window if max(new) == 1 else 0, n_sink)
    if not window or max(new) == 1: assert (np.abs(got - causal) <= 2 * bound).all()
    else: check_tree(gpu, pkg, b, 4, line, window, n_sink, q=q)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,page,new,ctx", [(128, 4, 1, 16, [4], [4000]), (128, 8, 2, 32, [4, 1, 3], [3000, 100, 900]), (64, 8, 8, 64, [100], [3000]), (128, 4, 2, 16, [1, 40, 1], [2000, 1500, 30])])
def test_workspaces(gpu, pkg, kind, dim, n_q, n_kv, page, new, ctx):
    """Without a workspace: within the formula's bound; with one that holds anything: the same bits, a hundred times."""
    torch, dev, lib = gpu
    b = Batch(sum(ctx) + kind, kind, dim, n_kv, page, new, ctx).upload(torch, dev)
    q, seen = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim)))), trees(b.rng, new)
    want = check_tree(gpu, pkg, b, n_q, seen, q=q)
    for part in (0, 0.1, 0.5, 0.9): check_tree(gpu, pkg, b, n_q, seen, q=q, workspace=part)
    cache, stride = b.descriptor(pkg), -(-max(new) // 64)
    need = lib.attention_paged_tree_workspace_bytes(cache, n_q, b.tokens, max(new), max(ctx))
    qd, wd, y = put(torch, dev, to_bf16(q)), torch.from_numpy(bits(seen, stride)).to(dev), torch.zeros(b.tokens, n_q * dim, dtype=torch.int16, device=dev)
    first = None
    for i in range(100):
        ws = torch.full((need,), i % 256, dtype=torch.uint8, device=dev) if i % 10 == 0 else ws
        y.zero_()
        assert lib.attention_paged_tree(cache, ptr(qd), ptr(y), ptr(wd), stride, ptr(ws), need, n_q, b.tokens, max(new), max(ctx), 0, 0, n_q * dim, n_q * dim) == 0
        got = y.cpu().numpy()
        first = got if first is None else first
        assert np.array_equal(got, first), i
    assert (np.abs(from_bf16(first.view(np.uint16)).reshape(want.shape) - want) <= 2 * tree_attend(b, q, n_q, seen)[1]).all()


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_a_captured_call_with_other_trees(gpu, pkg, kind):
    """Captured once, replayed with other lengths and bits on a stream of its own, two graphs on one workspace one behind the other: the bits of eager calls."""
    torch, dev, lib = gpu
    n_q, n_kv, dim, page, tokens, most = 8, 2, 128, 16, 40, 1600
    b = Batch(3, kind, dim, n_kv, page, [4, 4, 32], [1500, 40, 700], table_extra=70).upload(torch, dev)
    q = [put(torch, dev, to_bf16(b.rng.standard_normal((tokens, n_q * dim)))) for _ in range(2)]
    y = [torch.zeros(tokens, n_q * dim, dtype=torch.int16, device=dev) for _ in range(2)]
    words = torch.zeros(tokens, 1, dtype=torch.int64, device=dev)
    cache = b.descriptor(pkg)
    need = lib.attention_paged_tree_workspace_bytes(cache, n_q, tokens, tokens, most)
    spaces = [torch.full((need,), 0x55, dtype=torch.uint8, device=dev) for _ in range(2)]
    call = lambda i, ws: lib.attention_paged_tree(cache, ptr(q[i]), ptr(y[i]), ptr(words), 1, ptr(ws), need, n_q, tokens, tokens, most, 0, 0, n_q * dim, n_q * dim)  # noqa: E731
    stream = torch.cuda.Stream(device=dev)
    lib.set_sync(False)
    try:
        lib.set_stream(stream.cuda_stream)
        graphs = []
        for i in range(2):
            torch.cuda.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[i], stream=stream): assert call(i, spaces[0]) == 0
        for lengths, starts in (([1500, 40, 700], [0, 4, 8, 40]), ([1501, 41, 720], [0, 1, 2, 22]), ([17, 1300, 60], [0, 0, 19, 21]), ([1502, 42, 721], [0, 1, 2, 3]), ([0, 0, 0], [0, 0, 0, 0])):
            b.dev["ctx_len"].copy_(torch.tensor(lengths, dtype=torch.int32))
            b.dev["seq_start"].copy_(torch.tensor(starts, dtype=torch.int32))
            new = [starts[i + 1] - starts[i] for i in range(3)]
            words.zero_()
            words[:sum(new)] = torch.from_numpy(bits(trees(b.rng, new), 1)).to(dev) if sum(new) else words[:0]
            want = []
            for i in range(2):
                y[i].fill_(7)
                torch.cuda.synchronize()
                assert call(i, spaces[1]) == 0
                torch.cuda.synchronize()
                want.append(y[i].clone())
                y[i].fill_(7)
            for _ in range(2):
                with torch.cuda.stream(stream):
                    for g in graphs: g.replay()
                torch.cuda.synchronize()
                for i in range(2):
                    assert torch.equal(y[i], want[i])
                    y[i].fill_(7)
                torch.cuda.synchronize()
    finally:
        lib.set_stream(None)
        lib.set_sync(True)


@pytest.mark.parametrize("kind", KINDS)
def test_far_positions(gpu, pkg, kind):
    """A tree behind 2^30 - 70 rows, whose pages are three of 4096 rows over and over, with a window."""
    torch, dev, lib = gpu
    ctx, n_q, dim, window, n_sink, new = 1 << 30, 2, 128, 300, 70, 70
    b = Batch(kind, kind, dim, 1, 4096, [new], [3 * 4096], spare=0, table_extra=0)
    table = np.arange(ctx // 4096, dtype=np.int32) % 3
    b.upload(torch, dev)
    b.dev["table"], b.table_stride = torch.from_numpy(table).to(dev), len(table)
    b.dev["ctx_len"].fill_(ctx)
    q, seen = from_bf16(to_bf16(b.rng.standard_normal((new, n_q, dim)))), trees(b.rng, [new])
    got = from_bf16(run_tree(gpu, pkg, b, q, n_q, seen, window, n_sink, max_ctx=ctx))
    # the same over the rows that any token sees, one behind the other: the first ones, then from the first window on
    first = ctx - new
    pos = np.concatenate([np.arange(n_sink), np.arange(first - window, ctx)])
    k, v = (b.values(name)[table[pos // 4096], 0, pos % 4096] for name in ("k", "v"))
    for t in range(new):
        at = first + seen[0][t].sum() - 1
        see = np.where(pos < first, (pos > at - window) | (pos < n_sink), np.concatenate([np.zeros(n_sink + window, dtype=bool), seen[0][t]]))
        for h in range(n_q):
            score = k[see] @ q[t, h] / np.sqrt(dim)
            w = np.exp(score - score.max())
            w /= w.sum()
            # a probability's and the result's rounding, 2^-8 each, and room for FP32
            assert (np.abs(got[t, h] - w @ v[see]) <= 2.0 ** -7 * (w @ np.abs(v[see])) + 2.0 ** -8 * np.abs(w @ v[see])).all()


@pytest.mark.parametrize("kind", [BF16, E5M2])
@pytest.mark.parametrize("n_seqs,big,n_q,n_kv", [(300, 3, 2, 1), (520, 7, 4, 1), (90, 1, 32, 8), (257, 1, 4, 4)])
def test_many_sequences(gpu, pkg, kind, n_seqs, big, n_q, n_kv):
    """More sequences than are looked up at once, every `big`-th one in tiles, and more tiles than run at once."""
    rng = np.random.default_rng(n_seqs)
    new = [int(rng.integers(34, 50)) if s % big == 0 else int(rng.integers(0, 5)) for s in range(n_seqs)] if n_seqs != 257 else [int(rng.integers(0, 17)) for _ in range(n_seqs)]
    ctx = [n + int(rng.integers(0, 300)) for n in new]
    ctx[n_seqs // 2] = new[n_seqs // 2] + 2000
    b = Batch(n_seqs + kind, kind, 64, n_kv, 16, new, ctx).upload(*gpu[:2])
    seen = trees(rng, new)
    q = from_bf16(to_bf16(rng.standard_normal((b.tokens, n_q, 64))))
    values = {name: b.values(name) for name in ("k", "v")}
    rows = {name: [values[name][b.table[s, np.arange(c) // 16], :, np.arange(c) % 16].transpose(1, 0, 2) for s, c in enumerate(ctx)] for name in ("k", "v")}
    got = [from_bf16(run_tree(gpu, pkg, b, q, n_q, seen, workspace=part)) for part in (1.0, 0.3, 0)]
    few = np.zeros(b.tokens, dtype=bool)        # every third sequence and the long one, against the formula
    for s in range(n_seqs):
        if s % 3 == 0 or s == n_seqs // 2: few[b.seq_start[s]:b.seq_start[s + 1]] = True
    for s in range(n_seqs):
        if not (s % 3 == 0 or s == n_seqs // 2): b.new[s] = 0       # (the formula's; what lies on the device stays)
    want, bound = tree_attend(b, q, n_q, seen, rows=rows)
    for y in got:
        assert (np.abs(y - want) <= bound)[few].all()
        # the others: two results, each off by a weight's and a result's rounding, 2^-8 of a mean of |v| (under 4) and of itself
        assert (np.abs(y - got[0])[~few] <= 2.0 ** -6 * np.abs(got[0])[~few] + 4 * 2.0 ** -6).all()


def test_two_streams_at_once(gpu, pkg):
    """Two batches on streams and workspaces of their own, calls among each other: the bits of calls alone."""
    torch, dev, lib = gpu
    sides = []
    for i in range(2):
        b = Batch(i, E4M3, 128, 2, 16, [40, 4, 20], [3000 - 900 * i, 700, 1500 + 400 * i]).upload(torch, dev)
        q = put(torch, dev, to_bf16(b.rng.standard_normal((b.tokens, 8 * 128))))
        cache, words = b.descriptor(pkg), torch.from_numpy(bits(trees(b.rng, b.new), 1)).to(dev)
        need = lib.attention_paged_tree_workspace_bytes(cache, 8, b.tokens, 40, max(b.ctx))
        sides.append((b, q, torch.zeros_like(q), cache, words, need, torch.zeros(need, dtype=torch.uint8, device=dev), torch.cuda.Stream(device=dev)))
    def call(b, q, y, cache, words, need, ws, _):
        assert lib.attention_paged_tree(cache, ptr(q), ptr(y), ptr(words), 1, ptr(ws), need, 8, b.tokens, 40, max(b.ctx), 0, 0, 1024, 1024) == 0
    want = []
    for s in sides:
        call(*s)
        torch.cuda.synchronize()
        want.append(s[2].clone())
    lib.set_sync(False)
    try:
        for _ in range(20):
            for s in sides: s[2].zero_()
            torch.cuda.synchronize()
            for _ in range(5):
                for s in sides:
                    lib.set_stream(s[-1].cuda_stream)
                    call(*s)
            torch.cuda.synchronize()
            for s, w in zip(sides, want): assert torch.equal(s[2], w)
    finally:
        lib.set_stream(None)
        lib.set_sync(True)
