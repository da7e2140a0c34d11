"""Operators on a paged cache at the ends of what their entries take, and calls beside and behind each other: the most sequences, the most positions, the largest page, the most kv heads, windows and
first tokens past every length, two graphs on one workspace, two streams at once."""
import numpy as np
import pytest

from paged_util import BF16, E4M3, E5M2, Batch, attend, from_bf16, to_bf16
from test_gpu_paged import KINDS, check_attend, ptr, put, run_attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_65536_sequences(gpu, pkg, kind):
    """One token each on one to 33 rows, in pages that thousands share: read back exactly, attention as the formula; appended to pages of their own, every row where it belongs."""
    torch, dev, lib = gpu
    n, n_q, dim, pages = 65536, 2, 64, 50
    b = Batch(kind, kind, dim, 1, 16, [1], [16 * pages], spare=0)
    seq = np.arange(n)
    length = 1 + seq % 33
    table = np.stack([seq % pages, seq * 7 % pages, seq * 11 % pages], 1).astype(np.int32)
    b.upload(torch, dev)
    for name, a in (("table", table), ("ctx_len", length.astype(np.int32)), ("seq_start", np.arange(n + 1, dtype=np.int32))): b.dev[name] = torch.from_numpy(a).to(dev)
    b.n_seqs, b.table_stride = n, 3
    cache = b.descriptor(pkg)
    out = torch.full((2, n, dim), 0x1234, dtype=torch.int16, device=dev)
    assert lib.kv_paged_read(cache, ptr(out[0]), ptr(out[1]), n, dim, dim) == 0
    back, last = from_bf16(out.cpu().numpy().view(np.uint16)), length - 1
    for i, name in enumerate(("k", "v")): assert np.array_equal(back[i], b.values(name)[table[seq, last // 16], 0, last % 16])
    q = put(torch, dev, to_bf16(b.rng.standard_normal((n, n_q, dim))))
    y = torch.full_like(q, 0x1234)
    need = lib.attention_paged_workspace_bytes(cache, n_q, n, 1, 48)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    assert lib.attention_paged(cache, ptr(q), ptr(y), ptr(ws), need, n_q, n, 1, 48, 0, 0, n_q * dim, n_q * dim) == 0
    got, qf = from_bf16(y.cpu().numpy().view(np.uint16)), from_bf16(q.cpu().numpy().view(np.uint16))
    keys = np.arange(33)
    for at in range(0, n, 8192):
        s = seq[at:at + 8192]
        k, v = (b.values(name)[table[s][:, keys // 16], 0, keys % 16] for name in ("k", "v"))      # [sequence][key][dim]
        score = np.where(keys < length[s, None, None], qf[s] @ k.transpose(0, 2, 1) / 8.0, -np.inf)
        w = np.exp(score - score.max(-1, keepdims=True))
        w /= w.sum(-1, keepdims=True)
        # a probability's and the result's rounding, 2^-8 each, and room for FP32
        assert (np.abs(got[s] - w @ v) <= 2.0 ** -7 * (w @ np.abs(v)) + 2.0 ** -8 * np.abs(w @ v)).all()
    if kind == BF16:
        pool = torch.zeros(2, n, 1, 16, dim, dtype=torch.int16, device=dev)
        mine = torch.arange(n, dtype=torch.int32, device=dev).flip(0).contiguous()
        one = torch.from_numpy((1 + seq % 16).astype(np.int32)).to(dev)
        own = pkg.capi.make_paged_kv(BF16, dim, 1, 16, n, ptr(pool[0]), ptr(pool[1]), ptr(mine), 1, ptr(one), ptr(b.dev["seq_start"]), n)
        assert lib.qk_norm_rope_kv_paged(own, None, ptr(out[0]), ptr(out[1]), None, None, None, None, 0, None, 0, n, 0, dim, dim) == 0
        rows = pool[:, mine.long(), 0, (one - 1).long()]
        assert torch.equal(rows, out) and int((pool != 0).sum()) == int((out != 0).sum())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
def test_the_last_position(gpu, pkg, kind, dim, new):
    """A sequence of 2^30 rows, whose pages are three of 4096 rows over and over: append, read back, and attention of a window at its end."""
    torch, dev, lib = gpu
    ctx, n_q, window, n_sink = 1 << 30, 2, 300, 70
    b = Batch(dim + kind + new, kind, dim, 1, 4096, [new], [3 * 4096], spare=0, table_extra=0)
    table = np.arange(ctx // 4096, dtype=np.int32) % 3
    b.upload(torch, dev)
    b.dev["table"], b.table_stride = torch.from_numpy(table).to(dev), len(table)
    b.dev["ctx_len"].fill_(ctx)
    cache, pos = b.descriptor(pkg), np.arange(ctx - new, ctx)
    x = b.rng.integers(-3, 4, (2, new, dim)).astype(np.float64)              # codes hold them
    x[:, :, 0] = 3.0
    xd = put(torch, dev, to_bf16(x))
    before = {n: b.download(n).copy() for n in ("k", "v")}
    assert lib.qk_norm_rope_kv_paged(cache, None, ptr(xd[0]), ptr(xd[1]), None, None, None, None, 0, None, 0, new, 0, dim, dim) == 0
    keep = np.ones((3, 4096), dtype=bool)
    keep[table[pos // 4096], pos % 4096] = False
    for i, name in enumerate(("k", "v")):
        b.pool[name] = b.download(name)
        if kind != BF16: b.scale[name] = b.download(name + "_scale")
        assert np.array_equal(b.pool[name][keep[:, None]], before[name][keep[:, None]])
        assert np.array_equal(b.values(name)[table[pos // 4096], 0, pos % 4096], x[i])
    out = torch.full((2, new, dim), 0x1234, dtype=torch.int16, device=dev)
    assert lib.kv_paged_read(cache, ptr(out[0]), ptr(out[1]), new, dim, dim) == 0
    assert torch.equal(out, xd)
    q = from_bf16(to_bf16(b.rng.standard_normal((new, n_q, dim))))
    qd, y = put(torch, dev, to_bf16(q)), torch.zeros(new, n_q, dim, dtype=torch.int16, device=dev)
    need = lib.attention_paged_workspace_bytes(cache, n_q, new, new, ctx, window, n_sink)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    values = {n: b.values(n) for n in ("k", "v")}
    for given in (need, 0):
        assert lib.attention_paged(cache, ptr(qd), ptr(y), ptr(ws) if given else None, given, n_q, new, new, ctx, window, n_sink, n_q * dim, n_q * dim) == 0
        got = from_bf16(y.cpu().numpy().view(np.uint16))
        for t in range(new):
            seen = np.concatenate([np.arange(n_sink), np.arange(pos[t] - window + 1, pos[t] + 1)])
            k, v = (values[n][table[seen // 4096], 0, seen % 4096] for n in ("k", "v"))
            w = np.exp((score := q[t] @ k.T / np.sqrt(dim)) - score.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            # a probability's and the result's rounding, 2^-8 each, and room for FP32
            assert (np.abs(got[t] - w @ v) <= 2.0 ** -7 * (w @ np.abs(v)) + 2.0 ** -8 * np.abs(w @ v)).all(), (given, t)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,page,new,ctx", [(64, 1024, 1024, 16, [1, 2], [20, 40]), (128, 2, 2, 4096, [1, 30], [5000, 4100]), (64, 64, 1, 32, [1, 1], [700, 60]), (128, 18, 1, 16, [1, 4], [300, 900])])
def test_heads_and_pages(gpu, pkg, kind, dim, n_q, n_kv, page, new, ctx):
    """The most kv heads, the largest page, up to 64 query heads per kv head; a window and first tokens that are past every length, and first tokens alone past it."""
    b = Batch(kind + page, kind, dim, n_kv, page, new, ctx).upload(*gpu[:2])
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim))))
    got = check_attend(gpu, pkg, b, n_q, q=q)
    for window, n_sink in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (max(ctx), 0)): assert np.array_equal(from_bf16(run_attend(gpu, pkg, b, q, n_q, window, n_sink)), got)
    check_attend(gpu, pkg, b, n_q, 5, 2 ** 31 - 1, q=q)
    check_attend(gpu, pkg, b, n_q, max(ctx) - 1, 1, q=q)


class Call:
    """An attention call of a batch with what it needs, on any workspace."""

    def __init__(self, gpu, pkg, seed, kind, dim, n_q, n_kv, new, ctx):
        self.torch, dev, self.lib = gpu
        self.b = Batch(seed, kind, dim, n_kv, 16, new, ctx).upload(self.torch, dev)
        self.n_q, self.ld = n_q, n_q * dim
        self.q = put(self.torch, dev, to_bf16(self.b.rng.standard_normal((self.b.tokens, n_q, dim))))
        self.y = self.torch.zeros_like(self.q)
        self.cache = self.b.descriptor(pkg)
        self.need = self.lib.attention_paged_workspace_bytes(self.cache, n_q, self.b.tokens, max(new), max(ctx))
        assert self.need > 0

    def __call__(self, ws):
        assert self.lib.attention_paged(self.cache, ptr(self.q), ptr(self.y), ptr(ws), ws.numel(), self.n_q, self.b.tokens, max(self.b.new), max(self.b.ctx), 0, 0, self.ld, self.ld) == 0


def two_calls(gpu, pkg, kind):
    """Parts of short sequences; a chunk in ranges beside short sequences.  And the bits of each by itself."""
    torch, dev, _ = gpu
    calls = Call(gpu, pkg, 1, kind, 128, 8, 2, [1, 1, 2], [4000, 300, 2500]), Call(gpu, pkg, 2, kind, 64, 4, 2, [1, 70, 1], [3000, 2000, 90])
    want = []
    for c in calls:
        c(torch.empty(c.need, dtype=torch.uint8, device=dev))
        torch.cuda.synchronize()
        want.append(c.y.clone())
    return calls, want


@pytest.mark.parametrize("kind", [BF16, E5M2])
def test_two_graphs_on_one_workspace(gpu, pkg, kind):
    """Captured apart, replayed in turn in any order, eager calls of both on the same workspace between: the same bits each time."""
    torch, dev, lib = gpu
    calls, want = two_calls(gpu, pkg, kind)
    ws = torch.full((max(c.need for c in calls),), 0xAA, dtype=torch.uint8, device=dev)
    stream = torch.cuda.Stream(device=dev)
    lib.set_sync(False)
    try:
        lib.set_stream(stream.cuda_stream)
        torch.cuda.synchronize()
        graphs = []
        for c in calls:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream): c(ws)
        for round_, order in enumerate(([0, 1], [1, 0, 0], [0, 0, 1, 1], [1])):
            for c in calls: c.y.fill_(0x1234)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                for i in order: graphs[i].replay()
            torch.cuda.synchronize()
            for i in set(order): assert torch.equal(calls[i].y, want[i]), (round_, i)
            for c in calls: c.y.fill_(0x1234)
            torch.cuda.synchronize()
            for c in calls: c(ws)
            torch.cuda.synchronize()
            for c, w in zip(calls, want): assert torch.equal(c.y, w), round_
    finally:
        lib.set_stream(None)
        lib.set_sync(True)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_two_streams_at_once(gpu, pkg, kind):
    """Each with a workspace of its own."""
    torch, dev, lib = gpu
    calls, want = two_calls(gpu, pkg, kind)
    spaces = [torch.full((c.need,), 0x55, dtype=torch.uint8, device=dev) for c in calls]
    streams = [torch.cuda.Stream(device=dev) for _ in calls]
    for c in calls: c.y.fill_(0x1234)
    torch.cuda.synchronize()
    lib.set_sync(False)
    try:
        for _ in range(20):
            for c, ws, s in zip(calls, spaces, streams):
                lib.set_stream(s.cuda_stream)
                c(ws)
        torch.cuda.synchronize()
    finally:
        lib.set_stream(None)
        lib.set_sync(True)
    for c, w in zip(calls, want): assert torch.equal(c.y, w)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 5, 90])
@pytest.mark.parametrize("power", [88, -80])
@pytest.mark.parametrize("workspace", [True, False])
def test_large_and_small_values(gpu, pkg, kind, new, power, workspace):
    """Values times 2^88 or 2^-80: the formula's bound, which is relative to them."""
    b = Batch(kind + new, kind, 128, 1, 16, [new], [2500])
    if kind == BF16: b.pool["v"] = to_bf16(from_bf16(b.pool["v"]) * 2.0 ** power)
    else: b.scale["v"] = (b.scale["v"].astype(int) + power).astype(np.uint8)
    b.upload(*gpu[:2])
    assert np.abs(b.values("v")).max() < 2.0 ** 90
    check_attend(gpu, pkg, b, 4, workspace=workspace)


@pytest.mark.parametrize("kind", KINDS)
def test_calls_repeat_themselves(gpu, pkg, kind):
    """A thousand calls of either kind, one behind the other on one workspace, whose parts pass between workgroups of the whole GPU: the same bits each time."""
    torch, dev, lib = gpu
    calls, want = two_calls(gpu, pkg, kind)
    ws = torch.empty(max(c.need for c in calls), dtype=torch.uint8, device=dev)
    stream, differs = torch.cuda.Stream(device=dev), torch.zeros((), dtype=torch.int64, device=dev)
    torch.cuda.synchronize()
    lib.set_sync(False)
    try:
        lib.set_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            for _ in range(1000):
                for c, w in zip(calls, want):
                    c.y.fill_(0x1234)
                    c(ws)
                    differs += (c.y != w).sum()
        torch.cuda.synchronize()
    finally:
        lib.set_stream(None)
        lib.set_sync(True)
    assert int(differs) == 0
