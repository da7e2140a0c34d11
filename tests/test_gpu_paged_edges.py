"""Operators on a paged cache where they can go wrong: what a token does not see, pages and lengths that are not right, workspaces, graphs, streams, long offsets, shared pages,
many sequences, and the operators one after the other."""
import numpy as np
import pytest

from paged_util import BF16, E4M3, E5M2, Batch, attend, code_values, from_bf16, to_bf16
from test_gpu_paged import KINDS, check_attend, ptr, put, run_append, run_attend

pytestmark = pytest.mark.gpu


def odd_codes(kind):
    """Codes of +inf, -inf and NaN, as far as a type has them."""
    return {BF16: [0x7F80, 0xFF80, 0x7FC0], E4M3: [0x7F, 0xFF], E5M2: [0x7C, 0xFC, 0x7F]}[kind]


# single tokens, a few, tiles, in one piece and in parts; a window leaves rows on both sides unseen
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,new,ctx,window,n_sink", [(128, 4, 1, [1, 1], [37, 130], 0, 0), (64, 4, 2, [3, 5], [50, 300], 0, 0), (128, 4, 1, [40, 1], [90, 70], 0, 0), (64, 8, 1, [130], [200], 0, 0),
                                                                (128, 4, 1, [1, 2], [400, 3000], 70, 3), (128, 2, 1, [70, 20], [300, 500], 50, 5), (64, 2, 2, [200], [1400], 0, 0)])
def test_what_is_not_seen_does_not_reach_a_token(gpu, pkg, kind, dim, n_q, n_kv, new, ctx, window, n_sink):
    """Every row that no new token sees, and rows of the pool that hold nothing, are infinite or NaN, keys and values, their exponents at the limit; of the new tokens' own rows one value
    row is infinite or NaN in a few dims: tokens before it are as without it, tokens that see it are not finite there and as the formula elsewhere."""
    b = Batch(dim + sum(ctx) + kind, kind, dim, n_kv, 16, new, ctx)
    clean = {name: b.rows(name, s) for s in range(b.n_seqs) for name in ("k", "v")}
    keep = np.zeros((b.n_pages, 16), dtype=bool)
    for s in range(b.n_seqs):
        for pos in range(ctx[s]):
            if any(pos <= p and (not window or pos > p - window or pos < n_sink) for p in range(ctx[s] - new[s], ctx[s])):
                keep[b.table[s, pos // 16], pos % 16] = True
    rows = {name: [b.rows(name, s) for s in range(b.n_seqs)] for name in ("k", "v")}
    bad = odd_codes(kind)
    for name in ("k", "v"):
        wild = b.rng.choice(bad, size=b.pool[name].shape).astype(b.pool[name].dtype)
        b.pool[name] = np.where(keep[:, None, :, None], b.pool[name], wild)
        if kind != BF16: b.scale[name] = np.where(keep[:, None, :], b.scale[name], np.uint8(255))
    at = []                                                         # the second new token's values, or the last of a single one's
    for s in range(b.n_seqs):
        if new[s] < 2: continue
        pos = ctx[s] - new[s] + 1
        b.pool["v"][b.table[s, pos // 16], :, pos % 16, 3::17] = bad[s % len(bad)]
        rows["v"][s][:, pos, 3::17] = 0.0
        at.append((s, pos))
    del clean
    b.upload(*gpu[:2])
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim))))
    got = from_bf16(run_attend(gpu, pkg, b, q, n_q, window, n_sink))
    want, bound = attend(b, q, n_q, window, n_sink, rows=rows)
    value = code_values(kind)[bad].tolist() if kind != BF16 else [np.inf, -np.inf, np.nan]
    reached = np.zeros(got.shape, dtype=bool)
    for s, pos in at:
        v = value[s % len(bad)]
        for t, of, p in b.slots():
            if of == s and p >= pos and (not window or pos > p - window or pos < n_sink):
                reached[t, :, 3::17] = True
                assert np.array_equal(got[t, :, 3::17], np.full_like(got[t, :, 3::17], v), equal_nan=True), (t, v)
    assert np.isfinite(got[~reached]).all()
    assert (np.abs(got - want) <= bound)[~reached].all()


@pytest.mark.parametrize("kind", [BF16, E5M2])
@pytest.mark.parametrize("new", [[1], [5], [150]])
def test_scores_that_are_infinite(gpu, pkg, kind, new):
    """A row whose scores are all minus infinity gives 0; an infinite score gives NaN, as in a softmax; a NaN query is alone with it."""
    b = Batch(5, kind, 128, 1, 16, new, [200])
    wild = 0xFF80 if kind == BF16 else 0xFC
    for pos in range(200): b.pool["k"][b.table[0, pos // 16], 0, pos % 16, 0] = wild
    b.upload(*gpu[:2])
    q = np.zeros((b.tokens, 4, 128))
    q[:, :, 0] = 1.0
    got = run_attend(gpu, pkg, b, q, 4)
    assert not got.any()
    q[0, 1, 0] = -1.0
    q[0, 2, 5] = np.nan
    got = from_bf16(run_attend(gpu, pkg, b, q, 4))
    assert np.isnan(got[0, 1:3]).all() and not got[0, 0].any() and not got[0, 3].any() and not got[1:].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,ctx", [([1, 4], [100, 90]), ([70], [300]), ([1], [2500])])
@pytest.mark.parametrize("wrong", [-1, 10 ** 9, -2 ** 31])
def test_pages_outside_the_pool(gpu, pkg, kind, new, ctx, wrong):
    """Their rows are not written, read as 0 and seen by no token; entries behind a sequence's last page are not looked at."""
    torch, dev, lib = gpu
    n_q, n_kv, dim = 4, 2, 64
    b = Batch(sum(ctx) + kind, kind, dim, n_kv, 16, new, ctx)
    rows = {name: [b.rows(name, s) for s in range(b.n_seqs)] for name in ("k", "v")}
    lost = [np.zeros(c, dtype=bool) for c in ctx]
    right = b.table.copy()
    for s in range(b.n_seqs):
        pages = -(-ctx[s] // 16)
        b.table[s, pages:] = wrong
        for page in {1, pages // 2, pages - 1}:
            b.table[s, page] = wrong
            lost[s][16 * page:16 * page + 16] = True
    b.upload(torch, dev)
    out = torch.full((2, b.tokens, n_kv, dim), 0x1234, dtype=torch.int16, device=dev)
    assert lib.kv_paged_read(b.descriptor(pkg), ptr(out[0]), ptr(out[1]), b.tokens, n_kv * dim, dim) == 0
    back = from_bf16(out.cpu().numpy().view(np.uint16))
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim))))
    got = from_bf16(run_attend(gpu, pkg, b, q, n_q))
    for t, s, pos in b.slots():
        for i, name in enumerate(("k", "v")): assert np.array_equal(back[i, t], np.zeros((n_kv, dim)) if lost[s][pos] else rows[name][s][:, pos])
    # the same rows with their keys' scores at minus infinity
    for s in range(b.n_seqs):
        for t, of, pos in b.slots():
            if of != s: continue
            seen = ~lost[s][:pos + 1]
            for h in range(n_q):
                k, v = rows["k"][s][h // 2, :pos + 1][seen], rows["v"][s][h // 2, :pos + 1][seen]
                if not seen.any():
                    assert not got[t, h].any()
                    continue
                w = np.exp(k @ q[t, h] / 8.0 - (k @ q[t, h] / 8.0).max())
                y = (w / w.sum()) @ v
                assert (np.abs(got[t, h] - y) <= 2.0 ** -7 * (w / w.sum()) @ np.abs(v) + 2.0 ** -8 * np.abs(y)).all()      # a probability's and the result's rounding, 2^-8 each, and room for FP32
    before = {n: b.download(n).copy() for n in ("k", "v")}
    run_append(gpu, pkg, b, n_q, True, True)
    touched = np.zeros((b.n_pages, 16), dtype=bool)
    for t, s, pos in b.slots():
        if not lost[s][pos]: touched[right[s, pos // 16], pos % 16] = True
    for n in ("k", "v"):
        after = b.download(n)
        assert np.array_equal(after[~touched[:, None, :].repeat(n_kv, 1)], before[n][~touched[:, None, :].repeat(n_kv, 1)])
        assert (after != before[n]).any() == touched.any()


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_lengths_that_are_not_right(gpu, pkg, kind):
    """More new tokens than rows: those at negative positions give 0, are not written and read as 0.  Lengths beyond the table or max_ctx are cut, negative ones are 0.  A sequence with more new
    tokens than max_new is left out, ranges that are not in order name nobody or stay within what they name."""
    torch, dev, lib = gpu
    n_q, dim = 4, 64
    b = Batch(7, kind, dim, 1, 16, [4, 30, 2, 1], [2, 20, 64, 5]).upload(torch, dev)
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim))))
    check_attend(gpu, pkg, b, n_q, q=q)
    out = torch.full((2, b.tokens, dim), 0x1234, dtype=torch.int16, device=dev)
    assert lib.kv_paged_read(b.descriptor(pkg), ptr(out[0]), ptr(out[1]), b.tokens, dim, dim) == 0
    assert not out[:, :2].any() and not out[:, 4:14].any() and (out != 0x1234).all()
    before = b.download("k").copy()
    *_, q_out, _ = run_append(gpu, pkg, b, n_q, False, True)
    assert (q_out.reshape(-1, n_q, dim)[:2] == 0x1234).all() and (q_out.reshape(-1, n_q, dim)[4:14] == 0x1234).all()
    touched = np.zeros((b.n_pages, 16), dtype=bool)
    for t, s, pos in b.slots(): touched[b.table[s, pos // 16], pos % 16] = True
    assert np.array_equal(b.download("k")[~touched[:, None]], before[~touched[:, None]])

    b = Batch(8, kind, dim, 1, 16, [1, 20], [90, 100], table_extra=0).upload(torch, dev)
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim))))
    want = run_attend(gpu, pkg, b, q, n_q)
    capacity = b.table_stride * 16                                  # 112: the second sequence's last page is not full
    for lengths, cut in (([90, 2 ** 31 - 1], [90, capacity]), ([-5, -2 ** 31], [0, 0])):
        b.dev["ctx_len"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        got = run_attend(gpu, pkg, b, q, n_q, max_ctx=2 ** 31 - 1)
        b.ctx = cut
        ref, bound = attend(b, q, n_q)
        assert (np.abs(from_bf16(got) - ref) <= bound).all()
    assert not got.any()
    b.ctx, b.dev["ctx_len"] = [90, 64], torch.tensor([90, 100], dtype=torch.int32, device=dev)
    got = run_attend(gpu, pkg, b, q, n_q, max_ctx=64)
    b.ctx = [64, 64]
    ref, bound = attend(b, q, n_q)
    assert (np.abs(from_bf16(got) - ref) <= bound).all()
    b.ctx, b.dev["ctx_len"] = [90, 100], torch.tensor([90, 100], dtype=torch.int32, device=dev)
    got = run_attend(gpu, pkg, b, q, n_q, max_new=19, max_ctx=100)
    assert np.array_equal(got[0], want[0]) and (got[1:] == 0x1234).all()
    for starts in ([5, 1, 0], [-7, 3, 2], [21, 21, 21], [2 ** 31 - 1, -2 ** 31, 4], [0, 2 ** 31 - 1, 2 ** 31 - 1]):
        b.dev["seq_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        run_attend(gpu, pkg, b, q, n_q, max_new=64, max_ctx=100)
        assert lib.kv_paged_read(b.descriptor(pkg), ptr(out[0]), ptr(out[1]), b.tokens, dim, dim) == 0
        run_append(gpu, pkg, b, n_q, True, True)


CASES = [(128, 4, 1, 16, [1], [4000]), (128, 8, 2, 32, [1, 1, 3], [3000, 100, 900]), (64, 8, 8, 64, [100], [3000]), (128, 4, 2, 16, [1, 40, 1], [2000, 1500, 30])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,page,new,ctx", CASES)
def test_workspaces(gpu, pkg, kind, dim, n_q, n_kv, page, new, ctx):
    """Without a workspace, with one of another call's sums or of any bytes: within the formula's bound, and the same bits whatever lay in it."""
    torch, dev, lib = gpu
    b = Batch(sum(ctx) + kind, kind, dim, n_kv, page, new, ctx).upload(torch, dev)
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim))))
    with_parts = check_attend(gpu, pkg, b, n_q, q=q)
    check_attend(gpu, pkg, b, n_q, q=q, workspace=False)
    cache = b.descriptor(pkg)
    args = (n_q, b.tokens, max(new), max(ctx))
    need = lib.attention_paged_workspace_bytes(cache, *args)
    assert need > 0
    qd = put(torch, dev, to_bf16(q))
    for fill in (0, 0x7F, 0xFF, "again", "other", "short"):
        if isinstance(fill, int): ws = torch.full((need,), fill, dtype=torch.uint8, device=dev)
        if fill == "other": assert lib.attention_paged(cache, ptr(qd), ptr(torch.empty_like(qd)), ptr(ws), need, n_q, b.tokens, max(new), max(ctx), 200, 3, n_q * dim, n_q * dim) == 0
        y = torch.zeros(b.tokens, n_q * dim, dtype=torch.int16, device=dev)
        assert lib.attention_paged(cache, ptr(qd), ptr(y), ptr(ws), need // 2 & ~15 if fill == "short" else need, n_q, b.tokens, max(new), max(ctx), 0, 0, n_q * dim, n_q * dim) == 0
        got = from_bf16(y.cpu().numpy().view(np.uint16)).reshape(with_parts.shape)
        if fill == "short":
            want, bound = attend(b, q, n_q)
            assert (np.abs(got - want) <= bound).all()
        else: assert np.array_equal(got, with_parts), fill


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_a_captured_step_with_other_lengths(gpu, pkg, kind):
    """Append, attention and read back captured once and replayed with other lengths and pages, on a stream of its own, eager calls on another workspace between: the bits of eager calls."""
    torch, dev, lib = gpu
    n_q, n_kv, dim, page = 8, 2, 128, 16
    b = Batch(3, kind, dim, n_kv, page, [1, 1, 20], [1500, 40, 700], table_extra=40).upload(torch, dev)
    tokens, most, ld = 24, 1600, (n_q + 2 * n_kv) * dim
    x = put(torch, dev, to_bf16(b.rng.standard_normal((tokens, ld))))
    angle = np.arange(most)[:, None] * 1e4 ** (-np.arange(dim // 2) / (dim // 2))
    cos, sin = put(torch, dev, to_bf16(np.cos(angle))), put(torch, dev, to_bf16(np.sin(angle)))
    q_out, y, back = torch.zeros(tokens, n_q * dim, dtype=torch.int16, device=dev), torch.zeros(tokens, n_q * dim, dtype=torch.int16, device=dev), torch.zeros(2, tokens, n_kv, dim, dtype=torch.int16, device=dev)
    cache = b.descriptor(pkg)
    need = lib.attention_paged_workspace_bytes(cache, n_q, tokens, tokens, most)
    spaces = [torch.full((need,), 0x55, dtype=torch.uint8, device=dev) for _ in range(2)]

    def step(ws):
        at = x.data_ptr()
        assert lib.qk_norm_rope_kv_paged(cache, at, at + 2 * n_q * dim, at + 2 * (n_q + n_kv) * dim, None, None, ptr(cos), ptr(sin), most, ptr(q_out), n_q, tokens, ld, ld, ld) == 0
        assert lib.attention_paged(cache, ptr(q_out), ptr(y), ptr(ws), need, n_q, tokens, tokens, most, 0, 0, n_q * dim, n_q * dim) == 0
        assert lib.kv_paged_read(cache, ptr(back[0]), ptr(back[1]), tokens, n_kv * dim, dim) == 0

    stream = torch.cuda.Stream(device=dev)
    lib.set_sync(False)
    try:
        lib.set_stream(stream.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream): step(spaces[0])
        for lengths, starts in (([1500, 40, 700], [0, 1, 2, 22]), ([1501, 41, 720], [0, 1, 2, 22]), ([17, 1300, 60], [0, 0, 19, 21]), ([1502, 42, 721], [0, 1, 2, 3]), ([0, 0, 0], [0, 0, 0, 0])):
            b.dev["ctx_len"].copy_(torch.tensor(lengths, dtype=torch.int32))
            b.dev["seq_start"].copy_(torch.tensor(starts, dtype=torch.int32))
            for t in (y, back): t.fill_(0x1234)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream): graph.replay()
            torch.cuda.synchronize()
            replayed = [t.clone() for t in (y, back, b.dev["k"], b.dev["v"])]
            for t in (y, back): t.fill_(0x1234)
            torch.cuda.synchronize()
            step(spaces[1])
            torch.cuda.synchronize()
            for a, c in zip(replayed, (y, back, b.dev["k"], b.dev["v"])): assert torch.equal(a, c), lengths
            assert (y[starts[-1]:] == 0x1234).all() and (back[:, starts[-1]:] == 0x1234).all()
    finally:
        lib.set_stream(None)
        lib.set_sync(True)


@pytest.mark.parametrize("kind", KINDS)
def test_offsets_beyond_32_bits_and_strides_of_pages(gpu, pkg, kind):
    """A pool of which a page lies every 96 MiB (its other layers between), 6 GiB in all, and exponents likewise."""
    torch, dev, lib = gpu
    n_q, n_kv, dim, page, stride, scale_stride = 4, 2, 64, 32, 96 << 20, 80 << 20
    b = Batch(2, kind, dim, n_kv, page, [1, 70], [900, 1000], spare=4)
    assert b.n_pages * stride > 5 << 30
    size = n_kv * page * dim * (2 if kind == BF16 else 1)
    full = {}
    b.upload(torch, dev)
    for name in ("k", "v"):
        full[name] = torch.zeros((b.n_pages - 1) * stride + size, dtype=torch.uint8, device=dev)
        for i in range(b.n_pages): full[name][i * stride:i * stride + size] = b.dev[name][i].reshape(-1).view(torch.uint8)
        if kind != BF16:
            full[name + "_scale"] = torch.zeros((b.n_pages - 1) * scale_stride + n_kv * page, dtype=torch.uint8, device=dev)
            for i in range(b.n_pages): full[name + "_scale"][i * scale_stride:i * scale_stride + n_kv * page] = b.dev[name + "_scale"][i].reshape(-1)
    other = dict(page_stride=stride, k=ptr(full["k"]), v=ptr(full["v"]))
    if kind != BF16: other |= dict(scale_stride=scale_stride, k_scale=ptr(full["k_scale"]), v_scale=ptr(full["v_scale"]))
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim))))
    assert np.array_equal(run_attend(gpu, pkg, b, q, n_q, **other), run_attend(gpu, pkg, b, q, n_q))
    out = torch.zeros(2, 2, b.tokens, n_kv, dim, dtype=torch.int16, device=dev)
    for i, cache in enumerate((b.descriptor(pkg), b.descriptor(pkg, **other))): assert lib.kv_paged_read(cache, ptr(out[i, 0]), ptr(out[i, 1]), b.tokens, n_kv * dim, dim) == 0
    assert torch.equal(out[0], out[1])
    *_, call = run_append(gpu, pkg, b, n_q, True, True, **other)
    for i in range(b.n_pages):
        b.dev["k"][i].view(torch.uint8).copy_(full["k"][i * stride:i * stride + size].view(b.dev["k"][i].view(torch.uint8).shape))
        if kind != BF16: b.dev["k_scale"][i].copy_(full["k_scale"][i * scale_stride:i * scale_stride + n_kv * page].view(n_kv, page))
    got = b.dev["k"].clone()
    call.keep[0].data_ptr()
    assert lib.kv_paged_read(b.descriptor(pkg), ptr(out[0, 0]), ptr(out[0, 1]), b.tokens, n_kv * dim, dim) == 0
    assert lib.kv_paged_read(b.descriptor(pkg, **other), ptr(out[1, 0]), ptr(out[1, 1]), b.tokens, n_kv * dim, dim) == 0
    assert torch.equal(out[0, 0], out[1, 0]) and torch.equal(got, b.dev["k"])


@pytest.mark.parametrize("kind", [BF16, E5M2])
@pytest.mark.parametrize("n_seqs,chunk", [(65, 0), (150, 0), (130, 50)])
def test_many_sequences(gpu, pkg, kind, n_seqs, chunk):
    """More than a wave has lanes, empty ones among them, all with the same first pages."""
    rng = np.random.default_rng(n_seqs)
    new = [int(n) for n in rng.integers(0, 4, n_seqs)]
    if chunk: new[70] = chunk
    ctx = [n + int(c) for n, c in zip(new, rng.integers(0, 90, n_seqs))]
    ctx[64] = 1000
    b = Batch(n_seqs, kind, 64, 2, 16, new, ctx)
    for s in range(n_seqs):
        if ctx[s] - new[s] >= 32: b.table[s, :2] = b.table[64, :2]
    b.upload(*gpu[:2])
    check_attend(gpu, pkg, b, 4)
    torch, dev, lib = gpu
    out = torch.zeros(2, b.tokens, 2, 64, dtype=torch.int16, device=dev)
    assert lib.kv_paged_read(b.descriptor(pkg), ptr(out[0]), ptr(out[1]), b.tokens, 128, 64) == 0
    back, values = from_bf16(out.cpu().numpy().view(np.uint16)), {n: b.values(n) for n in ("k", "v")}
    for t, s, pos in b.slots():
        for i, name in enumerate(("k", "v")): assert np.array_equal(back[i, t], values[name][b.table[s, pos // 16], :, pos % 16])


def test_beside_the_contiguous_cache(gpu, pkg):
    """A BF16 prompt of one sequence, taken in by pieces through the pages, against the entries of the contiguous cache: the same rows up to one rounding between norm, rotation and cache, the
    attention of the same rows within the roundings of either (a score's and a probability's to BF16 there, a probability's here, the result's), and the rows read back into a contiguous cache
    the bytes of the pages."""
    torch, dev, lib = gpu
    n_q, n_kv, dim, T, t_kv = 8, 2, 128, 150, 160
    b = Batch(11, BF16, dim, n_kv, 16, [T], [T]).upload(torch, dev)
    rng = np.random.default_rng(1)
    x = to_bf16(rng.standard_normal((T, n_q + 2 * n_kv, dim)))
    w = [put(torch, dev, to_bf16(1 + 0.2 * rng.standard_normal(dim))) for _ in range(2)]
    angle = np.arange(t_kv)[:, None] * 1e4 ** (-np.arange(64) / 64)
    cos, sin = put(torch, dev, to_bf16(np.cos(angle))), put(torch, dev, to_bf16(np.sin(angle)))
    q, k, v = (put(torch, dev, np.ascontiguousarray(x[:, i:j])) for i, j in ((0, n_q), (n_q, n_q + n_kv), (n_q + n_kv, n_q + 2 * n_kv)))
    ref_q, ref_k, ref_v, ref_y = torch.zeros_like(q), torch.zeros(n_kv, t_kv, dim, dtype=torch.int16, device=dev), torch.zeros(n_kv, t_kv, dim, dtype=torch.int16, device=dev), torch.zeros_like(q)
    assert lib.c.hip_qk_norm_rope_kv_rows_bf16(ptr(q), ptr(k), ptr(v), ptr(w[0]), ptr(w[1]), ptr(cos), ptr(sin), ptr(ref_q), ptr(ref_k), ptr(ref_v), n_q, n_kv, dim, t_kv, T, 0, 1e-6) == 0
    y, mine = torch.zeros_like(q), q.clone()
    for begin, end in ((0, 1), (1, 70), (70, 71), (71, 75), (75, T)):
        b.dev["ctx_len"].fill_(end)
        b.dev["seq_start"].copy_(torch.tensor([0, end - begin], dtype=torch.int32))
        cache, n = b.descriptor(pkg), end - begin
        at = mine[begin:end]
        # the queries are turned where they lie
        assert lib.qk_norm_rope_kv_paged(cache, ptr(at), ptr(k[begin]), ptr(v[begin]), ptr(w[0]), ptr(w[1]), ptr(cos), ptr(sin), t_kv, ptr(at), n_q, n, n_q * dim, n_kv * dim, n_kv * dim) == 0
        need = lib.attention_paged_workspace_bytes(cache, n_q, n, n, T)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        assert lib.attention_paged(cache, ptr(at), ptr(y[begin]), ptr(ws), need, n_q, n, n, T, 0, 0, n_q * dim, n_q * dim) == 0
    f = lambda t: from_bf16(t.cpu().numpy().view(np.uint16))  # noqa: E731
    # there the norm's result is rounded once more, 2^-8 of either half
    assert (np.abs(f(mine) - f(ref_q)) <= 2.0 ** -8 * 3 * np.maximum(np.abs(f(ref_q)), np.abs(np.roll(f(ref_q), 64, -1)) * 2)).mean() > 0.999
    assert np.linalg.norm(f(mine) - f(ref_q)) <= 2.0 ** -8 * np.linalg.norm(f(ref_q))
    b.dev["ctx_len"].fill_(T)
    b.dev["seq_start"].copy_(torch.tensor([0, T], dtype=torch.int32))
    mk, mv = torch.zeros_like(ref_k), torch.zeros_like(ref_v)
    assert lib.kv_paged_read(b.descriptor(pkg), ptr(mk), ptr(mv), T, dim, t_kv * dim) == 0
    assert torch.equal(mv, ref_v) and np.linalg.norm(f(mk) - f(ref_k)) <= 2.0 ** -8 * np.linalg.norm(f(ref_k))
    assert lib.c.hip_attention_prefill_fused_bf16(ptr(mine), ptr(mk), ptr(mv), ptr(ref_y), n_q, n_kv, dim, t_kv, T, 0) == 0
    got, want = f(y), f(ref_y)
    # a score of size s is off by 2^-9 s there; scores here are below 8
    assert np.linalg.norm(got - want) <= (8 * 2.0 ** -9 + 3 * 2.0 ** -8) * np.linalg.norm(want)
    b.pool = {n: b.download(n) for n in ("k", "v")}
    ref, bound = attend(b, f(mine), n_q)
    assert (np.abs(got - ref) <= bound).all()


@pytest.mark.parametrize("n_seqs,kind,long,chunk", [(255, E4M3, 0, 0), (256, BF16, 255, 0), (257, E5M2, 256, 0), (257, BF16, 3, 40), (256, E4M3, 200, 70), (600, E4M3, 599, 0), (700, E5M2, 320, 65)])
def test_hundreds_of_sequences(gpu, pkg, n_seqs, kind, long, chunk):
    """Both sides of the most sequences whose keys are cut into parts, one much longer than the rest; a chunk far down the list; every operator."""
    rng = np.random.default_rng(n_seqs + kind)
    new = [int(n) for n in rng.integers(0, 3, n_seqs)]
    new[long] = 1
    if chunk: new[n_seqs - 9] = chunk
    ctx = [n + int(c) for n, c in zip(new, rng.integers(0, 60, n_seqs))]
    ctx[long] = 1500
    b = Batch(n_seqs, kind, 64, 2, 16, new, ctx).upload(*gpu[:2])
    check_attend(gpu, pkg, b, 4)
    torch, dev, lib = gpu
    out = torch.zeros(2, b.tokens, 2, 64, dtype=torch.int16, device=dev)
    assert lib.kv_paged_read(b.descriptor(pkg), ptr(out[0]), ptr(out[1]), b.tokens, 128, 64) == 0
    back, values = from_bf16(out.cpu().numpy().view(np.uint16)), {n: b.values(n) for n in ("k", "v")}
    for t, s, pos in b.slots():
        for i, name in enumerate(("k", "v")): assert np.array_equal(back[i, t], values[name][b.table[s, pos // 16], :, pos % 16])
    # the rows appended to an empty pool, BF16, no norm and no rotation: what was put in lies at the tokens' places and nothing else changed
    e = Batch(n_seqs, BF16, 64, 2, 16, new, ctx).upload(torch, dev)
    for name in ("k", "v"): e.dev[name].zero_()
    rows = put(torch, dev, to_bf16(rng.standard_normal((e.tokens, 4, 64))))
    assert lib.qk_norm_rope_kv_paged(e.descriptor(pkg), None, ptr(rows), ptr(rows) + 256, None, None, None, None, 0, None, 0, e.tokens, 0, 256, 256) == 0
    got, want = {n: e.dev[n].cpu().numpy() for n in ("k", "v")}, {n: np.zeros_like(e.dev[n].cpu().numpy()) for n in ("k", "v")}
    x = rows.cpu().numpy().reshape(e.tokens, 2, 2, 64)
    for t, s, pos in e.slots():
        for i, name in enumerate(("k", "v")): want[name][e.table[s, pos // 16], :, pos % 16] = x[t, i]
    for name in ("k", "v"): assert np.array_equal(got[name].reshape(want[name].shape), want[name])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
def test_pages_that_are_missing_far_down_a_sequence(gpu, pkg, kind, dim, new):
    """Runs of missing pages around every place where a wave or a tile looks up the next pages of its list (32, 64 and 128 blocks of a wave, 64 of a tile), keys in one piece and in parts."""
    torch, dev, lib = gpu
    ctx, n_q, n_kv = 9000, 2, 1
    b = Batch(dim + kind + new, kind, dim, n_kv, 16, [new], [ctx])
    rows = {name: b.rows(name, 0) for name in ("k", "v")}
    lost = np.zeros(ctx, dtype=bool)
    # the four waves' blocks n of 32 or 64 keys: keys 128 n or 256 n on
    for n in (7, 8, 15, 16, 31, 32, 63):
        for first in (128 * n, 256 * n):
            if first + 256 <= ctx - 100: lost[first:first + 128] = True
    b.table[0, np.flatnonzero(lost[::16])] = -1
    b.upload(torch, dev)
    q = from_bf16(to_bf16(b.rng.standard_normal((new, n_q, dim))))
    dq = put(torch, dev, to_bf16(q))
    need = lib.attention_paged_workspace_bytes(b.descriptor(pkg), n_q, new, new, ctx)
    ws = torch.full((need + 16,), 0x5A, dtype=torch.uint8, device=dev)
    for given in (0, need):
        y = torch.zeros(new, n_q, dim, dtype=torch.int16, device=dev)
        assert lib.attention_paged(b.descriptor(pkg), ptr(dq), ptr(y), ptr(ws) if given else None, given, n_q, new, new, ctx, 0, 0, n_q * dim, n_q * dim) == 0
        got = from_bf16(y.cpu().numpy().view(np.uint16))
        for t in (0, new // 2, new - 1):
            seen = ~lost[:ctx - new + t + 1]
            k, v = rows["k"][0, :len(seen)][seen], rows["v"][0, :len(seen)][seen]
            for h in range(n_q):
                w = np.exp(k @ q[t, h] / np.sqrt(dim) - (k @ q[t, h] / np.sqrt(dim)).max())
                w /= w.sum()
                # a probability's and the result's rounding, 2^-8 each, and room for FP32
                assert (np.abs(got[t, h] - w @ v) <= 2.0 ** -7 * w @ np.abs(v) + 2.0 ** -8 * np.abs(w @ v)).all(), (given, t, h)
