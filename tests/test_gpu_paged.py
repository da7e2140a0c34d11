"""Operators on a paged cache against their formulas in 64 bits: append of BF16 and FP8 rows with norm and rotation, rows read back, attention of one and more
new tokens per sequence with and without a window."""
import numpy as np
import pytest

from paged_util import BF16, BITS, E4M3, E5M2, LEAST, Batch, attend, code_values, from_bf16, norm_rope, quantize, to_bf16

pytestmark = pytest.mark.gpu

KINDS = [BF16, E4M3, E5M2]


def ptr(t):
    return None if t is None else t.data_ptr()


def put(torch, dev, a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int16)).to(dev)


def run_append(gpu, pkg, b, n_q, norm, rope, pad=0, entry_tokens=None, n_positions=None, **other):
    """q, k and v side by side in rows that are `pad` elements longer.  Returns the inputs and q_out (a row more than there are tokens)."""
    torch, dev, lib = gpu
    rng, dim = b.rng, b.dim
    tokens = entry_tokens or b.tokens
    heads = n_q + 2 * b.n_kv
    x = to_bf16(rng.standard_normal((tokens, heads, dim)) * 1.5)
    ld = heads * dim + pad
    qkv = np.zeros((tokens, ld), dtype=np.uint16)
    qkv[:, :heads * dim] = x.reshape(tokens, -1)
    w = [to_bf16(1 + 0.3 * rng.standard_normal(dim)) if norm else None for _ in range(2)]
    n_positions = n_positions or max(b.ctx)
    angle = np.arange(n_positions)[:, None] * 1e4 ** (-np.arange(dim // 2) / (dim // 2))
    tab = [to_bf16(np.cos(angle)), to_bf16(np.sin(angle))] if rope else [None, None]
    xd = put(torch, dev, qkv)
    q_out = torch.full(((tokens + 1) * max(n_q, 1) * dim,), 0x1234, dtype=torch.int16, device=dev)
    wd, td = ([None if a is None else put(torch, dev, a) for a in v] for v in (w, tab))
    at = xd.data_ptr()
    call = lambda: lib.qk_norm_rope_kv_paged(b.descriptor(pkg, **other), at if n_q else None, at + 2 * n_q * dim, at + 2 * (n_q + b.n_kv) * dim, ptr(wd[0]), ptr(wd[1]), ptr(td[0]), ptr(td[1]),
                                             n_positions, ptr(q_out) if n_q else None, n_q, tokens, ld, ld, ld)
    call.keep = (xd, wd, td)
    assert call() == 0
    torch.cuda.synchronize()
    f = lambda a: None if a is None else from_bf16(a)  # noqa: E731
    return from_bf16(x), [f(a) for a in w], [f(a) for a in tab], q_out.cpu().numpy().view(np.uint16), call


SHAPES = [  # dim, n_q, n_kv, page, new, ctx
    (128, 4, 1, 16, [1], [1]), (128, 8, 2, 16, [1, 0, 3], [17, 40, 3]), (64, 3, 3, 32, [33, 1, 5], [40, 64, 100]), (128, 32, 8, 64, [65, 2], [65, 130]), (64, 10, 2, 128, [7, 0, 0, 130], [300, 0, 9, 131]),
    (64, 0, 4, 16, [5, 4], [5, 20])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,page,new,ctx", SHAPES)
@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (False, False)])
def test_append(gpu, pkg, kind, dim, n_q, n_kv, page, new, ctx, norm, rope):
    """Queries: FP32 with some ten roundings of 2^-24 of the larger half, then one to BF16 (2^-8).  Cached rows: those, then one to the codes (2^-4 or 2^-3 of the value,
    half the smallest step next to 0); without norm and rotation, and of the values, exactly.  Nothing else in the pools changes."""
    b = Batch(dim + n_q + sum(new) + kind, kind, dim, n_kv, page, new, ctx).upload(*gpu[:2])
    before = {n: b.download(n).copy() for n in ("k", "v")}
    scales = {n: None if kind == BF16 else b.download(n + "_scale").copy() for n in ("k", "v")}
    x, w, tab, q_out, _ = run_append(gpu, pkg, b, n_q, norm, rope, pad=8)
    touched = np.zeros((b.n_pages, page), dtype=bool)
    got_values = {}
    for n in ("k", "v"):
        b.pool[n] = b.download(n)
        if kind != BF16: b.scale[n] = b.download(n + "_scale")
        got_values[n] = b.values(n)
    for t, s, pos in b.slots():
        cos, sin = (tab[0][pos], tab[1][pos]) if rope else (None, None)
        if n_q:
            q = norm_rope(x[t, :n_q], w[0], cos, sin)
            got = from_bf16(q_out.reshape(-1, n_q, dim)[t])
            assert (np.abs(got - q) <= 2.0 ** -8 * np.abs(q) + 2.0 ** -20 * np.abs(x[t, :n_q]).max() * 2).all(), t
        page_id, row = b.table[s, pos // page], pos % page
        touched[page_id, row] = True
        for name, want, turned in (("k", norm_rope(x[t, n_q:n_q + n_kv], w[1], cos, sin), norm or rope), ("v", x[t, n_q + n_kv:], False)):
            got = got_values[name][page_id, :, row]
            if kind == BF16:
                assert (np.abs(got - want) <= (2.0 ** -8 * np.abs(want) + 2.0 ** -20 * np.abs(want).max() if turned else 0)).all()
                continue
            codes, e = quantize(want, kind)
            assert np.array_equal(b.scale[name][page_id, :, row], (e + 127).astype(np.uint8))
            step = 2.0 ** e[:, None].astype(np.float64)
            if not turned: assert np.array_equal(got, codes * step)
            assert (np.abs(got - want) <= 2.0 ** -(BITS[kind] + 1) * np.abs(want) + 2.0 ** (LEAST[kind] - BITS[kind] - 1) * step + 2.0 ** -20 * np.abs(want).max()).all()
    for n in ("k", "v"):
        keep = ~touched[:, None, :].repeat(n_kv, 1)
        assert np.array_equal(b.pool[n][keep], before[n][keep])
        if kind != BF16: assert np.array_equal(b.scale[n][keep], scales[n][keep])
    assert (q_out[b.tokens * n_q * dim:] == 0x1234).all()


@pytest.mark.parametrize("kind", [E4M3, E5M2])
def test_rows_at_the_edges_of_a_type(gpu, pkg, kind):
    """Rows of zeros, of the smallest and the largest values, with the largest magnitude on either side of 1.75 2^k, with values half way between two codes, infinities and NaN."""
    torch, dev, lib = gpu
    dim, rows = 64, []
    base = np.zeros(dim)
    for first in (0.0, 2.0 ** -133, 2.0 ** -100, 2.0 ** -93, 448.0, 450.0, 1.75, 1.7578125, 57344.0, 3.3895313892515355e38, 1.75 * 2.0 ** 127, 1.7578125 * 2.0 ** 127, 2.0 ** 127, 1.0, -1.9921875):
        row = base.copy()
        row[0] = first
        row[1:21] = np.array([17, 19, 21, 23, 25, 27, 29, 31, -17, -19, 1.0625, 1.1875, 1.3125, 0.0107421875, 0.00927734375, 0.0009765625, 0.0029296875, 2.0 ** -17, -2.0 ** -16, 1.5 * 2.0 ** -16]) * (abs(first) / 64.0 if first else 0)
        rows.append(from_bf16(to_bf16(row)))
    special = rows[-1].copy()
    special[[3, 9, 20]] = np.inf, -np.inf, np.nan
    rows += [special, np.full(dim, np.inf), np.full(dim, np.nan)]
    b = Batch(1, kind, dim, 1, 16, [len(rows)], [len(rows)]).upload(torch, dev)
    x = np.stack(rows)
    xd = put(torch, dev, to_bf16(x))
    assert lib.qk_norm_rope_kv_paged(b.descriptor(pkg), None, ptr(xd), ptr(xd), None, None, None, None, 0, None, 0, len(rows), 0, dim, dim) == 0
    for n in ("k", "v"):
        b.pool[n], b.scale[n] = b.download(n), b.download(n + "_scale")
        codes, e = quantize(x, kind)
        got = b.rows(n, 0)[0]
        pos = np.arange(len(rows))
        assert np.array_equal(b.scale[n][b.table[0, pos // 16], 0, pos % 16], (e + 127).astype(np.uint8))
        with np.errstate(invalid="ignore"): want = codes * 2.0 ** e[:, None].astype(np.float64)
        assert np.array_equal(got, want, equal_nan=True), n
    out = torch.zeros(2, len(rows), dim, dtype=torch.int16, device=dev)
    assert lib.kv_paged_read(b.descriptor(pkg), ptr(out[0]), ptr(out[1]), len(rows), dim, dim) == 0
    back = from_bf16(out.cpu().numpy().view(np.uint16))
    assert np.array_equal(back[0], want, equal_nan=True) and np.array_equal(back[1], want, equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,page,new,ctx", SHAPES)
@pytest.mark.parametrize("contiguous", [False, True])
def test_read(gpu, pkg, kind, dim, n_q, n_kv, page, new, ctx, contiguous):
    """Exactly the values, in rows of a token or as a contiguous cache of each head; a row behind the last token stays."""
    torch, dev, lib = gpu
    b = Batch(dim + n_kv + sum(ctx) + kind, kind, dim, n_kv, page, new, ctx).upload(torch, dev)
    out = torch.full((2, b.tokens + 1, n_kv, dim), 0x1234, dtype=torch.int16, device=dev)
    strides = (dim, (b.tokens + 1) * dim) if contiguous else (n_kv * dim, dim)
    assert lib.kv_paged_read(b.descriptor(pkg), ptr(out[0]), ptr(out[1]), b.tokens + 1, *strides) == 0
    for i, name in enumerate(("k", "v")):
        got = out[i].cpu().numpy().view(np.uint16)
        got = got.reshape(n_kv, b.tokens + 1, dim).transpose(1, 0, 2) if contiguous else got
        values = b.values(name)
        for t, s, pos in b.slots():
            assert np.array_equal(from_bf16(got[t]), values[b.table[s, pos // page], :, pos % page])
        assert (got[b.tokens] == 0x1234).all()


def run_attend(gpu, pkg, b, q, n_q, window=0, n_sink=0, workspace=True, max_new=None, max_ctx=None, pad=0, extra=1, **other):
    """Rows of y (one more than there are tokens, ending as they began)."""
    torch, dev, lib = gpu
    tokens, dim = b.tokens, b.dim
    max_new, max_ctx = max_new or max(b.new), max_ctx or max(b.ctx)
    ld = n_q * dim + pad
    qd = torch.zeros(tokens + extra, ld, dtype=torch.int16, device=dev)
    qd[:tokens, :n_q * dim] = put(torch, dev, to_bf16(q).reshape(tokens, -1))
    y = torch.full((tokens + extra, ld), 0x1234, dtype=torch.int16, device=dev)
    cache = b.descriptor(pkg, **other)
    need = lib.attention_paged_workspace_bytes(cache, n_q, tokens + extra, max_new, max_ctx, window, n_sink)
    ws = torch.full((need + 16,), 0x7F, dtype=torch.uint8, device=dev) if workspace and need else None
    assert lib.attention_paged(cache, ptr(qd), ptr(y), ptr(ws), need if ws is not None else 0, n_q, tokens + extra, max_new, max_ctx, window, n_sink, ld, ld) == 0
    torch.cuda.synchronize()
    if ws is not None: assert (ws[need:] == 0x7F).all()
    out = y.cpu().numpy().view(np.uint16)
    assert (out[tokens:] == 0x1234).all() and (out[:, n_q * dim:] == 0x1234).all()
    return out[:tokens, :n_q * dim].reshape(tokens, n_q, dim)


def check_attend(gpu, pkg, b, n_q, window=0, n_sink=0, q=None, **kw):
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, b.dim)) * 1.3)) if q is None else q
    got = from_bf16(run_attend(gpu, pkg, b, q, n_q, window, n_sink, **kw))
    want, bound = attend(b, q, n_q, window, n_sink)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want)[bad][:5], bound[bad][:5])
    return got


ATTEND = [  # dim, n_q, n_kv, page, new, ctx
    (128, 4, 1, 16, [1], [1]), (128, 4, 1, 16, [1], [65]), (64, 8, 1, 16, [1, 1, 0, 1], [64, 300, 20, 7]), (128, 8, 8, 32, [1, 1], [127, 513]), (128, 3, 1, 64, [5, 2], [33, 129]), (64, 10, 2, 16, [3, 1, 4], [3, 200, 70]),
    (128, 8, 2, 16, [40], [40]), (128, 4, 1, 32, [129], [129]), (64, 4, 2, 64, [65, 1, 30], [65, 400, 90]), (128, 16, 1, 128, [9, 70], [500, 71]), (128, 2, 2, 16, [130, 3], [700, 64]), (64, 64, 1, 16, [1, 5], [90, 1030]),
    (128, 5, 1, 16, [17, 1, 1], [60, 1500, 2])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,page,new,ctx", ATTEND)
@pytest.mark.parametrize("window,n_sink", [(0, 0), (1, 0), (37, 0), (64, 4), (100, 70)])
def test_attention(gpu, pkg, kind, dim, n_q, n_kv, page, new, ctx, window, n_sink):
    b = Batch(dim + n_q + sum(ctx) + kind, kind, dim, n_kv, page, new, ctx).upload(*gpu[:2])
    check_attend(gpu, pkg, b, n_q, window, n_sink, pad=8)
