"""Append and read back of so many rows that a workgroup takes several tokens: groups that reach over the ends of sequences, over empty ones, over missing pages, over tokens at negative
positions or past the tables of angles, and the last tokens of a count that the groups do not divide."""
import numpy as np
import pytest

from paged_util import BF16, BITS, LEAST, Batch, from_bf16, norm_rope, quantize, to_bf16
from test_gpu_paged import KINDS, ptr, put, run_append

pytestmark = pytest.mark.gpu

NEW = [5, 0, 2, 65, 0, 1, 129, 30, 3, 27]
CTX = [5, 9, 32, 65, 4, 12, 146, 32, 3, 25]         # the last one has two tokens more than rows
BEHIND = 3                                          # tokens behind the last sequence


def batch(kind, dim, n_kv):
    """Rows 16 .. 31 of sequence 3 and 144 .. 159 of sequence 6 have no page."""
    b = Batch(dim + kind, kind, dim, n_kv, 16, NEW, CTX)
    b.lost = np.zeros((b.n_seqs, 160), dtype=bool)
    for s, page in ((3, 1), (6, 9)):
        b.table[s, page] = -1
        b.lost[s, 16 * page:16 * page + 16] = True
    return b


def several_tokens(torch, heads, dim, tokens):
    """From 32 workgroups per CU on; a workgroup of 256 lanes has 16 or 32 heads."""
    return tokens * -(-heads // (256 * 8 // dim)) >= 32 * torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv", [(128, 512, 5), (128, 3, 254), (64, 1024, 3), (64, 0, 513)])
@pytest.mark.parametrize("norm,rope", [(True, True), (False, False)])
def test_append(gpu, pkg, kind, dim, n_q, n_kv, norm, rope):
    """Tolerances as for few tokens: ten roundings of 2^-24 of the larger half and one to BF16 (2^-8) or the codes (2^-4, 2^-3, half the smallest step); values exactly."""
    torch, dev, lib = gpu
    b = batch(kind, dim, n_kv).upload(torch, dev)
    tokens, n_positions = b.tokens + BEHIND, 140
    assert several_tokens(torch, n_q + 2 * n_kv, dim, tokens)
    before = {n: b.download(n).copy() for n in ("k", "v")}
    scales = {n: None if kind == BF16 else b.download(n + "_scale").copy() for n in ("k", "v")}
    x, w, tab, q_out, _ = run_append(gpu, pkg, b, n_q, norm, rope, pad=8, entry_tokens=tokens, n_positions=n_positions)
    if n_q: q_out = q_out.reshape(tokens + 1, n_q, dim)
    t, s, pos = (np.array(c) for c in zip(*[c for c in b.slots() if not rope or c[2] < n_positions]))
    assert len(t) < b.tokens
    cos, sin = (a[pos][:, None] for a in tab) if rope else (None, None)
    if n_q:
        q = norm_rope(x[t, :n_q], w[0], cos, sin)
        assert (np.abs(from_bf16(q_out[t]) - q) <= 2.0 ** -8 * np.abs(q) + 2.0 ** -19 * np.abs(x[t, :n_q]).max((1, 2), keepdims=True)).all()
        left = np.ones(tokens + 1, dtype=bool)
        left[t] = False
        assert (q_out[left] == 0x1234).all()
    k = norm_rope(x[t, n_q:n_q + n_kv], w[1], cos, sin)
    there = ~b.lost[s, pos]
    assert not there.all()
    page, row = b.table[s, pos // 16][there], pos[there] % 16
    untouched = np.ones((b.n_pages, 16), dtype=bool)
    untouched[page, row] = False
    for name, want, turned in (("k", k[there], norm or rope), ("v", x[t, n_q + n_kv:][there], False)):
        b.pool[name] = b.download(name)
        if kind != BF16: b.scale[name] = b.download(name + "_scale")
        got = b.values(name)[page, :, row]
        if kind == BF16:
            assert (np.abs(got - want) <= (2.0 ** -8 * np.abs(want) + 2.0 ** -20 * np.abs(want).max(-1, keepdims=True) if turned else 0)).all()
        else:
            codes, e = quantize(want, kind)
            step = 2.0 ** e[..., None].astype(np.float64)
            if not turned: assert np.array_equal(got, codes * step)
            # a largest value within FP32's roundings of 1.75 2^k may lie on its other side
            off = b.scale[name][page, :, row].astype(int) - 127 - e
            edge = np.abs(np.abs(want).max(-1) / (2.0 ** (np.where(off < 0, e - 1.0, e) + (8 if BITS[kind] == 3 else 15))) / 1.75 - 1) < 2.0 ** -20
            assert ((off == 0) | (edge & (np.abs(off) == 1) & turned)).all()
            assert (np.abs(got - want) <= 2.0 ** -(BITS[kind] + 1) * np.abs(want) + 2.0 ** (LEAST[kind] - BITS[kind]) * step + 2.0 ** -20 * np.abs(want).max(-1, keepdims=True)).all()
        still = untouched[:, None, :].repeat(n_kv, 1)
        assert np.array_equal(b.pool[name][still], before[name][still])
        if kind != BF16: assert np.array_equal(b.scale[name][still], scales[name][still])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q", [(128, 512), (64, 1024)])
def test_queries_turned_where_they_lie(gpu, pkg, kind, dim, n_q):
    """The bits of a call with another buffer, and tokens that are not named as they were."""
    torch, dev, lib = gpu
    n_kv = 2
    b = batch(kind, dim, n_kv).upload(torch, dev)
    tokens = b.tokens + BEHIND
    assert several_tokens(torch, n_q + 2 * n_kv, dim, tokens)
    q, kv = (put(torch, dev, to_bf16(b.rng.standard_normal((tokens, n, dim)))) for n in (n_q, n_kv))
    angle = np.arange(160)[:, None] * 1e4 ** (-np.arange(dim // 2) / (dim // 2))
    cos, sin = put(torch, dev, to_bf16(np.cos(angle))), put(torch, dev, to_bf16(np.sin(angle)))
    w = put(torch, dev, to_bf16(1 + 0.3 * b.rng.standard_normal(dim)))
    out = torch.full_like(q, 0x1234)
    args = lambda src, dst: (b.descriptor(pkg), ptr(src), ptr(kv), ptr(kv), ptr(w), ptr(w), ptr(cos), ptr(sin), 160, ptr(dst), n_q, tokens, n_q * dim, n_kv * dim, n_kv * dim)  # noqa: E731
    assert lib.qk_norm_rope_kv_paged(*args(q, out)) == 0
    pools = [b.dev[n].clone() for n in ("k", "v")]
    mine = q.clone()
    assert lib.qk_norm_rope_kv_paged(*args(mine, mine)) == 0
    named = torch.zeros(tokens, dtype=torch.bool, device=dev)
    named[[t for t, _, _ in b.slots()]] = True
    assert torch.equal(mine[named], out[named]) and torch.equal(mine[~named], q[~named]) and (out[~named] == 0x1234).all()
    for n, p in zip(("k", "v"), pools): assert torch.equal(b.dev[n], p)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_kv", [(128, 254), (64, 513)])
@pytest.mark.parametrize("contiguous", [False, True])
def test_read(gpu, pkg, kind, dim, n_kv, contiguous):
    """Exactly the values, 0 for rows that are not there, and nothing of a token behind the last sequence."""
    torch, dev, lib = gpu
    b = batch(kind, dim, n_kv).upload(torch, dev)
    tokens = b.tokens + BEHIND
    assert several_tokens(torch, 2 * n_kv, dim, tokens)
    out = torch.full((2, tokens, n_kv, dim), 0x1234, dtype=torch.int16, device=dev)
    strides = (dim, tokens * dim) if contiguous else (n_kv * dim, dim)
    assert lib.kv_paged_read(b.descriptor(pkg), ptr(out[0]), ptr(out[1]), tokens, *strides) == 0
    t, s, pos = (np.array(c) for c in zip(*b.slots()))
    for i, name in enumerate(("k", "v")):
        got = out[i].cpu().numpy().view(np.uint16)
        got = got.reshape(n_kv, tokens, dim).transpose(1, 0, 2) if contiguous else got
        want = np.zeros((b.tokens, n_kv, dim))
        want[t] = np.where(b.lost[s, pos][:, None, None], 0.0, b.values(name)[b.table[s, pos // 16], :, pos % 16])
        assert np.array_equal(from_bf16(got[:b.tokens]), want)
        assert (got[b.tokens:] == 0x1234).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_kv", [(128, 254), (64, 513)])
def test_hundreds_of_sequences(gpu, pkg, kind, dim, n_kv):
    """Groups of which every token is another sequence's, more sequences than a trip to memory tells of, each second one empty: rows appended without norm and rotation come back, BF16 to the
    bit and FP8 as the values of their codes."""
    torch, dev, lib = gpu
    n_seqs = 700
    new = [s % 2 if s % 100 else 2 for s in range(n_seqs)]
    b = Batch(dim + kind, kind, dim, 1, 16, new, [n + s % 3 for s, n in enumerate(new)])
    # (the values of one kv head drawn and every head the same pool: only places matter here)
    b.n_kv = n_kv
    for name in ("k", "v"):
        b.pool[name] = np.zeros((b.n_pages, n_kv, 16, dim), dtype=b.pool[name].dtype)
        if kind != BF16: b.scale[name] = np.zeros((b.n_pages, n_kv, 16), dtype=np.uint8)
    b.upload(torch, dev)
    assert several_tokens(torch, 2 * n_kv, dim, b.tokens)
    x = to_bf16(b.rng.standard_normal((b.tokens, 2, n_kv, dim)))
    xd = put(torch, dev, x)
    assert lib.qk_norm_rope_kv_paged(b.descriptor(pkg), None, ptr(xd), ptr(xd) + 2 * n_kv * dim, None, None, None, None, 0, None, 0, b.tokens, 0, 2 * n_kv * dim, 2 * n_kv * dim) == 0
    out = torch.full((2, b.tokens, n_kv, dim), 0x1234, dtype=torch.int16, device=dev)
    assert lib.kv_paged_read(b.descriptor(pkg), ptr(out[0]), ptr(out[1]), b.tokens, n_kv * dim, dim) == 0
    back, want = from_bf16(out.cpu().numpy().view(np.uint16)), from_bf16(x).transpose(1, 0, 2, 3)
    if kind != BF16:
        codes, e = quantize(want, kind)
        want = codes * 2.0 ** e[..., None].astype(np.float64)
    assert np.array_equal(back, want)
    touched = np.zeros((b.n_pages, 16), dtype=bool)
    for _, s, pos in b.slots(): touched[b.table[s, pos // 16], pos % 16] = True
    for name in ("k", "v"): assert not b.download(name)[~touched[:, None, :].repeat(n_kv, 1)].any()
