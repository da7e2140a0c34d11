"""Append to a paged cache with the positions of the rotation given, against the formula in 64 bits and the entry that takes positions from the slots."""
import numpy as np
import pytest

from paged_util import BF16, BITS, E4M3, E5M2, LEAST, Batch, from_bf16, norm_rope, quantize, to_bf16
from test_gpu_paged import KINDS, SHAPES, ptr, put

pytestmark = pytest.mark.gpu


def run_at(gpu, pkg, b, n_q, norm, positions, axis, n_positions, stride=None, pad=8, x=None, fn="at"):
    """positions [axis][token]; axis: a byte per pair or None.  Returns inputs in 64 bits and q_out (a row more than there are tokens)."""
    torch, dev, lib = gpu
    rng, dim, tokens, heads = np.random.default_rng(9), b.dim, b.tokens, n_q + 2 * b.n_kv
    x = to_bf16(rng.standard_normal((tokens, heads, dim)) * 1.5) if x is None else x
    ld = heads * dim + pad
    qkv = np.zeros((tokens, ld), dtype=np.uint16)
    qkv[:, :heads * dim] = x.reshape(tokens, -1)
    w = [to_bf16(1 + 0.3 * rng.standard_normal(dim)) if norm else None for _ in range(2)]
    angle = np.arange(n_positions)[:, None] * 1e4 ** (-np.arange(dim // 2) / (dim // 2))
    tab = [to_bf16(np.cos(angle)), to_bf16(np.sin(angle))]
    xd, wd, td = put(torch, dev, qkv), [None if a is None else put(torch, dev, a) for a in w], [put(torch, dev, a) for a in tab]
    q_out = torch.full(((tokens + 1) * max(n_q, 1) * dim,), 0x1234, dtype=torch.int16, device=dev)
    at = xd.data_ptr()
    qkv_at = (at if n_q else None, at + 2 * n_q * dim, at + 2 * (n_q + b.n_kv) * dim)
    if fn == "at":
        stride = stride or tokens
        pd = torch.full((len(positions), stride), 1 << 30, dtype=torch.int32, device=dev)
        pd[:, :tokens] = torch.from_numpy(np.asarray(positions, dtype=np.int32)).to(dev)
        ad = None if axis is None else torch.from_numpy(np.asarray(axis, dtype=np.uint8)).to(dev)
        assert lib.qk_norm_rope_kv_paged_at(b.descriptor(pkg), *qkv_at, ptr(wd[0]), ptr(wd[1]), ptr(td[0]), ptr(td[1]), n_positions, ptr(pd), len(positions), stride, ptr(ad),
                                            ptr(q_out) if n_q else None, n_q, tokens, ld, ld, ld) == 0
    else:
        assert lib.qk_norm_rope_kv_paged(b.descriptor(pkg), *qkv_at, ptr(wd[0]), ptr(wd[1]), ptr(td[0]), ptr(td[1]), n_positions, ptr(q_out) if n_q else None, n_q, tokens, ld, ld, ld) == 0
    torch.cuda.synchronize()
    f = lambda a: None if a is None else from_bf16(a)  # noqa: E731
    return from_bf16(x), [f(a) for a in w], [f(a) for a in tab], q_out.cpu().numpy().view(np.uint16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,page,new,ctx", SHAPES)
@pytest.mark.parametrize("axes,layout", [(1, None), (1, "some"), (2, "blocks"), (3, "mixed"), (3, "blocks"), (4, "some")])
@pytest.mark.parametrize("norm", [True, False])
def test_append_at(gpu, pkg, kind, dim, n_q, n_kv, page, new, ctx, axes, layout, norm):
    """Queries: FP32 with some ten roundings of 2^-24 of the larger half, then one to BF16 (2^-8).  Cached rows: those, then one to the codes (2^-4 or 2^-3 of the value, half the smallest step next to 0).
    Nothing else in the pools changes."""
    b = Batch(dim + n_q + sum(new) + kind, kind, dim, n_kv, page, new, ctx).upload(*gpu[:2])
    half = dim // 2
    axis = {None: None, "blocks": np.arange(half) * axes // half, "mixed": np.arange(half) % axes, "some": b.rng.choice(list(range(axes)) + [axes, 200, 255], half)}[layout]
    n_positions = 50
    positions = b.rng.integers(0, n_positions, (axes, b.tokens))
    before = {n: b.download(n).copy() for n in ("k", "v")}
    x, w, tab, q_out = run_at(gpu, pkg, b, n_q, norm, positions, axis, n_positions, stride=b.tokens + 3)
    touched, got_values = np.zeros((b.n_pages, page), dtype=bool), {}
    for n in ("k", "v"):
        b.pool[n] = b.download(n)
        if kind != BF16: b.scale[n] = b.download(n + "_scale")
        got_values[n] = b.values(n)
    which = np.zeros(half, dtype=int) if axis is None else np.asarray(axis, dtype=int)
    for t, s, pos in b.slots():
        turned = which < axes
        at = positions[np.where(turned, which, 0), t]
        cos, sin = np.where(turned, tab[0][at, np.arange(half)], 1.0), np.where(turned, tab[1][at, np.arange(half)], 0.0)
        if n_q:
            q = norm_rope(x[t, :n_q], w[0], cos, sin)
            assert (np.abs(from_bf16(q_out.reshape(-1, n_q, dim)[t]) - q) <= 2.0 ** -8 * np.abs(q) + 2.0 ** -20 * np.abs(x[t, :n_q]).max() * 2).all(), t
        page_id, row = b.table[s, pos // page], pos % page
        touched[page_id, row] = True
        for name, want in (("k", norm_rope(x[t, n_q:n_q + n_kv], w[1], cos, sin)), ("v", x[t, n_q + n_kv:])):
            got = got_values[name][page_id, :, row]
            if kind == BF16:
                assert (np.abs(got - want) <= (2.0 ** -8 * np.abs(want) + 2.0 ** -20 * np.abs(want).max() if name == "k" else 0)).all()
                continue
            codes, e = quantize(want, kind)
            step = 2.0 ** e[:, None].astype(np.float64)
            if name == "v": assert np.array_equal(got, codes * step)
            # (a largest magnitude next to a power's limit may get the next one: twice the smallest step)
            assert (np.abs(got - want) <= 2.0 ** -(BITS[kind] + 1) * np.abs(want) + 2.0 ** (LEAST[kind] - BITS[kind]) * step + 2.0 ** -20 * np.abs(want).max()).all()
    for n in ("k", "v"):
        stays = ~touched[:, None, :].repeat(n_kv, 1)
        assert np.array_equal(b.pool[n][stays], before[n][stays])
    assert (q_out[b.tokens * n_q * dim:] == 0x1234).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,n_q,n_kv,page,new,ctx", SHAPES + [(128, 8, 2, 16, [3000, 1], [3000, 40])])
def test_positions_of_the_slots(gpu, pkg, kind, dim, n_q, n_kv, page, new, ctx):
    """The slots' positions, on one axis or the same on three: the bits of the entry without positions."""
    results = []
    for fn, axes in (("slot", 1), ("at", 1), ("at", 3)):
        b = Batch(dim + n_q + sum(new) + kind, kind, dim, n_kv, page, new, ctx).upload(*gpu[:2])
        positions = np.zeros((axes, b.tokens), dtype=int)
        for t, _, pos in b.slots(): positions[:, t] = pos
        *_, q_out = run_at(gpu, pkg, b, n_q, True, positions, np.arange(dim // 2) % 3 if axes == 3 else None, max(ctx), fn=fn)
        results.append([q_out] + [b.download(n) for n in (("k", "v") if kind == BF16 else ("k", "v", "k_scale", "v_scale"))])
    for other in results[1:]:
        assert all(np.array_equal(u, v) for u, v in zip(results[0], other))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,ctx", [([7], [30]), ([1500, 600], [1500, 700])])
def test_positions_outside_the_tables(gpu, pkg, kind, new, ctx):
    """A token with one on any axis, used by a pair or not, is left out: its query and its rows stay as they were."""
    b = Batch(kind, kind, 64, 2, 16, new, ctx).upload(*gpu[:2])
    n_q, n_positions = 4, 20
    positions = b.rng.integers(0, n_positions, (3, b.tokens))
    wrong = {1: (0, -1), 3: (2, n_positions), 4: (1, 2 ** 31 - 1), 6: (0, -2 ** 31), b.tokens - 1: (2, n_positions)}
    for t, (a, value) in wrong.items(): positions[a, t] = value
    before = {n: b.download(n).copy() for n in ("k", "v")}
    *_, q_out = run_at(gpu, pkg, b, n_q, True, positions, np.arange(32) % 2, n_positions)
    out = q_out.reshape(-1, n_q, 64)
    after = {n: b.download(n) for n in ("k", "v")}
    for t, s, pos in b.slots():
        page, row = b.table[s, pos // 16], pos % 16
        same = [(out[t] == 0x1234).all()] + [np.array_equal(after[n][page, :, row], before[n][page, :, row]) for n in ("k", "v")]
        assert all(same) if t in wrong else not any(same), t


def test_pairs_that_are_not_turned_stay(gpu, pkg):
    """Their halves do not meet: an infinity in one leaves the other alone."""
    b = Batch(2, BF16, 64, 1, 16, [2], [2]).upload(*gpu[:2])
    x = to_bf16(np.random.default_rng(1).standard_normal((2, 2, 64)))
    x[:, 0, 32] = 0x7F80
    x[:, 0, 7] = 0xFF80
    run_at(gpu, pkg, b, 0, False, [[3, 4]], np.full(32, 1), 8, x=x)
    b.pool["k"] = b.download("k")
    assert np.array_equal(b.pool["k"][b.table[0, 0], 0, :2], x[:, 0])
