"""Which rows of the activations and of the pages a call touches for what seq_start says: gaps in front and behind, ranges that begin before the first row or end behind the last one, ranges
that are not in order."""
import numpy as np
import pytest

from paged_util import BF16, E4M3, Batch, attend, from_bf16, norm_rope, to_bf16
from test_gpu_paged import ptr, put

pytestmark = pytest.mark.gpu

FILL = 0x1234
TOKENS, N_Q, DIM = 21, 4, 64
BIG = 2 ** 31 - 1
# ascending: the tokens of each range, whatever part of it lies among the rows; the others: no token that no range holds
STARTS = [[0, 1, 21], [3, 10, 21], [0, 9, 9], [4, 4, 17], [-7, 3, 21], [0, 1, 30], [-3, -1, 5], [21, 21, 21], [-9, -9, -2], [25, 30, 40], [0, BIG, BIG], [5, 1, 0], [-7, 3, 2], [BIG, -BIG - 1, 4], [4, 0, 21], [10, 20, 5], [8, -2, 8]]


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("max_new", [3, 64])
@pytest.mark.parametrize("starts", STARTS, ids=str)
def test_what_a_call_touches(gpu, pkg, kind, max_new, starts):
    torch, dev, lib = gpu
    ctx = [90, 100]
    b = Batch(kind, kind, DIM, 1, 16, [1, 20], ctx).upload(torch, dev)
    b.dev["seq_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    cache = b.descriptor(pkg)
    ascending = starts == sorted(starts)
    # (token, sequence, position, new tokens of the sequence)
    named = [(t, s, ctx[s] - (starts[s + 1] - t), starts[s + 1] - starts[s]) for s in range(2) for t in range(TOKENS) if starts[s] <= t < starts[s + 1]]
    assert len({t for t, *_ in named}) == len(named)

    # attention: sequences of up to max_new new tokens
    q = from_bf16(to_bf16(b.rng.standard_normal((TOKENS, N_Q, DIM))))
    qd = put(torch, dev, to_bf16(q))
    y = torch.full((TOKENS + 1, N_Q, DIM), FILL, dtype=torch.int16, device=dev)
    need = lib.attention_paged_workspace_bytes(cache, N_Q, TOKENS, max_new, 100)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    assert lib.attention_paged(cache, ptr(qd), ptr(y), ptr(ws), need, N_Q, TOKENS, max_new, 100, 0, 0, N_Q * DIM, N_Q * DIM) == 0
    got = y.cpu().numpy().view(np.uint16)
    attended = [(t, s, pos) for t, s, pos, n in named if n <= max_new]
    left = np.ones(TOKENS + 1, dtype=bool)
    left[[t for t, *_ in attended]] = False
    assert (got[left] == FILL).all()
    b.tokens, b.new, slots = TOKENS, [1, 1], [a for a in attended if a[2] >= 0]
    b.slots = lambda: slots
    want, bound = attend(b, q, N_Q)
    for t, *_ in attended:
        if ascending or not (got[t] == FILL).all(): assert (np.abs(from_bf16(got[t]) - want[t]) <= bound[t]).all(), t

    # read back: rows at negative positions are 0
    out = torch.full((2, TOKENS + 1, DIM), FILL, dtype=torch.int16, device=dev)
    assert lib.kv_paged_read(cache, ptr(out[0]), ptr(out[1]), TOKENS, DIM, DIM) == 0
    left = np.ones(TOKENS + 1, dtype=bool)
    left[[t for t, *_ in named]] = False
    for i, name in enumerate(("k", "v")):
        back, values = out[i].cpu().numpy().view(np.uint16), b.values(name)
        assert (back[left] == FILL).all()
        for t, s, pos, _ in named:
            if ascending or not (back[t] == FILL).all(): assert np.array_equal(from_bf16(back[t]), values[b.table[s, pos // 16], 0, pos % 16] if pos >= 0 else np.zeros(DIM)), t

    # append, BF16 inputs that the values' codes hold exactly: a row is as it was or what its token says
    x = np.where(b.rng.random((TOKENS, N_Q + 2, DIM)) < 0.5, -1.0, 1.0) * 2.0 ** b.rng.integers(-3, 4, (TOKENS, N_Q + 2, DIM))
    xd = put(torch, dev, to_bf16(x))
    angle = np.arange(100)[:, None] * 1e4 ** (-np.arange(DIM // 2) / (DIM // 2))
    tab = [to_bf16(np.cos(angle)), to_bf16(np.sin(angle))]
    cos, sin = (put(torch, dev, a) for a in tab)
    q_out = torch.full((TOKENS + 1, N_Q, DIM), FILL, dtype=torch.int16, device=dev)
    before = {n: b.download(n).copy() for n in ("k", "v")}
    ld, at = (N_Q + 2) * DIM, ptr(xd)
    assert lib.qk_norm_rope_kv_paged(cache, at, at + 2 * N_Q * DIM, at + 2 * (N_Q + 1) * DIM, None, None, ptr(cos), ptr(sin), 100, ptr(q_out), N_Q, TOKENS, ld, ld, ld) == 0
    turned = q_out.cpu().numpy().view(np.uint16)
    there = [(t, s, pos) for t, s, pos, _ in named if pos >= 0]
    left = np.ones(TOKENS + 1, dtype=bool)
    left[[t for t, *_ in there]] = False
    assert (turned[left] == FILL).all()
    may = np.zeros((b.n_pages, 16), dtype=bool)
    b.pool = {n: b.download(n) for n in ("k", "v")}
    if kind != BF16: b.scale = {n: b.download(n + "_scale") for n in ("k", "v")}
    v = b.values("v")
    for t, s, pos in there:
        page, row = b.table[s, pos // 16], pos % 16
        may[page, row] = True
        if not ascending and (turned[t] == FILL).all():
            for n in ("k", "v"): assert np.array_equal(b.pool[n][page, :, row], before[n][page, :, row])
            continue
        angles = [from_bf16(a)[pos] for a in tab]
        want = norm_rope(x[t, :N_Q], None, *angles)
        # FP32 and one rounding to BF16
        assert (np.abs(from_bf16(turned[t]) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -20 * np.abs(x[t, :N_Q]).max()).all()
        assert np.array_equal(v[page, 0, row], x[t, N_Q + 1])
    for n in ("k", "v"): assert np.array_equal(b.pool[n][~may[:, None]], before[n][~may[:, None]])
