"""Beam selection against totals in 64 bits: sizes, ties, beams that have ended or not begun, logits that are not finite, all in one place, graphs."""
import numpy as np
import pytest

from branch_util import beam
from paged_util import from_bf16, to_bf16
from test_gpu_paged import ptr, put

pytestmark = pytest.mark.gpu


def select(gpu, x, score, last, eos, n_groups, n_beams, n_out, pad=0, in_place=False):
    """x BF16 bits [row][vocab].  (rows, tokens, scores); what lies behind them and behind the workspace stays."""
    torch, dev, lib = gpu
    vocab = x.shape[1]
    ld = -(-vocab // 8) * 8 + pad
    wide = np.full((len(x), ld), 0x7F80, dtype=np.uint16)                   # behind a row: plus infinity
    wide[:, :vocab] = x
    xd = put(torch, dev, wide)
    sd = None if score is None else torch.from_numpy(np.asarray(score, dtype=np.float32)).to(dev)
    ld_ = None if last is None else torch.from_numpy(np.asarray(last, dtype=np.int32)).to(dev)
    n = n_groups * n_out
    parent, token = (torch.full((n + 1,), -7, dtype=torch.int32, device=dev) for _ in range(2))
    out = torch.full((n + 1,), -7.0, device=dev)
    if in_place: token, out = ld_, sd
    need = lib.beam_select_workspace_bytes(n_groups, n_beams, vocab, n_out)
    assert need > 0
    ws = torch.full((need + 16,), 0x7F, dtype=torch.uint8, device=dev)
    assert lib.beam_select(ptr(xd), ld, ptr(sd), ptr(ld_), eos, n_groups, n_beams, vocab, n_out, ptr(parent), ptr(token), ptr(out), ptr(ws), need) == 0
    torch.cuda.synchronize()
    assert (ws[need:] == 0x7F).all() and int(parent[n]) == -7
    if not in_place: assert int(token[n]) == -7 and float(out[n]) == -7.0
    return parent[:n].cpu().numpy().reshape(n_groups, -1), token[:n].cpu().numpy().reshape(n_groups, -1), out[:n].cpu().numpy().reshape(n_groups, -1).astype(np.float64)


def check(gpu, x, score, last, eos, n_groups, n_beams, n_out, **kw):
    """Rows and tokens exactly.  Scores: one rounding to FP32 (2^-24 of it) and the sum's error.  A weight 2^t of the sum, t = d log2 e of an exact difference d, has t's two roundings (2^-24 |t| each, times ln 2
    of the weight: no more than 0.7 * 2 * 2^-24 * 2^t |t|, and what is added up of 2^t |t| is no more than log2(vocab) times the sum) and two units of 2^-23 from the exponential; a thread's sum has a rounding of
    2^-24 for each of 4 values per 8 logits and one rescaling of 4 per 8 logits, 64 at most: 2^-24 (2 * 20 + 4 + 32 + 32 + 4) in all."""
    rows, tokens, totals = select(gpu, x, score, last, eos, n_groups, n_beams, n_out, **kw)
    s = np.zeros(len(x)) if score is None else np.asarray(score, dtype=np.float32).astype(np.float64)
    ended = np.zeros(len(x), dtype=bool) if last is None else np.asarray(last) == eos
    want_rows, want_tokens, want = beam(from_bf16(x), s, ended, eos, n_groups, n_beams, n_out)
    assert np.array_equal(rows, want_rows) and np.array_equal(tokens, want_tokens), (np.argwhere((rows != want_rows) | (tokens != want_tokens))[:5], rows, want_rows, tokens, want_tokens)
    finite = np.isfinite(want)
    assert np.array_equal(np.isfinite(totals), finite) and (totals[~finite] == -np.inf).all()
    assert (np.abs(totals[finite] - want[finite]) <= 2.0 ** -24 * np.abs(want[finite]) + 112 * 2.0 ** -24).all()
    return rows, tokens, totals


SIZES = [  # groups, beams, vocab, n_out
    (1, 1, 1, 1), (1, 1, 7, 7), (1, 4, 151936, 4), (3, 2, 1000, 2), (2, 8, 32000, 16), (16, 8, 12003, 8), (1, 64, 5000, 128), (2, 5, 50257, 10), (64, 1, 2049, 1), (1, 3, 2, 6), (5, 4, 4097, 3), (1, 2, 1 << 20, 5), (150, 4, 9000, 8),
    (40, 16, 20000, 32), (1, 64, 2, 128), (1, 16, 300000, 128), (700, 4, 16385, 4)]


@pytest.mark.parametrize("groups,beams,vocab,n_out", SIZES)
@pytest.mark.parametrize("scores", ["given", "none", "first"])
def test_sizes(gpu, groups, beams, vocab, n_out, scores):
    rng = np.random.default_rng(vocab + beams)
    x = to_bf16(rng.standard_normal((groups * beams, vocab), dtype=np.float32) * 3)
    score = {"given": -20 * rng.random(groups * beams), "none": None, "first": np.where(np.arange(groups * beams) % beams == 0, -1.5, -np.inf)}[scores]
    check(gpu, x, score, None, 0, groups, beams, n_out, pad=8 * (beams % 3))


@pytest.mark.parametrize("vocab,n_out", [(5000, 4), (32000, 12), (3000, 128)])
def test_ties(gpu, vocab, n_out):
    """All logits alike, few different ones, beams that are alike, zeros of both signs: the lower beam, then the lower token."""
    rng = np.random.default_rng(vocab)
    beams = 6
    same = np.full((beams, vocab), 0x3F80, dtype=np.uint16)
    check(gpu, same, np.zeros(beams), None, 0, 1, beams, n_out)
    check(gpu, same, -np.arange(beams)[::-1] * 0.25, None, 0, 1, beams, n_out)
    few = to_bf16(rng.integers(-2, 3, (beams, vocab)))
    check(gpu, few, np.zeros(beams), None, 0, 2, 3, n_out)
    alike = np.repeat(to_bf16(rng.standard_normal((1, vocab))), beams, 0)
    check(gpu, alike, np.full(beams, -3.0), None, 0, 1, beams, n_out)
    zeros = np.where(rng.random((beams, vocab)) < 0.5, 0x8000, 0).astype(np.uint16)
    check(gpu, zeros, np.zeros(beams), None, 0, 1, beams, n_out)


@pytest.mark.parametrize("vocab", [600, 40000])
@pytest.mark.parametrize("beams,n_out", [(4, 4), (4, 8), (8, 60)])
def test_ended_and_not_begun(gpu, vocab, beams, n_out):
    rng = np.random.default_rng(vocab + beams)
    groups = 5
    x = to_bf16(rng.standard_normal((groups * beams, vocab)) * 2)
    for eos in (0, 7, vocab - 1, vocab + 3, -1):
        last = np.where(rng.random(groups * beams) < 0.5, eos, 5)
        last[:beams] = eos                      # a group that has ended altogether
        score = -15 * rng.random(groups * beams)
        score[rng.random(groups * beams) < 0.3] = -np.inf
        score[beams:2 * beams] = -np.inf        # one in which nothing has begun
        score[2 * beams], score[2 * beams + 1] = np.nan, np.inf
        check(gpu, x, score, last, eos, groups, beams, n_out)


@pytest.mark.parametrize("vocab", [900, 70000])
def test_logits_that_are_not_finite(gpu, vocab):
    """Barred tokens, all but a few, all of a row or of a group; NaN as barred; plus infinity, once and several times; the largest and smallest numbers."""
    rng = np.random.default_rng(vocab)
    groups, beams, n_out = 6, 4, 8
    x = to_bf16(rng.standard_normal((groups * beams, vocab)) * 2)
    x[rng.random(x.shape) < 0.5] = 0xFF80
    x[3, 2:] = 0xFF80
    x[4:8] = 0xFF80
    x[8, ::3] = 0x7FC0
    x[9] = 0xFFC1
    x[12, 17] = 0x7F80
    x[13, [5, 9, vocab - 1]] = 0x7F80
    x[16] = 0x0001
    x[17, ::2] = 0x7F7F
    x[18] = 0xFF7F
    check(gpu, x, -5 * rng.random(groups * beams), None, 0, groups, beams, n_out)


@pytest.mark.parametrize("vocab,beams,n_out", [(131072, 2, 128), (40000, 8, 64), (300000, 4, 33)])
@pytest.mark.parametrize("place", ["ascending", "descending", "one block", "one thread", "all but one place"])
def test_the_best_in_one_place(gpu, vocab, beams, n_out, place):
    """What a workgroup keeps is its n_out best also where all lie with one thread, or in order."""
    rng = np.random.default_rng(vocab)
    order = np.sort(rng.standard_normal((beams, vocab), dtype=np.float32) * 4, 1)
    if place == "descending": order = order[:, ::-1]
    if place in ("one block", "one thread", "all but one place"):
        x = rng.standard_normal((beams, vocab), dtype=np.float32) * 0.01
        at = np.arange(vocab)
        best = {"one block": (at >= 5000) & (at < 5000 + 3 * n_out), "one thread": at // 8 % 256 == 37, "all but one place": at // 8 % 256 != 37}[place]
        order = np.where(best, x * 100 + 20, x)
    x = to_bf16(order)
    check(gpu, x, -rng.random(beams), None, 0, 1, beams, n_out)
    check(gpu, x, -rng.random(beams), None, 0, beams, 1, n_out)


def test_in_place(gpu):
    rng = np.random.default_rng(3)
    groups, beams, vocab = 9, 4, 5000
    x = to_bf16(rng.standard_normal((groups * beams, vocab)) * 2)
    last = np.where(rng.random(groups * beams) < 0.3, 2, 5)
    check(gpu, x, -9 * rng.random(groups * beams), last, 2, groups, beams, beams, in_place=True)


def test_captured_and_repeated(gpu):
    """Replayed with other logits and scores on a stream of its own, eager calls between; a hundred calls give the same bits."""
    torch, dev, lib = gpu
    groups, beams, vocab, n_out = 4, 5, 33000, 10
    rng = np.random.default_rng(4)
    x, score = torch.zeros(groups * beams, vocab, dtype=torch.int16, device=dev), torch.zeros(groups * beams, device=dev)
    parent, token = (torch.zeros(groups * n_out, dtype=torch.int32, device=dev) for _ in range(2))
    out = torch.zeros(groups * n_out, device=dev)
    need = lib.beam_select_workspace_bytes(groups, beams, vocab, n_out)
    spaces = [torch.full((need,), 0x55, dtype=torch.uint8, device=dev) for _ in range(2)]
    call = lambda ws: lib.beam_select(ptr(x), vocab, ptr(score), None, 0, groups, beams, vocab, n_out, ptr(parent), ptr(token), ptr(out), ptr(ws), need)  # noqa: E731
    stream = torch.cuda.Stream(device=dev)
    lib.set_sync(False)
    try:
        lib.set_stream(stream.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream): assert call(spaces[0]) == 0
        for _ in range(4):
            x.copy_(put(torch, dev, to_bf16(rng.standard_normal((groups * beams, vocab)) * 3)))
            score.copy_(torch.from_numpy(-9 * rng.random(groups * beams).astype(np.float32)))
            torch.cuda.synchronize()
            want = None
            for i in range(30):
                for t in (parent, token, out): t.fill_(-3)
                torch.cuda.synchronize()
                if i % 3 == 0: assert call(spaces[1]) == 0
                else:
                    with torch.cuda.stream(stream): graph.replay()
                torch.cuda.synchronize()
                got = [t.clone() for t in (parent, token, out)]
                want = got if want is None else want
                assert all(torch.equal(u, v) for u, v in zip(got, want)), i
    finally:
        lib.set_stream(None)
        lib.set_sync(True)
