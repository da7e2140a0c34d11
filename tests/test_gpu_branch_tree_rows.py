"""Tree attention beside causal attention with a window, and every sequence of large batches against the formula in 64 bits, with a whole workspace, a part of it and none."""
import numpy as np
import pytest

from branch_util import tree_attend, trees
from paged_util import BF16, E5M2, Batch, from_bf16, to_bf16
from test_gpu_branch_tree import run_tree
from test_gpu_paged import KINDS, run_attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,ctx", [([4], [3000]), ([100], [500]), ([2, 60], [30, 2000]), ([33, 3, 90], [1500, 70, 400])])
@pytest.mark.parametrize("window,n_sink", [(90, 5), (20, 0), (3, 40)])
def test_a_line_with_a_window_is_causal_attention(gpu, pkg, kind, new, ctx, window, n_sink):
    """A token of a line stands where a causal one does, and sees the same rows as long as no new token is outside its window: the first `window` tokens.  Both within the formula's bound."""
    b = Batch(sum(ctx) + kind, kind, 128, 1, 16, new, ctx).upload(*gpu[:2])
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, 4, 128))))
    line = [np.tril(np.ones((n, n), dtype=bool)) for n in new]
    got = from_bf16(run_tree(gpu, pkg, b, q, 4, line, window, n_sink))
    causal = from_bf16(run_attend(gpu, pkg, b, q, 4, window, n_sink))
    _, bound = tree_attend(b, q, 4, line, window, n_sink)
    alike = np.concatenate([np.arange(n) < window for n in new])
    assert (np.abs(got - causal) <= 2 * bound)[alike].all()


@pytest.mark.parametrize("kind", [BF16, E5M2])
@pytest.mark.parametrize("n_seqs,big,n_q,n_kv", [(300, 3, 2, 1), (520, 7, 4, 1), (70, 1, 16, 4), (257, 1, 4, 4)])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (50, 9)])
def test_every_sequence_of_many(gpu, pkg, kind, n_seqs, big, n_q, n_kv, window, n_sink):
    """More sequences than are looked up at once, every `big`-th one in tiles, and more tiles than run at once, lengths far apart."""
    rng = np.random.default_rng(n_seqs + window)
    new = [int(rng.integers(34, 50)) if s % big == 0 else int(rng.integers(0, 5)) for s in range(n_seqs)] if n_seqs != 257 else [int(rng.integers(0, 17)) for _ in range(n_seqs)]
    ctx = [n + int(rng.integers(0, 200)) for n in new]
    ctx[n_seqs // 2], ctx[n_seqs - 1] = new[n_seqs // 2] + 2000, new[n_seqs - 1] + 1100
    b = Batch(n_seqs + kind, kind, 64, n_kv, 16, new, ctx).upload(*gpu[:2])
    seen = trees(rng, new)
    q = from_bf16(to_bf16(rng.standard_normal((b.tokens, n_q, 64))))
    values = {name: b.values(name) for name in ("k", "v")}
    rows = {name: [values[name][b.table[s, np.arange(c) // 16], :, np.arange(c) % 16].transpose(1, 0, 2) for s, c in enumerate(ctx)] for name in ("k", "v")}
    want, bound = tree_attend(b, q, n_q, seen, window, n_sink, rows=rows)
    for part in (1.0, 0.3, 0):
        got = from_bf16(run_tree(gpu, pkg, b, q, n_q, seen, window, n_sink, workspace=part))
        bad = ~(np.abs(got - want) <= bound)
        assert not bad.any(), (part, np.argwhere(bad)[:5], np.abs(got - want)[bad][:5], bound[bad][:5])
