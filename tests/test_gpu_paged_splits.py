"""Attention on a paged cache whose keys are split over workgroups -- parts of short sequences, ranges of tiles -- where statistics of a split are not numbers, minus infinity or far
below another's: the answer is that of the keys in one piece."""
import numpy as np
import pytest

from paged_util import BF16, E4M3, E5M2, Batch, attend, from_bf16, to_bf16
from test_gpu_paged import KINDS, ptr, run_attend

pytestmark = pytest.mark.gpu

# one and three tokens of four heads: parts; five and 150: tiles, and with only one sequence of max_new tokens nothing else
NEW = [1, 3, 5, 150]


def split(gpu, pkg, b, n_q, window=0):
    """Bytes for sums of parts or ranges are asked for, so that a call that gets them splits the keys."""
    return gpu[2].attention_paged_workspace_bytes(b.descriptor(pkg), n_q, b.tokens + 1, max(b.new), max(b.ctx), window, 0) > 0


@pytest.mark.parametrize("kind", [BF16, E5M2])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("workspace", [True, False])
def test_scores_that_are_infinite_in_every_split(gpu, pkg, kind, dim, new, workspace):
    """Scores that are all minus infinity give 0, an infinite one and a NaN query give NaN, and the other rows know nothing of it, with and without a workspace."""
    b = Batch(5 + dim, kind, dim, 1, 16, [new], [4000])
    wild = 0xFF80 if kind == BF16 else 0xFC
    pos = np.arange(4000)
    b.pool["k"][b.table[0, pos // 16], 0, pos % 16, 0] = wild
    b.upload(*gpu[:2])
    assert split(gpu, pkg, b, 4)
    q = np.zeros((b.tokens, 4, dim))
    q[:, :, 0] = 1.0
    q[0, 1, 0] = -1.0
    q[0, 2, 5] = np.nan
    q[-1, 3, 7] = np.nan
    got = from_bf16(run_attend(gpu, pkg, b, q, 4, workspace=workspace))
    want = np.zeros(got.shape)
    want[0, 1:3] = want[-1, 3] = np.nan
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("window", [0, 2250])
def test_keys_that_are_not_numbers_in_some_splits(gpu, pkg, kind, dim, new, workspace, window):
    """Rows of keys that are NaN throughout parts and ranges, of one of two kv heads: the tokens that see one of them give NaN in its heads, all else is as the formula."""
    n_q, n_kv, first, last = 4, 2, 1000, 1680 if window else 1800
    b = Batch(dim + kind + new, kind, dim, n_kv, 16, [new], [4000])
    rows = {name: [b.rows(name, 0)] for name in ("k", "v")}
    pos = np.arange(first, last)
    b.pool["k"][b.table[0, pos // 16], 1, pos % 16, 9] = 0x7FC0 if kind == BF16 else 0x7F
    b.upload(*gpu[:2])
    assert split(gpu, pkg, b, n_q, window)
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim))))
    got = from_bf16(run_attend(gpu, pkg, b, q, n_q, window, workspace=workspace))
    want, bound = attend(b, q, n_q, window, rows=rows)
    for t, _, p in b.slots():
        if not window or last - 1 > p - window:
            assert np.isnan(got[t, 2:]).all(), t
        else: assert (np.abs(got[t, 2:] - want[t, 2:]) <= bound[t, 2:]).all(), t
    assert (np.abs(got[:, :2] - want[:, :2]) <= bound[:, :2]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_a_query_that_is_not_a_number_beside_others(gpu, pkg, kind, dim):
    """In a batch of short and long sequences, one of a chunk among them: NaN where the query is, whatever the lengths of the others do to the split."""
    b = Batch(dim + kind, kind, dim, 2, 16, [1, 1, 30, 2], [300, 6000, 2500, 40]).upload(*gpu[:2])
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, 8, dim))))
    want, bound = attend(b, q, 8)
    q[0, 3, 1] = q[1, 5, 2] = q[20, 0, 3] = q[33, 7, 0] = np.nan
    for workspace in (True, False):
        got = from_bf16(run_attend(gpu, pkg, b, q, 8, workspace=workspace))
        odd = np.isnan(q).any(-1)
        assert np.isnan(got[odd]).all() and (np.abs(got - want) <= bound)[~odd].all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 5])
def test_splits_of_which_every_key_is_not_a_number(gpu, pkg, kind, new):
    """The first 64, 128, ... rows of keys are NaN: for some of them whole parts and ranges are, and no key beside them.  Every token sees them."""
    torch, dev, lib = gpu
    n_q, dim, ctx = 4, 128, 2000
    b = Batch(kind + new, kind, dim, 1, 16, [new], [ctx]).upload(torch, dev)
    assert split(gpu, pkg, b, n_q)
    q = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim))))
    assert np.isfinite(from_bf16(run_attend(gpu, pkg, b, q, n_q))).all()
    wild = 0x7FC0 if kind == BF16 else 0x7F
    for upto in range(64, ctx - 64, 64):
        pos = np.arange(upto - 64, upto)
        b.dev["k"][torch.from_numpy(b.table[0, pos // 16]).long(), 0, torch.from_numpy(pos % 16), 9] = wild
        assert np.isnan(from_bf16(run_attend(gpu, pkg, b, q, n_q))).all(), upto


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("first,last", [(1024, 1088), (1024, 1536), (896, 2048)])
def test_values_that_are_infinite_where_weights_vanish(gpu, pkg, kind, dim, new, workspace, first, last):
    """A block, a part or more whose scores lie so far below the rest that their weights are 0 in 32 bits, with values that are infinite or NaN in a few dims: those dims are not finite, whether
    or not the keys are split, and the others are as the formula."""
    n_q, n_kv = 4, 2
    b = Batch(dim + kind + new + first, kind, dim, n_kv, 16, [new], [4000])
    rows = {name: [b.rows(name, 0)] for name in ("k", "v")}
    pos = np.arange(first, last)
    page, row = b.table[0, pos // 16], pos % 16
    # 8 times the key's first element over 8 or 11: a score under -600, all others within some 10
    if kind == BF16: b.pool["k"][page, 1, row, 0] = to_bf16(np.float32(-1024.0))
    else:
        b.pool["k"][page, 1, row] = 0
        b.pool["k"][page, 1, row, 0] = 0xB8 if kind == E4M3 else 0xBC           # -1
        b.scale["k"][page, 1, row] = 127 + 10
    b.pool["v"][page, 1, row, 3::17] = {BF16: 0x7F80, E4M3: 0x7F, E5M2: 0x7C}[kind]
    # the reference: scores of -100 or so, e^-100 of the sum, which the bound does not notice
    rows["k"][0][1, pos] = 0.0
    rows["k"][0][1, pos, 0] = -100.0 * np.sqrt(dim) / 8.0
    b.upload(*gpu[:2])
    assert split(gpu, pkg, b, n_q)
    q = np.zeros((b.tokens, n_q, dim))
    q[:, :, 0] = 8.0
    q[:, :, 1:] = from_bf16(to_bf16(b.rng.standard_normal((b.tokens, n_q, dim - 1)) * 0.25))
    got = from_bf16(run_attend(gpu, pkg, b, q, n_q, workspace=workspace))
    want, bound = attend(b, q, n_q, rows=rows)
    reached = np.zeros(got.shape, dtype=bool)
    reached[:, 2:, 3::17] = True
    assert not np.isfinite(got[reached]).any()
    assert (np.abs(got - want) <= bound)[~reached].all()
