"""Beam selection where the end token is no token of the vocabulary: ended beams then have no continuation that can be, and theirs come last, by beam and token."""
import numpy as np
import pytest

from paged_util import to_bf16
from test_gpu_beam import check

pytestmark = pytest.mark.gpu


# rows whose vocabulary is one chunk of 2048 and of 16384 logits, and several chunks of each size with a last one in part
@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 1000), (3, 1, 600), (2, 2, 600), (1, 4, 2040), (520, 1, 9000), (300, 2, 2500), (200, 1, 9000), (300, 1, 8200), (2, 2, 5000), (1, 1, 7)])
@pytest.mark.parametrize("n_out", [1, 2, 3])
def test_an_end_token_behind_the_vocabulary(gpu, groups, beams, vocab, n_out):
    rng = np.random.default_rng(vocab + beams + n_out)
    x = to_bf16(rng.standard_normal((groups * beams, vocab), dtype=np.float32) * 2)
    score = -15 * rng.random(groups * beams)
    for eos in (vocab, vocab + 3, -(-vocab // 2048) * 2048 - 1, -(-vocab // 16384) * 16384 - 1, 2 ** 31 - 1, -1, -2 ** 31):
        last = np.full(groups * beams, eos)
        check(gpu, x, score, last, eos, groups, beams, n_out)           # all have ended
        last[::2] = 5
        check(gpu, x, score, last, eos, groups, beams, n_out)           # every second one
