"""Entries for sequences that branch: sizes past what a launch can have, buffers that overlap, calls with nothing to do; all answered before any HIP call."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def setup(pkg):
    raw = np.zeros(1 << 16, dtype=np.uint8)
    return pkg.QuantLibrary(), pkg.capi, (raw.ctypes.data + 63) & ~63, raw


def select(lib, p, groups, beams=1, vocab=8, n_out=1, nb=1 << 40, **other):
    a = dict(logits=p, score=p + 256, last=p + 512, parent=p + 1024, token=p + 2048, out=p + 4096, ws=p + 8192) | other
    return lib.beam_select(a["logits"], 1 << 20, a["score"], a["last"], 3, groups, beams, vocab, n_out, a["parent"], a["token"], a["out"], a["ws"], nb)


def test_beam_groups(setup):
    """A group is a workgroup of 1024 lanes, and a grid has fewer than 2^32 lanes."""
    lib, _, p, raw = setup
    for beams, vocab in ((1, 8), (1, 2048), (2, 100), (3, 100)):
        assert lib.beam_select_workspace_bytes(4194303, beams, vocab, 1) > 0
        for groups in (4194304, 5000000, 16777215 // beams):
            assert lib.beam_select_workspace_bytes(groups, beams, vocab, 1) == 0 and select(lib, p, groups, beams, vocab) == -1, (groups, beams, vocab)
    assert not raw.any()


def test_no_groups(setup):
    """The workspace of no groups is 0 bytes, and its call has nothing to do, whatever the buffers."""
    lib, _, p, raw = setup
    assert lib.beam_select_workspace_bytes(0, 4, 1000, 4) == 0
    nothing = dict(logits=None, score=None, last=None, parent=None, token=None, out=None)
    assert select(lib, p, 0, 4, 1000, 4, ws=None, nb=0) == 0 and select(lib, p, 0, 4, 1000, 4, ws=None, nb=0, **nothing) == 0
    assert select(lib, p, 0, 65, 1000, 4, ws=None, nb=0) == select(lib, p, 0, 4, 0, 4, ws=None, nb=0) == -1
    assert not raw.any()
