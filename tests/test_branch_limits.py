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


N_SEQS, STRIDE, TOKENS, LAYERS = 5, 6, 40, 3
# where each buffer of a call begins, and its bytes
AT = {"page_table": (4096, 4 * N_SEQS * STRIDE), "ctx_len": (8192, 4 * N_SEQS), "seq_start": (12288, 4 * N_SEQS + 4), "keep": (16384, 4 * TOKENS), "n_keep": (20480, 4 * N_SEQS)}


def caches(capi, p):
    one = capi.make_paged_kv(type=4, head_dim=128, n_kv_heads=2, page_size=16, n_pages=9, k=p, v=p, page_table=p + AT["page_table"][0], table_stride=STRIDE, ctx_len=p + AT["ctx_len"][0], seq_start=p + AT["seq_start"][0],
                             n_seqs=N_SEQS, k_scale=p, v_scale=p)
    return capi.paged_layers([one] * LAYERS)


@pytest.mark.parametrize("name", ["page_table", "ctx_len", "seq_start", "keep", "n_keep"])
def test_keep_writes_none_of_what_it_reads(setup, name):
    """All workgroups of all layers read these; the lengths that are left are written by some of them."""
    lib, capi, p, raw = setup
    begin, size = AT[name]
    for out in (begin, begin + 4, begin + size - 4, begin - 4, begin - 4 * N_SEQS + 4):
        assert lib.kv_paged_keep(caches(capi, p), LAYERS, p + AT["keep"][0], p + AT["n_keep"][0], TOKENS, 8, p + out) == -1, out - begin
    assert not raw.any()


N_OUT = 7
FORK = {"page_table": AT["page_table"], "ctx_len": AT["ctx_len"], "parent": (24576, 4 * N_OUT), "rows": (25600, 4 * N_OUT), "grow": (26624, 4 * N_OUT), "reserved": (27648, 9),
        "table_out": (32768, 4 * N_OUT * STRIDE), "ctx_out": (36864, 4 * N_OUT), "missing": (40960, 4), "workspace": (45056, None)}


@pytest.mark.parametrize("written", ["table_out", "ctx_out", "missing", "workspace"])
@pytest.mark.parametrize("name", list(FORK))
def test_fork_writes_none_of_what_it_reads(setup, written, name):
    """The second launch reads parents, rows, growth, lengths and tables anew; what is written lies in buffers of its own."""
    lib, capi, p, raw = setup
    if written == name: return
    c = caches(capi, p)
    need = lib.kv_paged_fork_workspace_bytes(c, LAYERS, N_OUT)
    size = lambda n: FORK[n][1] or need  # noqa: E731
    step = 16 if written == "workspace" else 4
    begin, end = FORK[name][0], FORK[name][0] + size(name)
    for first in {begin, (end - 1) // step * step, (begin - size(written)) // step * step + step}:      # its first byte, its last, what ends in it
        a = {n: p + FORK[n][0] for n in FORK} | {written: p + first}
        assert lib.kv_paged_fork(c, LAYERS, N_OUT, a["parent"], a["rows"], a["grow"], a["reserved"], a["table_out"], a["ctx_out"], a["missing"], a["workspace"], need) == -1, (first - begin)
    assert not raw.any()


def test_fork_arguments(setup):
    """Each argument by itself, all buffers apart."""
    lib, capi, p, raw = setup
    c = caches(capi, p)
    need = lib.kv_paged_fork_workspace_bytes(c, LAYERS, N_OUT)
    def call(n_layers=LAYERS, n_out=N_OUT, nb=need, **other):
        a = {n: p + FORK[n][0] for n in FORK} | other
        return lib.kv_paged_fork(c, n_layers, n_out, a["parent"], a["rows"], a["grow"], a["reserved"], a["table_out"], a["ctx_out"], a["missing"], a["workspace"], nb)
    missing = [{n: None} for n in ("parent", "grow", "table_out", "ctx_out", "missing", "workspace")]
    odd = [{n: p + FORK[n][0] + by} for n in ("parent", "rows", "grow", "table_out", "ctx_out", "missing") for by in (1, 2)] + [dict(workspace=p + FORK["workspace"][0] + by) for by in (4, 8)]
    for bad in missing + odd + [dict(nb=need - 1), dict(nb=0), dict(n_out=0), dict(n_out=-1), dict(n_out=65537, nb=1 << 40), dict(n_layers=0), dict(n_layers=65537)]:
        assert call(**bad) == -1, bad
    assert not raw.any()
