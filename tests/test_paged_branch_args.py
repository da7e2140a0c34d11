"""Arguments of the entries for sequences that branch that are refused before any HIP call, and the calls that have nothing to do."""
import numpy as np
import pytest

from test_paged_args import BAD


@pytest.fixture(scope="module")
def setup(pkg):
    lib = pkg.QuantLibrary()
    raw = np.zeros(65536, dtype=np.uint8)
    p = (raw.ctypes.data + 63) & ~63
    good = dict(type=4, head_dim=128, n_kv_heads=2, page_size=16, n_pages=3, k=p, v=p, page_table=p, table_stride=4, ctx_len=p + 64, seq_start=p, n_seqs=2, k_scale=p, v_scale=p)
    return lib, pkg.capi, good, p, raw


def at(lib, cache, p, q=None, k=None, v=None, qw=None, kw=None, cos="p", sin="p", n_pos=8, positions="p", axes=1, stride=1, axis=None, out=None, n_q=4, n=1, ldq=512, ldk=256, ldv=256):
    use = lambda x: p if x == "p" else x  # noqa: E731
    return lib.qk_norm_rope_kv_paged_at(cache, q or p, k or p, v or p, qw, kw, use(cos), use(sin), n_pos, use(positions), axes, stride, use(axis), out or p, n_q, n, ldq, ldk, ldv)


def tree(lib, cache, p, q=None, y=None, seen="p", stride=1, ws=None, nb=0, n_q=4, n=1, new=1, ctx=16, win=0, sink=0, ldq=512, ldy=512):
    return lib.attention_paged_tree(cache, q or p, y or p + 4096, p if seen == "p" else seen, stride, ws, nb, n_q, n, new, ctx, win, sink, ldq, ldy)


def keep(lib, caches, p, n_layers=1, keep="p", n_keep="p", n=1, new=1, out=None):
    use = lambda x: p if x == "p" else x  # noqa: E731
    return lib.kv_paged_keep(caches, n_layers, use(keep), use(n_keep), n, new, out)


def fork(lib, caches, p, n_layers=1, n_out=2, parent="p", rows=None, grow="p", reserved=None, table="t", ctx="t", missing="t", ws="w", nb=4096):
    use = lambda x: {"p": p, "t": p + 8192, "w": p + 16384}.get(x, x)  # noqa: E731
    return lib.kv_paged_fork(caches, n_layers, n_out, use(parent), use(rows), use(grow), reserved, use(table), use(ctx), use(missing), use(ws), nb)


@pytest.mark.parametrize("change", BAD, ids=str)
def test_descriptors(setup, change):
    lib, capi, good, p, raw = setup
    c = capi.make_paged_kv(**(good | change))
    one = capi.paged_layers([c])
    assert lib.attention_paged_tree_workspace_bytes(c, 4, 1, 1, 16) == 0
    assert at(lib, c, p) == tree(lib, c, p) == keep(lib, one, p) == fork(lib, one, p) == -1
    assert lib.kv_paged_fork_workspace_bytes(one, 1, 2) == 0
    assert not raw.any()


def test_append_arguments(setup):
    lib, capi, good, p, raw = setup
    c = capi.make_paged_kv(**good)
    for bad in (dict(cos=None), dict(sin=None), dict(cos=None, sin=None), dict(n_pos=0), dict(positions=None), dict(positions=p + 2), dict(axes=0), dict(axes=5), dict(axes=2, stride=0, n=1), dict(axes=4, n=3, stride=2),
                dict(axis=p + 1), dict(axis=p + 2), dict(q=p + 8), dict(out=p + 4), dict(qw=p), dict(n=-1), dict(n=2 ** 31 - 1), dict(n_q=-1), dict(ldq=504), dict(ldk=248)):
        assert at(lib, c, p, **bad) == -1, bad
    assert at(lib, c, p, n=0) == 0 and at(lib, c, p, n=0, axes=4, stride=0, axis="p") == 0
    assert lib.c.hip_qk_norm_rope_kv_paged_at_bf16(None, p, p, p, None, None, p, p, 8, p, 1, 1, None, p, 4, 1, 512, 256, 256, 1e-6) == -1
    assert not raw.any()


def test_tree_arguments(setup):
    lib, capi, good, p, raw = setup
    c = capi.make_paged_kv(**good)
    for bad in (dict(seen=None), dict(seen=p + 4), dict(stride=0), dict(stride=-1), dict(new=65), dict(new=129, stride=2), dict(new=2 ** 31 - 1, stride=2 ** 17), dict(y=p), dict(q=p + 2), dict(y=p + 8), dict(ws=p + 8, nb=64),
                dict(nb=64), dict(n_q=0), dict(n_q=3), dict(n_q=130), dict(n=-1), dict(new=0), dict(ctx=0), dict(win=-1), dict(sink=-1), dict(ldq=256), dict(ldy=516), dict(n=2 ** 31 - 1)):
        assert tree(lib, c, p, **bad) == -1, bad
    assert lib.c.hip_attention_paged_tree_bf16(None, p, p, p, 1, None, 0, 4, 1, 1, 16, 0, 0, 512, 512) == -1
    assert tree(lib, c, p, n=0) == 0 and not raw.any()


def test_layers_have_to_be_alike(setup):
    lib, capi, good, p, raw = setup
    pair = lambda **change: capi.paged_layers([capi.make_paged_kv(**good), capi.make_paged_kv(**(good | change))])  # noqa: E731
    same = pair(k=p + 128, v=p + 256, k_scale=p + 16, v_scale=p + 32)
    assert lib.kv_paged_fork_workspace_bytes(same, 2, 2) > 0 and keep(lib, same, p, n_layers=2, n=0) == 0
    for change in (dict(type=5), dict(head_dim=64), dict(n_kv_heads=4), dict(page_size=32), dict(n_pages=4), dict(n_seqs=3), dict(table_stride=5), dict(page_stride=8192), dict(scale_stride=64), dict(page_table=p + 4),
                   dict(ctx_len=p + 68), dict(seq_start=p + 4), dict(k=None), dict(v=p + 8)):
        assert keep(lib, pair(**change), p, n_layers=2) == fork(lib, pair(**change), p, n_layers=2) == -1, change
        assert lib.kv_paged_fork_workspace_bytes(pair(**change), 2, 2) == 0
    for n in (0, -1, 65537):
        assert keep(lib, same, p, n_layers=n) == fork(lib, same, p, n_layers=n) == -1
    assert lib.c.hip_kv_paged_keep(None, 1, p, p, 1, 1, None) == -1 and lib.c.hip_kv_paged_fork(None, 1, 1, p, None, p, None, p, p, p, p, 4096) == -1
    assert not raw.any()


def test_keep_arguments(setup):
    lib, capi, good, p, raw = setup
    c = capi.paged_layers([capi.make_paged_kv(**good)])
    for bad in (dict(keep=None), dict(n_keep=None), dict(keep=p + 1), dict(n_keep=p + 2), dict(out=p + 66), dict(out=p + 64), dict(n=-1), dict(new=0), dict(new=-1)):
        assert keep(lib, c, p, **bad) == -1, bad
    assert keep(lib, c, p, n=0) == 0 and not raw.any()


def test_fork_arguments(setup):
    lib, capi, good, p, raw = setup
    c = capi.paged_layers([capi.make_paged_kv(**good)])
    need = lib.kv_paged_fork_workspace_bytes(c, 1, 2)
    assert need > 0
    for bad in (dict(parent=None), dict(grow=None), dict(table=None), dict(ctx=None), dict(missing=None), dict(ws=None), dict(parent=p + 2), dict(rows=p + 1), dict(grow=p + 2), dict(table=p + 8194), dict(ctx=p + 8193),
                dict(missing=p + 8195), dict(ws=p + 16392), dict(nb=need - 1), dict(nb=0), dict(n_out=0), dict(n_out=-1), dict(n_out=65537), dict(table=p), dict(ctx=p + 64)):
        assert fork(lib, c, p, **bad) == -1, bad
    wide = capi.paged_layers([capi.make_paged_kv(**(good | dict(table_stride=2 ** 20)))])
    assert lib.kv_paged_fork_workspace_bytes(wide, 1, 1024) == 0 and fork(lib, wide, p, n_out=1024, nb=1 << 40) == -1
    assert lib.kv_paged_fork_workspace_bytes(wide, 1, 1023) > 0
    assert lib.kv_paged_fork_workspace_bytes(c, 1, 0) == 0
    assert not raw.any()


def test_beam_arguments(setup):
    lib, capi, good, p, raw = setup
    def call(logits=p, ld=104, score=p, last=p + 64, eos=3, groups=1, beams=2, vocab=100, n_out=4, parent=p + 256, token=p + 512, out=p + 768, ws=p + 1024, nb=1 << 20):
        return lib.beam_select(logits, ld, score, last, eos, groups, beams, vocab, n_out, parent, token, out, ws, nb)
    for bad in (dict(logits=None), dict(parent=None), dict(token=None), dict(out=None), dict(ws=None), dict(logits=p + 8), dict(ws=p + 8), dict(score=p + 2), dict(last=p + 1), dict(parent=p + 258), dict(token=p + 513),
                dict(out=p + 770), dict(ld=96), dict(ld=100), dict(groups=-1), dict(beams=0), dict(beams=65), dict(vocab=0), dict(vocab=2 ** 20 + 1, ld=2 ** 21), dict(n_out=0), dict(n_out=129), dict(n_out=201, vocab=100),
                dict(vocab=1, ld=8, n_out=3), dict(out=p), dict(token=p + 64), dict(groups=2 ** 31 - 1)):
        assert call(**bad) == -1, bad
    assert lib.beam_select_workspace_bytes(1, 65, 100, 4) == 0 and lib.beam_select_workspace_bytes(-1, 2, 100, 4) == 0 and lib.beam_select_workspace_bytes(1, 2, 100, 201) == 0
    assert not raw.any()
