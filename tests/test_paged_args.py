"""Arguments of the paged-cache entries that are refused before any HIP call, and the calls that have nothing to do."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def setup(pkg):
    lib = pkg.QuantLibrary()
    raw = np.zeros(4096, dtype=np.uint8)
    p = (raw.ctypes.data + 63) & ~63
    good = dict(type=4, head_dim=128, n_kv_heads=2, page_size=16, n_pages=3, k=p, v=p, page_table=p, table_stride=4, ctx_len=p, seq_start=p, n_seqs=2, k_scale=p, v_scale=p)
    return lib, pkg.capi.make_paged_kv, good, p, raw


BAD = [dict(type=t) for t in (0, 1, 2, 6, 7, -1)] + [dict(head_dim=d) for d in (0, 32, 96, 256)] + [dict(n_kv_heads=n) for n in (0, -1, 1025)] + [dict(page_size=n) for n in (0, 1, 8, 24, 8192, -16)] + \
      [dict(n_pages=0), dict(n_seqs=0), dict(n_seqs=-1), dict(table_stride=0), dict(k=None), dict(v=None), dict(page_table=None), dict(ctx_len=None), dict(seq_start=None), dict(k_scale=None), dict(v_scale=None),
       dict(page_stride=16), dict(page_stride=4096 + 8), dict(scale_stride=16), dict(scale_stride=33)]


@pytest.mark.parametrize("change", BAD, ids=str)
def test_descriptors(setup, change):
    lib, make, good, p, raw = setup
    c = make(**(good | change))
    assert lib.qk_norm_rope_kv_paged(c, p, p, p, None, None, None, None, 0, p, 4, 1, 512, 256, 256) == -1
    assert lib.kv_paged_read(c, p, p, 1, 256, 128) == -1
    assert lib.attention_paged(c, p, p, None, 0, 4, 1, 1, 16, 0, 0, 512, 512) == -1
    assert lib.attention_paged_workspace_bytes(c, 4, 1, 1, 16) == 0
    assert not raw.any()


@pytest.mark.parametrize("name", ["k", "v"])
def test_alignment(setup, name):
    lib, make, good, p, raw = setup
    assert lib.kv_paged_read(make(**(good | {name: p + 8})), p, p, 1, 256, 128) == -1
    for table in ("page_table", "ctx_len", "seq_start"):
        assert lib.kv_paged_read(make(**(good | {table: p + 2})), p, p, 1, 256, 128) == -1


def test_append_arguments(setup):
    lib, make, good, p, raw = setup
    call = lambda cache=make(**good), q=p, k=p, v=p, qw=None, kw=None, cos=None, sin=None, n_pos=0, out=p, n_q=4, n=1, ldq=512, ldk=256, ldv=256: lib.qk_norm_rope_kv_paged(  # noqa: E731
        cache, q, k, v, qw, kw, cos, sin, n_pos, out, n_q, n, ldq, ldk, ldv)
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(qw=p), dict(kw=p), dict(cos=p), dict(sin=p), dict(cos=p, sin=p), dict(n_q=-1), dict(n=-1), dict(ldq=504), dict(ldk=248), dict(ldv=257),
                dict(q=p + 8), dict(k=p + 2), dict(v=p + 4), dict(out=p + 8), dict(n=2 ** 31 - 1)):
        assert call(**bad) == -1, bad
    assert lib.c.hip_qk_norm_rope_kv_paged_bf16(None, p, p, p, None, None, None, None, 0, p, 4, 1, 512, 256, 256, 1e-6) == -1
    assert call(n=0) == 0 and call(n=0, q=None, out=None, n_q=0) == 0
    assert not raw.any()


def test_read_arguments(setup):
    lib, make, good, p, raw = setup
    call = lambda c=make(**good), k=p, v=p, n=1, ts=256, hs=128: lib.kv_paged_read(c, k, v, n, ts, hs)  # noqa: E731
    for bad in (dict(k=None), dict(v=None), dict(k=p + 8), dict(v=p + 2), dict(n=-1), dict(ts=0), dict(ts=120), dict(hs=132), dict(hs=-128)):
        assert call(**bad) == -1, bad
    assert lib.c.hip_kv_paged_read_bf16(None, p, p, 1, 256, 128) == -1
    assert call(n=0) == 0 and not raw.any()


def test_attention_arguments(setup):
    lib, make, good, p, raw = setup
    call = lambda c=make(**good), q=p, y=p, ws=None, nb=0, n_q=4, n=1, new=1, ctx=16, win=0, sink=0, ldq=512, ldy=512: lib.attention_paged(c, q, y, ws, nb, n_q, n, new, ctx, win, sink, ldq, ldy)  # noqa: E731
    for bad in (dict(q=None), dict(y=None), dict(q=p + 2), dict(y=p + 8), dict(ws=p + 8, nb=64), dict(nb=64), dict(n_q=0), dict(n_q=3), dict(n_q=130), dict(n=-1), dict(new=0), dict(ctx=0), dict(win=-1), dict(sink=-1),
                dict(ldq=256), dict(ldy=516), dict(n=2 ** 31 - 1)):
        assert call(**bad) == -1, bad
    assert lib.c.hip_attention_paged_bf16(None, p, p, None, 0, 4, 1, 1, 16, 0, 0, 512, 512) == -1
    assert call(n=0) == 0 and not raw.any()
    assert lib.attention_paged_workspace_bytes(make(**good), 3, 1, 1, 16) == 0


@pytest.mark.parametrize("kind", [4, 5])
@pytest.mark.parametrize("name", ["k_scale", "v_scale"])
def test_alignment_of_exponents(setup, name, kind):
    lib, make, good, p, raw = setup
    for off in (1, 2, 8):
        c = make(**(good | {"type": kind, name: p + off}))
        assert lib.qk_norm_rope_kv_paged(c, p, p, p, None, None, None, None, 0, p, 4, 1, 512, 256, 256) == -1
        assert lib.kv_paged_read(c, p, p, 1, 256, 128) == -1
        assert lib.attention_paged(c, p, p + 1024, None, 0, 4, 1, 1, 16, 0, 0, 512, 512) == -1
        assert lib.attention_paged_workspace_bytes(c, 4, 1, 1, 16) == 0
    # of a BF16 cache they are not looked at
    c = make(**(good | {"type": 3, name: p + 1}))
    assert lib.kv_paged_read(c, p, p, 0, 256, 128) == 0 and lib.attention_paged_workspace_bytes(c, 4, 1, 1, 16) > 0
    assert not raw.any()


def test_results_over_inputs(setup):
    """Queries of a wider projection are not rotated onto themselves, where one row's dense result lies on another's queries; attention does not write over its queries."""
    lib, make, good, p, raw = setup
    c = make(**good)
    assert lib.qk_norm_rope_kv_paged(c, p, p + 1024, p + 1536, None, None, None, None, 0, p, 4, 2, 1024, 1024, 1024) == -1
    assert lib.attention_paged(c, p, p, None, 0, 4, 1, 1, 16, 0, 0, 512, 512) == -1
    assert not raw.any()


def test_most_sequences(setup):
    lib, make, good, p, raw = setup
    assert lib.attention_paged_workspace_bytes(make(**(good | dict(n_seqs=256))), 4, 256, 1, 16) > 0
    for n, status in ((65536, 0), (65537, -1), (2 ** 31 - 1, -1)):
        c = make(**(good | dict(n_seqs=n)))
        assert lib.qk_norm_rope_kv_paged(c, p, p, p, None, None, None, None, 0, p, 4, 0, 512, 256, 256) == status
        assert lib.kv_paged_read(c, p, p, 0, 256, 128) == status
        assert lib.attention_paged(c, p, p, None, 0, 4, 0, 1, 16, 0, 0, 512, 512) == status
    assert not raw.any()
