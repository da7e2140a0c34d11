"""The attention half of a layer as a batch is served: quantized linears around the operators of the paged cache, over a prompt, single tokens, drafted tokens and a chunk beside
single tokens, each result of a step against 64 bits from what the step before it left in memory."""
import numpy as np
import pytest
from oracle import synth

from gpu_util import check_rows, from_dev, to_dev
from paged_util import BF16, BITS, E4M3, E5M2, LEAST, Batch, attend, from_bf16, norm_rope, to_bf16
from test_gpu_paged import ptr

pytestmark = pytest.mark.gpu

WIDTH, N_Q, N_KV, DIM, PAGE = 512, 8, 2, 64, 16
STEPS = [[37, 1, 90], [1, 1, 1], [5, 0, 3], [1, 41, 1], [1, 1, 1]]


def weights(oracle, kind, seed, n_out, K):
    """(weight, type number, scale, block scales, the dequantised weight)"""
    if kind == "fp4":
        W, sc = synth.weights_fp4(seed, n_out, K)
        return W, oracle.FP4, 1.0, sc, oracle.dequant_weight(W, oracle.FP4, n_out, K, blk_sc=sc)
    if kind == "e4m3":
        W, inv = synth.weights_e4m3(seed, n_out, K)
        return W, oracle.E4M3, inv, None, oracle.dequant_weight(W, oracle.E4M3, n_out, K, inv)
    W = synth.weights_e5m2(seed, n_out, K)
    return W, oracle.E5M2, 1.0, None, oracle.dequant_weight(W, oracle.E5M2, n_out, K)


@pytest.mark.parametrize("weight,cache_kind", [("e5m2", BF16), ("e4m3", E4M3), ("fp4", E5M2), ("fp4", BF16)])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (40, 4)])
def test_a_batch_over_some_steps(gpu, pkg, oracle, weight, cache_kind, window, n_sink):
    torch, dev, lib = gpu
    total = np.sum(STEPS, 0)
    b = Batch(cache_kind, cache_kind, DIM, N_KV, PAGE, STEPS[0], [int(n) for n in total])
    b.upload(torch, dev)
    heads = N_Q + 2 * N_KV
    linear = {}
    for i, (name, n_out) in enumerate((("qkv", heads * DIM), ("o", WIDTH))):
        W, kind, inv, sc, dense = weights(oracle, weight, synth.seed_for(5, 40 + i), n_out, WIDTH)
        linear[name] = (to_dev(torch, dev, W), kind, inv, None if sc is None else to_dev(torch, dev, sc), n_out, dense)
    w = [to_bf16(1 + 0.2 * b.rng.standard_normal(DIM)) for _ in range(2)]
    angle = np.arange(int(total.max()))[:, None] * 1e4 ** (-np.arange(DIM // 2) / (DIM // 2))
    tab = [to_bf16(np.cos(angle)), to_bf16(np.sin(angle))]
    wd, td = [to_dev(torch, dev, a) for a in w], [to_dev(torch, dev, a) for a in tab]
    ctx = np.zeros(3, dtype=np.int32)
    for step, new in enumerate(STEPS):
        ctx += np.array(new, dtype=np.int32)
        T = sum(new)
        b.new, b.ctx, b.tokens, b.seq_start = list(new), [int(c) for c in ctx], T, np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        b.dev["ctx_len"].copy_(torch.from_numpy(ctx))
        b.dev["seq_start"].copy_(torch.from_numpy(b.seq_start))
        cache = b.descriptor(pkg)
        x = synth.activations(synth.seed_for(6, step), T, WIDTH)
        xd = to_dev(torch, dev, x)
        make = lambda n: torch.zeros(T, n, dtype=torch.int16, device=dev)  # noqa: E731
        qkv, q, y, out = make(heads * DIM), make(N_Q * DIM), make(N_Q * DIM), make(WIDTH)
        before = {n: b.download(n).copy() for n in ("k", "v")}
        need = lib.attention_paged_workspace_bytes(cache, N_Q, T, max(new), int(total.max()), window, n_sink)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        lib.set_sync(False)                     # one behind the other, as they would run
        try:
            W, kind, inv, sc, n_out, _ = linear["qkv"]
            assert lib.linear(ptr(W), kind, ptr(xd), ptr(qkv), n_out, T, WIDTH, inv, ptr(sc)) == 0
            at, ld = ptr(qkv), heads * DIM
            assert lib.qk_norm_rope_kv_paged(cache, at, at + 2 * N_Q * DIM, at + 2 * (N_Q + N_KV) * DIM, ptr(wd[0]), ptr(wd[1]), ptr(td[0]), ptr(td[1]), len(angle), ptr(q), N_Q, T, ld, ld, ld) == 0
            assert lib.attention_paged(cache, ptr(q), ptr(y), ptr(ws), need, N_Q, T, max(new), int(total.max()), window, n_sink, N_Q * DIM, N_Q * DIM) == 0
            W, kind, inv, sc, n_out, _ = linear["o"]
            assert lib.linear(ptr(W), kind, ptr(y), ptr(out), n_out, T, WIDTH, inv, ptr(sc)) == 0
            torch.cuda.synchronize()
        finally:
            lib.set_sync(True)
        got = {name: from_dev(t, np.uint16) for name, t in (("qkv", qkv), ("q", q), ("y", y), ("out", out))}
        check_rows(from_bf16(got["qkv"]), oracle.linear_exact(linear["qkv"][5], x), f"qkv, step {step}")
        rows = from_bf16(got["qkv"]).reshape(T, heads, DIM)
        b.pool = {n: b.download(n) for n in ("k", "v")}
        if cache_kind != BF16: b.scale = {n: b.download(n + "_scale") for n in ("k", "v")}
        values = {n: b.values(n) for n in ("k", "v")}
        touched = np.zeros((b.n_pages, PAGE), dtype=bool)
        for t, s, pos in b.slots():
            page, row = b.table[s, pos // PAGE], pos % PAGE
            touched[page, row] = True
            angles = [from_bf16(a)[pos] for a in tab]
            want = norm_rope(rows[t, :N_Q], from_bf16(w[0]), *angles)
            # FP32 (ten roundings of 2^-24 of the larger half, a norm's size) and one rounding to BF16 or to the codes
            assert (np.abs(from_bf16(got["q"]).reshape(T, N_Q, DIM)[t] - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -19 * np.abs(want).max()).all()
            for n, want in (("k", norm_rope(rows[t, N_Q:N_Q + N_KV], from_bf16(w[1]), *angles)), ("v", rows[t, N_Q + N_KV:])):
                most = np.abs(want).max(-1, keepdims=True)
                half = 2.0 ** -8 if cache_kind == BF16 else 2.0 ** -(BITS[cache_kind] + 1)
                # next to 0 half the smallest step, 2^(least - bits - 1) times the power of two, which is less than 2^(1 - top) of the largest value
                floor = 0.0 if cache_kind == BF16 else most * 2.0 ** (LEAST[cache_kind] - BITS[cache_kind] - {E4M3: 8, E5M2: 15}[cache_kind])
                assert (np.abs(values[n][page, :, row] - want) <= half * np.abs(want) + floor + 2.0 ** -19 * most).all(), (n, t)
        for n in ("k", "v"):
            still = ~touched[:, None].repeat(N_KV, 1)
            assert np.array_equal(b.pool[n][still], before[n][still])
        want, bound = attend(b, from_bf16(got["q"]).reshape(T, N_Q, DIM), N_Q, window, n_sink)
        assert (np.abs(from_bf16(got["y"]).reshape(T, N_Q, DIM) - want) <= bound).all(), step
        check_rows(from_bf16(got["out"]), oracle.linear_exact(linear["o"][5], got["y"]), f"o, step {step}")
