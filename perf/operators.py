"""Operators of a batch of sequences on a paged key / value cache, in plain torch and through this library's entry points.

* append  q/k RMSNorm per head, RoPE and the append of the new tokens' keys and values to the pages of their sequences, held as BF16 or as
          FP8 codes with one power of two per row                                              hip_qk_norm_rope_kv_paged_bf16
* read    rows of the pages back as BF16 rows, one behind the other                             hip_kv_paged_read_bf16
* attend  causal attention of each sequence's new tokens (one, a few, a whole chunk) over its pages, optionally within a window of the
          newest keys and a few first ones                                                      hip_attention_paged_bf16

The batch: sequence s has n_new new tokens, rows seq_start[s] .. seq_start[s + 1] - 1 of the activations, and ctx_len[s] rows in the cache, the
new ones included; row `pos` lies in page page_table[s][pos / page] at row pos % page.  Pages are [kv head][row][dim].

An FP8 row is held as codes c = fp8(x / 2^e), nearest even, with the smallest 2^e >= 2^-100 for which its largest magnitude stays within the
type's largest value (e at most 127 less the type's largest exponent; beyond it codes saturate) and the byte e + 127.

Lengths are those of the case; the values, and where in the pool a sequence's pages lie, come from the seed.
"""
import math

import torch

own = False

#: cache type -> (type number of the library, torch type, exponent and value of the largest number, mantissa bits, exponent of the smallest normal)
CACHES = {"bf16": (3, torch.bfloat16, None, None, None, None),
          "e4m3": (4, torch.float8_e4m3fn, 8, 448.0, 3, -6),
          "e5m2": (5, torch.float8_e5m2, 15, 57344.0, 2, -14)}
EPS = 1e-6

GQA = dict(n_q=32, n_kv=8, dim=128)             # the head layout of the Qwen3-8B and Llama-3.1-8B shapes
SMALL = dict(n_q=16, n_kv=8, dim=64)            # a small model
WIDE = dict(n_q=64, n_kv=8, dim=64)             # eight query heads per kv head


def listed():
    return [
        # one step of sixteen chats: the smallest call, between the projections and the attention of every layer
        dict(name="append_16_seqs_1_token_e4m3", kind="append", cache="e4m3", page=16, seqs=16, chunk=0, new_lo=1, new_hi=1, behind_lo=300, behind_hi=4000, norm=True, **GQA),
        # four prompts of different lengths taken in together
        dict(name="append_4_prompts_e5m2", kind="append", cache="e5m2", page=64, seqs=4, chunk=0, new_lo=1501, new_hi=2600, behind_lo=0, behind_hi=0, norm=False, **GQA),
        # a short conversation of a small model handed over to a contiguous cache
        dict(name="read_301_rows_e5m2", kind="read", cache="e5m2", page=16, seqs=1, chunk=0, new_lo=301, new_hi=301, behind_lo=0, behind_hi=0, **SMALL),
        # long documents read back, the part behind a shared beginning
        dict(name="read_4_documents_e4m3", kind="read", cache="e4m3", page=32, seqs=4, chunk=0, new_lo=5000, new_hi=12000, behind_lo=1000, behind_hi=1000, **GQA),
        # batch-1 decoding at the context the benchmark is quoted on
        dict(name="decode_1_seq_bf16", kind="attend", cache="bf16", page=64, seqs=1, chunk=0, new_lo=1, new_hi=1, behind_lo=4095, behind_hi=4095, window=0, sinks=0, **GQA),
        # a full serving batch, one token each
        dict(name="decode_64_seqs_e4m3", kind="attend", cache="e4m3", page=16, seqs=64, chunk=0, new_lo=1, new_hi=1, behind_lo=1000, behind_hi=8000, window=0, sinks=0, **GQA),
        # long streams that keep a window and the first tokens
        dict(name="decode_16_seqs_window_e4m3", kind="attend", cache="e4m3", page=32, seqs=16, chunk=0, new_lo=1, new_hi=1, behind_lo=16000, behind_hi=32000, window=4096, sinks=4, **GQA),
        # four drafted tokens and one more checked at once
        dict(name="verify_8_seqs_5_tokens_e5m2", kind="attend", cache="e5m2", page=16, seqs=8, chunk=0, new_lo=5, new_hi=5, behind_lo=500, behind_hi=3000, window=0, sinks=0, **WIDE),
        # the next turn of a conversation
        dict(name="chunk_512_behind_3000_bf16", kind="attend", cache="bf16", page=64, seqs=1, chunk=0, new_lo=512, new_hi=512, behind_lo=3000, behind_hi=3000, window=0, sinks=0, **GQA),
        # a piece of a long prompt on an FP8 cache: the largest call
        dict(name="chunk_2048_behind_6000_e4m3", kind="attend", cache="e4m3", page=32, seqs=1, chunk=0, new_lo=2048, new_hi=2048, behind_lo=6000, behind_hi=6000, window=0, sinks=0, **GQA),
        # a piece of one prompt beside the decoding sequences
        dict(name="mixed_24_seqs_e4m3", kind="attend", cache="e4m3", page=16, seqs=24, chunk=509, new_lo=1, new_hi=1, behind_lo=200, behind_hi=4000, window=0, sinks=0, **GQA),
        # prompts of a model whose layers see a window
        dict(name="prompts_4_window_bf16", kind="attend", cache="bf16", page=16, seqs=4, chunk=0, new_lo=1501, new_hi=2600, behind_lo=0, behind_hi=0, window=1024, sinks=4, **GQA),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """More of the same: what a listed case costs at most, and what its plain form can hold."""
    kind = rng.choice(["append", "read", "attend", "attend", "attend", "attend"])
    while True:
        n_kv = rng.choice([1, 2, 4, 8, 8, 8])
        c = dict(kind=kind, cache=rng.choice(sorted(CACHES)), page=rng.choice([16, 16, 32, 64, 128]), n_kv=n_kv, n_q=n_kv * rng.choice([1, 2, 3, 4, 4, 5, 8]), dim=rng.choice([64, 128, 128]), chunk=0)
        seqs = _log(rng, 1, 64)
        if kind == "attend":
            step = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
            window = rng.choice([0, 0, _log(rng, 64, 4096)])
            c |= dict(window=window, sinks=rng.choice([0, 1, 4, 16]) if window else 0)
            behind = _log(rng, 16, 32000)
            c |= dict(seqs=seqs, behind_lo=rng.randint(0, behind), behind_hi=behind)
            if step == "decode":
                c |= dict(new_lo=1, new_hi=1)
            elif step == "verify":
                c |= dict(new_lo=rng.randint(0, 2), new_hi=rng.randint(2, 9))
            elif step == "chunk":
                n = _log(rng, 17, 2048)
                c |= dict(seqs=rng.choice([1, 1, 2, 5]), new_lo=rng.randint(1, n), new_hi=n)
            else:
                c |= dict(chunk=_log(rng, 17, 600), new_lo=1, new_hi=1)
        else:
            n = _log(rng, 1, 4000)
            c |= dict(seqs=seqs, new_lo=rng.randint(0, n), new_hi=n, behind_lo=0, behind_hi=rng.randint(0, 2000))
            if kind == "append":
                c |= dict(norm=rng.random() < 0.5)
        new, ctx = lengths(c)
        w = work(c)
        if sum(new) == 0 or w["bytes"] > 6e8 or w["flops"] > 2.3e11 or sum(ctx) * n_kv * c["dim"] > 4.5e8:
            continue
        if kind == "attend" and c["seqs"] * c["n_q"] * max(new) * max(ctx) > 2.2e9:
            continue
        if c["seqs"] * max(ctx) * n_kv * c["dim"] > 9e8:
            continue
        return c


def lengths(case):
    """New tokens and rows in the cache of each sequence, spread over their ranges."""
    part = [(0.5 + 0.6180339887498949 * s) % 1.0 for s in range(case["seqs"])]
    other = [(0.25 + 0.7548776662466927 * s) % 1.0 for s in range(case["seqs"])]
    new = [case["new_lo"] + int(p * (case["new_hi"] - case["new_lo"] + 1)) for p in part]
    if case["chunk"]:
        new[case["seqs"] // 2] = case["chunk"]
    behind = [case["behind_lo"] + int(p * (case["behind_hi"] - case["behind_lo"] + 1)) for p in other]
    return new, [n + b for n, b in zip(new, behind)]


def work(case):
    new, ctx = lengths(case)
    tokens, n_q, n_kv, dim = sum(new), case["n_q"], case["n_kv"], case["dim"]
    row = 2 * dim if case["cache"] == "bf16" else dim + 1           # bytes of a cached row
    if case["kind"] == "append":
        tables = 2 * 2 * (dim // 2) * min(tokens, max(ctx)) + (4 * dim if case["norm"] else 0)
        heads = n_q + n_kv
        return {"bytes": 2 * dim * tokens * (2 * n_q + 2 * n_kv) + 2 * n_kv * tokens * row + tables, "flops": tokens * heads * dim * (3 + (4 if case["norm"] else 0))}
    if case["kind"] == "read":
        return {"bytes": 2 * n_kv * tokens * (row + 2 * dim), "flops": 2 * n_kv * tokens * dim}
    window, sinks = case["window"], case["sinks"]
    rows = pairs = 0
    for n, c in zip(new, ctx):
        if not n:
            continue
        first = c - n                                               # position of the first new token
        if not window:
            rows += c
            pairs += n * first + n * (n + 1) // 2
            continue
        rows += c if first + 1 <= window + sinks else sinks + window + n - 1
        pairs += sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(first, c))
    return {"bytes": 2 * 2 * dim * n_q * tokens + 2 * n_kv * rows * row, "flops": 4 * dim * n_q * pairs}


# ---------------------------------------------------------------------------------------------------------------- inputs

def _power(e):
    """2^e in 32 bits, e from -126 to 127."""
    return (e.int() + 127 << 23).view(torch.float32)


def _quantized(x, cache):
    """Codes (as bytes) and exponent bytes of rows x, in plain form."""
    _, kind, top, largest, _, _ = CACHES[cache]
    amax = x.abs().amax(-1).float()
    mantissa, exponent = torch.frexp(amax)                          # amax = mantissa 2^exponent, mantissa in [1/2, 1)
    e = exponent - 1 - top + (mantissa * 2 > largest / 2.0 ** top).int()
    e = torch.where(amax > 0, e, torch.full_like(e, -100)).clamp(-100, 127 - top)
    codes = (x.float() * _power(-e)[..., None]).clamp(-largest, largest).to(kind)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    new, ctx = lengths(case)
    seqs, page, n_q, n_kv, dim = case["seqs"], case["page"], case["n_q"], case["n_kv"], case["dim"]
    tokens, most = sum(new), max(ctx)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731

    # a pool whose pages lie in any order, with a few that belong to nobody
    pages = [-(-c // page) for c in ctx]
    n_pages, per_seq = sum(pages) + 5, -(-most // page)
    order = torch.randperm(n_pages, generator=g, device=dev).int()
    first = ints([sum(pages[:s]) for s in range(seqs)])
    at = torch.arange(per_seq, device=dev, dtype=torch.int32)
    table = torch.where(at < ints(pages)[:, None], order[(first[:, None] + at).clamp(max=n_pages - 1)], torch.zeros_like(at)).contiguous()

    # keys have a few strong channels, values are narrower
    gain = 0.5 + 0.5 * torch.rand(n_kv, 1, dim, generator=g, device=dev) + 2.0 * (torch.rand(n_kv, 1, dim, generator=g, device=dev) < 0.03)
    s = dict(case=case, max_new=max(new), max_ctx=most, tokens=tokens, n_pages=n_pages, table=table, ctx_len=ints(ctx), seq_start=ints([sum(new[:i]) for i in range(seqs + 1)]))
    for name, by in (("k", gain), ("v", 0.5)):
        rows = (normal(n_pages, n_kv, page, dim) * by).bfloat16()
        s[name], s[name + "_scale"] = (rows, None) if case["cache"] == "bf16" else _quantized(rows, case["cache"])
        del rows
    if case["kind"] == "append":
        # q, k and v as one projection writes them, side by side
        s["qkv"] = normal(tokens, (n_q + 2 * n_kv) * dim).bfloat16()
        s["q_out"] = torch.empty(tokens, n_q, dim, dtype=torch.bfloat16, device=dev)
        s["norm_w"] = [(1.0 + 0.2 * normal(dim)).bfloat16() if case["norm"] else None for _ in range(2)]
        angle = torch.arange(most, device=dev, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(dim // 2, device=dev, dtype=torch.float64) / (dim // 2))
        s["cos"], s["sin"] = angle.cos().bfloat16(), angle.sin().bfloat16()
    elif case["kind"] == "read":
        s["k_out"], s["v_out"] = (torch.empty(tokens, n_kv, dim, dtype=torch.bfloat16, device=dev) for _ in range(2))
    else:
        s["q"] = (1.3 * normal(tokens, n_q, dim)).bfloat16()
        s["y"] = torch.empty(tokens, n_q, dim, dtype=torch.bfloat16, device=dev)
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms

def _tokens(s):
    """Sequence, index among its new tokens and position of every token."""
    t = torch.arange(s["tokens"], device=s["ctx_len"].device, dtype=torch.int32)
    seq = torch.searchsorted(s["seq_start"][1:].contiguous(), t, right=True)
    index = t - s["seq_start"][seq]
    return seq, index, s["ctx_len"][seq] - (s["seq_start"][seq + 1] - s["seq_start"][seq]) + index


def _slots(s, seq, pos):
    page = s["case"]["page"]
    return s["table"][seq, (pos // page).long()].long(), (pos % page).long()


def _values(s, name, page, row):
    """Cached rows [...][kv head][dim] as 32-bit numbers."""
    x = s[name][page, :, row]
    if s["case"]["cache"] == "bf16":
        return x.float()
    return x.view(CACHES[s["case"]["cache"]][1]).float() * _power(s[name + "_scale"][page, :, row].int() - 127)[..., None]


def _append_plain(s):
    c = s["case"]
    n_q, n_kv, dim = c["n_q"], c["n_kv"], c["dim"]
    seq, _, pos = _tokens(s)
    page, row = _slots(s, seq, pos)
    x = s["qkv"].view(s["tokens"], n_q + 2 * n_kv, dim)
    cos, sin = s["cos"][pos.long()].float()[:, None], s["sin"][pos.long()].float()[:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.float()
        lo, hi = x[..., :dim // 2], x[..., dim // 2:]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    s["q_out"].copy_(turned(x[:, :n_q], s["norm_w"][0]))
    for name, rows in (("k", turned(x[:, n_q:n_q + n_kv], s["norm_w"][1])), ("v", x[:, n_q + n_kv:])):
        if c["cache"] == "bf16":
            s[name][page, :, row] = rows.bfloat16()
        else:
            s[name][page, :, row], s[name + "_scale"][page, :, row] = _quantized(rows, c["cache"])
    return _appended(s)


def _appended(s):
    """The turned queries and the whole pools, FP8 codes and powers of two as the values they stand for."""
    if s["case"]["cache"] == "bf16":
        return s["q_out"], s["k"], s["v"]
    kind = CACHES[s["case"]["cache"]][1]
    return (s["q_out"], s["k"].view(kind), s["v"].view(kind), s["k_scale"].view(torch.float8_e8m0fnu), s["v_scale"].view(torch.float8_e8m0fnu))


def _read_plain(s):
    seq, _, pos = _tokens(s)
    page, row = _slots(s, seq, pos)
    return _values(s, "k", page, row).bfloat16(), _values(s, "v", page, row).bfloat16()


def _attend_plain(s):
    c = s["case"]
    seqs, n_q, n_kv, dim = c["seqs"], c["n_q"], c["n_kv"], c["dim"]
    group = n_q // n_kv
    key = torch.arange(s["max_ctx"], device=s["q"].device, dtype=torch.int32)
    page, row = _slots(s, torch.arange(seqs, device=key.device)[:, None], key.expand(seqs, -1))
    keys = _values(s, "k", page, row).permute(0, 2, 3, 1).contiguous()                 # [seq][kv head][dim][key]
    # each sequence's new tokens, the heads of a kv head side by side: [seq][kv head][token x head][dim]
    new = s["seq_start"][1:] - s["seq_start"][:-1]
    index = torch.arange(s["max_new"], device=key.device, dtype=torch.int32)
    at = (s["seq_start"][:-1, None] + index).clamp(max=s["tokens"] - 1).long()
    q = s["q"][at].float().view(seqs, -1, n_kv, group, dim).transpose(1, 2).reshape(seqs, n_kv, -1, dim)
    score = torch.matmul(q, keys).mul_(1.0 / math.sqrt(dim)).view(seqs, n_kv, -1, group, s["max_ctx"])
    del keys, q
    pos = (s["ctx_len"] - new)[:, None, None] + index[None, :, None]                   # [seq][token][1]
    seen = key <= pos
    if c["window"]:
        seen &= (key > pos - c["window"]) | (key < c["sinks"])
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    score.div_(score.sum(-1, keepdim=True))
    values = _values(s, "v", page, row).permute(0, 2, 1, 3).contiguous()               # [seq][kv head][key][dim]
    y = torch.matmul(score.view(seqs, n_kv, -1, s["max_ctx"]), values).view(seqs, n_kv, -1, group, dim).transpose(1, 2).reshape(seqs, -1, n_q, dim)
    seq, index, _ = _tokens(s)
    return y[seq, index.long()].bfloat16()


# ------------------------------------------------------------------------------------------------- the library's operators

def _bound(s):
    """The call that a user's program keeps: descriptor, workspace and the rest of the arguments."""
    import importlib

    pkg = importlib.import_module("cccc-lite_amd")
    lib, c = pkg.library(), s["case"]
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    cache = pkg.capi.make_paged_kv(CACHES[c["cache"]][0], c["dim"], c["n_kv"], c["page"], s["n_pages"], ptr(s["k"]), ptr(s["v"]), ptr(s["table"]), s["table"].shape[1], ptr(s["ctx_len"]),
                                   ptr(s["seq_start"]), c["seqs"], k_scale=ptr(s["k_scale"]), v_scale=ptr(s["v_scale"]))
    if c["kind"] == "append":
        n_q, n_kv, dim = c["n_q"], c["n_kv"], c["dim"]
        ld, at = (n_q + 2 * n_kv) * dim, s["qkv"].data_ptr()
        args = (cache, at, at + 2 * n_q * dim, at + 2 * (n_q + n_kv) * dim, ptr(s["norm_w"][0]), ptr(s["norm_w"][1]), ptr(s["cos"]), ptr(s["sin"]), s["cos"].shape[0], ptr(s["q_out"]),
                n_q, s["tokens"], ld, ld, ld, EPS)
        return lib.qk_norm_rope_kv_paged, args, _appended(s)
    if c["kind"] == "read":
        args = (cache, ptr(s["k_out"]), ptr(s["v_out"]), s["tokens"], c["n_kv"] * c["dim"], c["dim"])
        return lib.kv_paged_read, args, (s["k_out"], s["v_out"])
    need = lib.attention_paged_workspace_bytes(cache, c["n_q"], s["tokens"], s["max_new"], s["max_ctx"], c["window"], c["sinks"])
    s["workspace"] = torch.empty(need, dtype=torch.uint8, device=s["q"].device)
    ld = c["n_q"] * c["dim"]
    args = (cache, ptr(s["q"]), ptr(s["y"]), ptr(s["workspace"]), need, c["n_q"], s["tokens"], s["max_new"], s["max_ctx"], c["window"], c["sinks"], ld, ld)
    return lib.attention_paged, args, s["y"]


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _bound(state)
        entry, args, out = state["call"]
        status = entry(*args)
        if status:
            raise RuntimeError(f"{state['case']['kind']}: {status}")
        return out
    return {"append": _append_plain, "read": _read_plain, "attend": _attend_plain}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------------------- in 64 bits

def _table(cache):
    """The value of every FP8 code, by its bits."""
    _, _, top, _, bits, least = CACHES[cache]
    code = torch.arange(256, dtype=torch.float64)
    sign = torch.where(code >= 128, -1.0, 1.0)
    field, fraction = torch.floor(code % 128 / 2 ** bits), code % 2 ** bits
    value = torch.where(field == 0, fraction * 2.0 ** (least - bits), (1 + fraction * 2.0 ** -bits) * 2.0 ** (field - 1 + least))
    if cache == "e4m3":
        value[127::128] = math.nan
    else:
        value[124::128], value[125::128], value[126::128], value[127::128] = math.inf, math.nan, math.nan, math.nan
    return sign * value


def _two(e):
    """2^e in 64 bits."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _rows64(s, name, seq, lo, hi):
    """Rows lo .. hi - 1 of a sequence, [row][kv head][dim]."""
    page = s["case"]["page"]
    pos = torch.arange(lo, hi, device=s["table"].device)
    at = s["table"][seq].long()[pos // page]
    x = s[name][at, :, pos % page]
    if s["case"]["cache"] == "bf16":
        return x.double()
    return _table(s["case"]["cache"]).to(x.device)[x.long()] * _two(s[name + "_scale"][at, :, pos % page].long() - 127)[..., None]


def _codes64(x, cache):
    """Code values (not yet times their power of two) and powers of two of rows in 64 bits."""
    _, _, top, largest, bits, least = CACHES[cache]
    amax = x.abs().amax(-1)
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -140) / largest))
    e = torch.where(amax > largest * _two(e), e + 1, torch.where(amax <= largest * _two(e - 1), e - 1, e)).clamp(-100, 127 - top)
    y = x * _two(-e)[..., None]
    step = _two(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** least))).clamp(min=least) - bits)
    return (torch.round(y / step) * step).clamp(-largest, largest), _two(e)


def exact(case, seed):
    s = prepare(case, seed)
    new, ctx = lengths(case)
    n_q, n_kv, dim, page = case["n_q"], case["n_kv"], case["dim"], case["page"]
    dev, group = s["table"].device, n_q // n_kv
    if case["kind"] == "read":
        rows = [[_rows64(s, name, i, c - n, c) for i, (n, c) in enumerate(zip(new, ctx))] for name in ("k", "v")]
        return tuple(torch.cat(r) for r in rows)
    at = 0
    if case["kind"] == "append":
        fp8 = case["cache"] != "bf16"
        pools = {name: _table(case["cache"]).to(dev)[s[name].long()] if fp8 else s[name].double() for name in ("k", "v")}
        scales = {name: _two(s[name + "_scale"].long() - 127) if fp8 else None for name in ("k", "v")}
        q_out = torch.zeros(s["tokens"], n_q, dim, dtype=torch.float64, device=dev)
        for i, (n, c) in enumerate(zip(new, ctx)):
            x = s["qkv"][at:at + n].double().view(n, -1, dim)
            pos = torch.arange(c - n, c, device=dev)
            turned = []
            for part, w in ((x[:, :n_q], s["norm_w"][0]), (x[:, n_q:n_q + n_kv], s["norm_w"][1])):
                if w is not None:
                    part = part / torch.sqrt((part * part).sum(-1, keepdim=True) / dim + EPS) * w.double()
                z = torch.complex(part[..., :dim // 2], part[..., dim // 2:]) * torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
                turned.append(torch.cat([z.real, z.imag], -1))
            q_out[at:at + n] = turned[0]
            where = s["table"][i].long()[pos // page]
            for name, rows in (("k", turned[1]), ("v", x[:, n_q + n_kv:])):
                if fp8:
                    pools[name][where, :, pos % page], scales[name][where, :, pos % page] = _codes64(rows, case["cache"])
                else:
                    pools[name][where, :, pos % page] = rows
            at += n
        return (q_out, pools["k"], pools["v"]) + ((scales["k"], scales["v"]) if fp8 else ())
    y = torch.zeros(s["tokens"], n_q, dim, dtype=torch.float64, device=dev)
    for i, (n, c) in enumerate(zip(new, ctx)):
        if not n:
            continue
        first = c - n                                                   # keys that no new token sees are left out
        skip = max(0, first + 1 - case["window"]) if case["window"] else 0
        skip = skip if skip > case["sinks"] else 0
        pos = torch.arange(c, device=dev)
        kept = torch.cat([pos[:case["sinks"]], pos[skip:]]) if skip else pos
        k, v = (_rows64(s, name, i, 0, c)[kept] for name in ("k", "v"))
        me = torch.arange(first, c, device=dev)[:, None]
        hidden = kept > me
        if case["window"]:
            hidden |= (kept <= me - case["window"]) & (kept >= case["sinks"])
        for h in range(n_q):
            score = s["q"][at:at + n, h].double() @ k[:, h // group].t().contiguous() / math.sqrt(dim)
            weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            y[at:at + n, h] = weight @ v[:, h // group].contiguous()
        at += n
    return y
