"""Operators of a batch whose sequences branch, on a paged key / value cache, in plain torch and through this library's entry points.

* tree    attention of drafted tokens that form a tree: each sees all rows in front of its sequence's new tokens (or a window of the newest and a
          few first ones) and those new tokens that its bits name                                     hip_attention_paged_tree_bf16
* append  q/k RMSNorm per head, RoPE by positions that are given per token, on one axis or three, and the append of the keys and values to
          the pages of their sequences                                                                hip_qk_norm_rope_kv_paged_at_bf16
* keep    the accepted tokens' rows move up behind the rows in front of them, in all layers            hip_kv_paged_keep
* fork    sequences take over the rows of others: whole pages shared, partly filled last ones copied in all layers, pages for what comes next
          taken from those that nobody holds                                                          hip_kv_paged_fork
* beam    the best continuations of each group of beams over the vocabulary                            hip_beam_select_bf16

The batch: sequence s has n_new new tokens, rows seq_start[s] .. seq_start[s + 1] - 1 of the activations, and ctx_len[s] rows in the cache, the
new ones included; row `pos` lies in page page_table[s][pos / page] at row pos % page.  Pages are [kv head][row][dim].  FP8 rows are codes with a power of
two each, 2^(byte - 127), the smallest >= 2^-100 for which the row's largest magnitude stays within the type's largest value.

Lengths are those of the case; the values, the trees' shapes, the parents, and where in the pool a sequence's pages lie, come from the seed.
"""
import math
import random

import torch

own = False

#: cache type -> (type number of the library, torch type, exponent and value of the largest number, mantissa bits, exponent of the smallest normal)
CACHES = {"bf16": (3, torch.bfloat16, None, None, None, None),
          "e4m3": (4, torch.float8_e4m3fn, 8, 448.0, 3, -6),
          "e5m2": (5, torch.float8_e5m2, 15, 57344.0, 2, -14)}
EPS = 1e-6
NOBODY = 1 << 30                                # a page that no sequence holds

GQA = dict(n_q=32, n_kv=8, dim=128)             # the head layout of the Qwen3-8B and Llama-3.1-8B shapes
KV = dict(n_kv=8, dim=128)
WIDE = dict(n_q=64, n_kv=8, dim=64)             # eight query heads per kv head


def listed():
    return [
        # one chat, a small tree of drafts behind the context that the benchmark is quoted on
        dict(name="tree_1_seq_13_nodes_bf16", kind="tree", cache="bf16", page=64, seqs=1, new_lo=13, new_hi=13, behind_lo=4095, behind_hi=4095, window=0, sinks=0, **GQA),
        # two drafts of two tokens for each of sixteen long streams that keep a window and the first tokens
        dict(name="tree_16_seqs_4_nodes_window_e4m3", kind="tree", cache="e4m3", page=32, seqs=16, new_lo=4, new_hi=4, behind_lo=16000, behind_hi=32000, window=4096, sinks=4, **GQA),
        # a few chats with wide trees, many query heads per kv head
        dict(name="tree_8_seqs_60_nodes_e5m2", kind="tree", cache="e5m2", page=16, seqs=8, new_lo=60, new_hi=60, behind_lo=500, behind_hi=3000, window=0, sinks=0, **WIDE),
        # a full serving batch with trees of different sizes: the largest call
        dict(name="tree_32_seqs_17_to_33_nodes_e4m3", kind="tree", cache="e4m3", page=16, seqs=32, new_lo=17, new_hi=33, behind_lo=1000, behind_hi=8000, window=0, sinks=0, **GQA),
        # the keys and values of eight trees, each token at its depth
        dict(name="append_8_trees_26_nodes_e4m3", kind="append", cache="e4m3", page=16, axes=1, mixed=False, seqs=8, new_lo=26, new_hi=26, behind_lo=500, behind_hi=4000, norm=True, **GQA),
        # prompts of text around an image, positions in time, height and width
        dict(name="append_4_images_bf16", kind="append", cache="bf16", page=64, axes=3, mixed=False, seqs=4, new_lo=1101, new_hi=2600, behind_lo=0, behind_hi=0, norm=False, **GQA),
        # what one chat accepted of its tree, in the layers of the 8B shape
        dict(name="keep_1_seq_of_13_bf16", kind="keep", cache="bf16", page=64, layers=36, seqs=1, new_lo=13, new_hi=13, behind_lo=300, behind_hi=300, kept_lo=4, kept_hi=4, **KV),
        # the same of a batch
        dict(name="keep_32_seqs_of_26_e4m3", kind="keep", cache="e4m3", page=16, layers=36, seqs=32, new_lo=26, new_hi=26, behind_lo=100, behind_hi=600, kept_lo=1, kept_hi=9, **KV),
        # four beams of one chat take their next step
        dict(name="fork_4_beams_bf16", kind="fork", cache="bf16", page=16, layers=36, groups=1, beams=4, alive=3, leave=0, ctx_lo=1003, ctx_hi=1003, fresh=0, **KV),
        # a batch of beam searches, two of which end and make room for new prompts
        dict(name="fork_16_groups_4_beams_e4m3", kind="fork", cache="e4m3", page=64, layers=32, groups=16, beams=4, alive=2, leave=2, ctx_lo=200, ctx_hi=2000, fresh=700, **KV),
        # one chat's four beams over the vocabulary of the Qwen3-8B shape
        dict(name="beam_1_group_of_4", kind="beam", groups=1, beams=4, vocab=151936, n_out=4, done=0, first=False, barred=0.0),
        # a batch of beam searches over the vocabulary of the Llama-3.1-8B shape, with room for those that end
        dict(name="beam_16_groups_of_8", kind="beam", groups=16, beams=8, vocab=128256, n_out=16, done=1, first=False, barred=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """More of the same: what a listed case costs at most, and what its plain form can hold."""
    kind = rng.choice(["tree", "tree", "tree", "append", "keep", "fork", "beam"])
    while True:
        if kind == "beam":
            beams = rng.choice([1, 2, 3, 4, 4, 5, 8, 16])
            vocab = _log(rng, 1000, 151936)
            c = dict(kind=kind, groups=_log(rng, 1, 64), beams=beams, vocab=vocab, n_out=beams * rng.choice([1, 1, 2]), done=rng.choice([0, 0, 1]) if beams > 1 else 0,
                     first=rng.random() < 0.2, barred=rng.choice([0.0, 0.0, 0.9]))
            if c["groups"] * beams * vocab > 1.6e7:
                continue
            return c
        n_kv = rng.choice([1, 2, 4, 8, 8, 8])
        c = dict(kind=kind, cache=rng.choice(sorted(CACHES)), page=rng.choice([16, 16, 32, 64, 128]), n_kv=n_kv, dim=rng.choice([64, 128, 128]))
        if kind in ("tree", "append"):
            c |= dict(n_q=n_kv * rng.choice([1, 2, 3, 4, 4, 5, 8]))
        if kind == "fork":
            groups, beams, lo = _log(rng, 1, 32), rng.choice([1, 2, 3, 4, 4, 8]), _log(rng, 1, 2000)
            c |= dict(layers=rng.randint(1, 36), groups=groups, beams=beams, alive=rng.randint(1, beams), leave=rng.randint(0, groups // 3), ctx_lo=lo, ctx_hi=min(2000, 2 * lo), fresh=_log(rng, 1, 2000))
            if sum(_fork_pages(c)) * c["page"] * c["layers"] * n_kv * c["dim"] > 1.6e9 or work(c)["bytes"] > 4e8:
                continue
            return c
        seqs, n, behind = _log(rng, 1, 64), _log(rng, 2, 100), _log(rng, 16, 16000)
        c |= dict(seqs=seqs, new_lo=rng.randint(1, n), new_hi=n, behind_lo=rng.randint(0, behind), behind_hi=behind)
        if kind == "tree":
            window = rng.choice([0, 0, 0, _log(rng, 64, 4096)])
            c |= dict(window=window, sinks=rng.choice([0, 1, 4, 16]) if window else 0)
        elif kind == "append":
            axes = rng.choice([1, 3])
            c |= dict(axes=axes, mixed=axes == 3 and rng.random() < 0.5, norm=rng.random() < 0.5)
            if axes == 3:
                n = _log(rng, 16, 4000)
                c |= dict(seqs=min(seqs, 16), new_lo=rng.randint(1, n), new_hi=n)
        else:
            behind = min(behind, 600)
            hi = rng.randint(1, min(n, 12))
            c |= dict(layers=rng.randint(1, 36), behind_lo=rng.randint(0, behind), behind_hi=behind, kept_lo=rng.randint(1, hi), kept_hi=hi)
        new, ctx = lengths(c)
        w = work(c)
        if w["bytes"] > 3.2e8 or w["flops"] > 1e11 or sum(ctx) * n_kv * c["dim"] * c.get("layers", 1) > 1.2e9:
            continue
        if kind == "tree" and (c["seqs"] * c["n_q"] * max(new) * max(ctx) > 4e8 or c["seqs"] * max(ctx) * n_kv * c["dim"] > 9e8):
            continue
        if kind == "keep" and w["bytes"] == 0:
            continue
        return c


def _spread(n, lo, hi, start, step):
    return [lo + int((start + step * i) % 1.0 * (hi - lo + 1)) for i in range(n)]


def lengths(case):
    """New tokens and rows in the cache of each sequence, spread over their ranges."""
    new = _spread(case["seqs"], case["new_lo"], case["new_hi"], 0.5, 0.6180339887498949)
    behind = _spread(case["seqs"], case["behind_lo"], case["behind_hi"], 0.25, 0.7548776662466927)
    return new, [n + b for n, b in zip(new, behind)]


def _kept(case):
    """How many new tokens of each sequence are kept, and how many of those are where they belong already."""
    kept = [min(k, n) for k, n in zip(_spread(case["seqs"], case["kept_lo"], case["kept_hi"], 0.7, 0.5698402909980532), lengths(case)[0])]
    return kept, [max(1, 2 * k - n) for k, n in zip(kept, lengths(case)[0])]


def _fork_lengths(case):
    """Rows of each group's beams, of which so many are shared by them."""
    ctx = _spread(case["groups"], case["ctx_lo"], case["ctx_hi"], 0.5, 0.6180339887498949)
    return ctx, [int(0.7 * c) // case["page"] * case["page"] for c in ctx]


def _fork_pages(case):
    """Pages held by all beams before, and the most that they take."""
    page, beams = case["page"], case["beams"]
    held = sum(s // page + beams * (-(-c // page) - s // page) for c, s in zip(*_fork_lengths(case)))
    return held, case["groups"] * beams * 2 + case["leave"] * (-(-case["fresh"] // page))


def row_bytes(case):
    return 2 * case["dim"] if case["cache"] == "bf16" else case["dim"] + 1


def work(case):
    kind = case["kind"]
    if kind == "beam":
        rows = case["groups"] * (1 if case["first"] else case["beams"] - case["done"])          # what lives
        return {"bytes": 2 * rows * case["vocab"] + 4 * case["groups"] * (2 * case["beams"] + 3 * case["n_out"]), "flops": 4 * rows * case["vocab"]}
    n_kv, dim, row = case["n_kv"], case["dim"], row_bytes(case)
    if kind == "fork":
        page, beams = case["page"], case["beams"]
        ctx, _ = _fork_lengths(case)
        stay = ctx[:case["groups"] - case["leave"]]
        copied = sum((beams - case["alive"]) * (c % page) for c in stay)
        entries = sum(beams * -(-c // page) for c in stay)
        return {"bytes": 2 * copied * case["layers"] * 2 * n_kv * row + 4 * (entries + case["groups"] * beams * _table_stride(case)), "flops": 0}
    new, ctx = lengths(case)
    tokens = sum(new)
    if kind == "keep":
        kept, there = _kept(case)
        return {"bytes": 2 * sum(k - t for k, t in zip(kept, there)) * case["layers"] * 2 * n_kv * row, "flops": 0}
    n_q = case["n_q"]
    if kind == "append":
        tables = 2 * 2 * (dim // 2) * tokens + (4 * dim if case["norm"] else 0)
        return {"bytes": 2 * dim * tokens * (2 * n_q + 2 * n_kv) + 2 * n_kv * tokens * row + tables + 4 * case["axes"] * tokens,
                "flops": tokens * (n_q + n_kv) * dim * (3 + (4 if case["norm"] else 0))}
    rows = pairs = 0
    for n, c in zip(new, ctx):
        first = c - n                                                   # position of the first new token
        seen = min(first, case["window"] + case["sinks"]) if case["window"] else first
        rows += seen + n
        pairs += n * (seen + 1)                                         # of the new ones itself, at least
    return {"bytes": 2 * 2 * dim * n_q * tokens + 2 * n_kv * rows * row + 8 * tokens * -(-max(new) // 64), "flops": 4 * dim * n_q * pairs}


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


def _trees(seqs, most, g, dev):
    """Which tokens of its tree each token descends from, itself among them: [seq][token][token]; token 0 is the root, a parent comes before its children."""
    at = torch.arange(most, device=dev)
    u = torch.rand(seqs, most, generator=g, device=dev)
    parent = (u.pow(1.5) * at).long().clamp(min=0)                  # more children near the root
    up = torch.nn.functional.one_hot(parent, most).float()
    up[:, 0] = 0.0
    line = up + torch.eye(most, device=dev)
    for _ in range(max(1, (most - 1).bit_length())):                # twice as many generations each time
        line = (torch.bmm(line, line) > 0).float()
    return line > 0


def _table_stride(case):
    ctx, _ = _fork_lengths(case)
    return max(max(ctx) + 2 * case["page"], case["fresh"] + 1 if case["leave"] else 0) // case["page"] + 1


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, generator=g, device=dev)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    if case["kind"] == "beam":
        return _prepare_beam(case, g, normal, uniform, dev)
    if case["kind"] == "fork":
        return _prepare_fork(case, seed, g, normal, ints, dev)
    new, ctx = lengths(case)
    seqs, page, n_kv, dim = case["seqs"], case["page"], case["n_kv"], case["dim"]
    tokens, most, layers = sum(new), max(ctx), case.get("layers", 1)

    # a pool whose pages lie in any order, with a few that belong to nobody
    pages = [-(-c // page) for c in ctx]
    n_pages, per_seq = sum(pages) + 5, -(-most // page)
    order = torch.randperm(n_pages, generator=g, device=dev).int()
    first = ints([sum(pages[:s]) for s in range(seqs)])
    at = torch.arange(per_seq, device=dev, dtype=torch.int32)
    table = torch.where(at < ints(pages)[:, None], order[(first[:, None] + at).clamp(max=n_pages - 1)], torch.zeros_like(at)).contiguous()
    s = dict(case=case, max_new=max(new), max_ctx=most, tokens=tokens, n_pages=n_pages, table=table, ctx_len=ints(ctx), seq_start=ints([sum(new[:i]) for i in range(seqs + 1)]))
    _pools(s, layers, n_pages, g, normal, dev)
    if case["kind"] == "keep":
        rng = random.Random(seed)
        kept, there = _kept(case)
        keep = torch.zeros(tokens, dtype=torch.int32)
        begin = 0
        for n, k, t in zip(new, kept, there):
            # none of those that move comes from where another goes, so that a second pass finds what the first did
            keep[begin:begin + k] = torch.tensor(list(range(t)) + sorted(rng.sample(range(k, n), k - t)), dtype=torch.int32)
            begin += n
        s |= dict(keep=keep.to(dev), n_keep=ints(kept), ctx_out=torch.empty(seqs, dtype=torch.int32, device=dev))
        return s
    n_q = case["n_q"]
    lines = _trees(seqs, max(new), g, dev) if case["kind"] == "tree" or case["axes"] == 1 else None
    seq, index, _ = _tokens(s)
    if case["kind"] == "tree":
        words = -(-max(new) // 64)
        bits = torch.zeros(tokens, words * 64, dtype=torch.int64, device=dev)
        bits[:, :max(new)] = lines[seq, index.long()].long()
        s["seen"] = (bits.view(tokens, words, 64) << torch.arange(64, device=dev)).sum(-1)
        s["q"] = (1.3 * normal(tokens, n_q, dim)).bfloat16()
        s["y"] = torch.empty(tokens, n_q, dim, dtype=torch.bfloat16, device=dev)
        return s
    # q, k and v as one projection writes them, side by side
    s["qkv"] = normal(tokens, (n_q + 2 * n_kv) * dim).bfloat16()
    s["q_out"] = torch.empty(tokens, n_q, dim, dtype=torch.bfloat16, device=dev)
    s["norm_w"] = [(1.0 + 0.2 * normal(dim)).bfloat16() if case["norm"] else None for _ in range(2)]
    angle = torch.arange(most, device=dev, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(dim // 2, device=dev, dtype=torch.float64) / (dim // 2))
    s["cos"], s["sin"] = angle.cos().bfloat16(), angle.sin().bfloat16()
    behind = (s["ctx_len"] - (s["seq_start"][1:] - s["seq_start"][:-1]))[seq]
    if case["axes"] == 1:
        s["positions"] = (behind + lines[seq, index.long()].sum(-1).int() - 1)[None].contiguous()
        s["axis"] = None
    else:
        # a quarter text, an image of rows of `wide` patches, text again behind its largest position
        n = (s["seq_start"][1:] - s["seq_start"][:-1])[seq]
        text = n // 4
        wide = (n // 2).float().sqrt().int().clamp(min=1)
        patches = wide * (n // 2 // wide)
        p = index - text
        later = torch.where(p >= patches, p - patches + wide.maximum(patches // wide), torch.zeros_like(p))
        image = (p >= 0) & (p < patches)
        s["positions"] = torch.stack([torch.where(p < 0, index, text + torch.where(image, by, later)) for by in (torch.zeros_like(p), p // wide, p % wide)]).int().add_(behind.int()).contiguous()
        pair = torch.arange(dim // 2, device=dev)
        s["axis"] = (pair % 3 if case["mixed"] else (pair >= dim // 8).int() + (pair >= dim // 8 + dim * 3 // 16).int()).to(torch.uint8)
    return s


def _pools(s, layers, n_pages, g, normal, dev):
    """Keys with a few strong channels, and narrower values; one pool per layer."""
    c = s["case"]
    n_kv, dim, page = c["n_kv"], c["dim"], c["page"]
    gain = 0.5 + 0.5 * torch.rand(n_kv, 1, dim, generator=g, device=dev) + 2.0 * (torch.rand(n_kv, 1, dim, generator=g, device=dev) < 0.03)
    for name, by in (("k", gain), ("v", 0.5)):
        got = []
        for _ in range(layers):
            rows = (normal(n_pages, n_kv, page, dim) * by).bfloat16()
            got.append((rows, None) if c["cache"] == "bf16" else _quantized(rows, c["cache"]))
        s[name] = torch.stack([r for r, _ in got])
        s[name + "_scale"] = None if c["cache"] == "bf16" else torch.stack([e for _, e in got])


def _prepare_fork(case, seed, g, normal, ints, dev):
    rng = random.Random(seed)
    groups, beams, page, stride = case["groups"], case["beams"], case["page"], _table_stride(case)
    ctx, shared = _fork_lengths(case)
    held, more = _fork_pages(case)
    n_pages = held + more + 7
    order = list(range(n_pages))
    rng.shuffle(order)
    table = torch.full((groups * beams, stride), -1, dtype=torch.int32)
    reserved = torch.zeros(n_pages, dtype=torch.uint8)
    parent, grow = [], []
    for i in range(groups):
        common = [order.pop() for _ in range(shared[i] // page)]
        for b in range(beams):
            mine = common + [order.pop() for _ in range(-(-ctx[i] // page) - len(common))]
            table[i * beams + b, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
        if i >= groups - case["leave"]:
            # this search is over: a new prompt takes its first place
            parent += [-1] * beams
            grow += [case["fresh"]] + [0] * (beams - 1)
            continue
        alive = rng.sample(range(beams), case["alive"])
        chosen = alive + [rng.choice(alive) for _ in range(beams - len(alive))]
        rng.shuffle(chosen)
        parent += [i * beams + b for b in chosen]
        grow += [1] * beams
    reserved[order.pop()] = reserved[order.pop()] = 1               # pages of a prefix that the program keeps for later
    s = dict(case=case, n_pages=n_pages, table=table.to(dev), ctx_len=ints([c for c in ctx for _ in range(beams)]), seq_start=ints(list(range(groups * beams + 1))),
             parent=ints(parent), grow=ints(grow), reserved=reserved.to(dev))
    s |= dict(table_out=torch.empty_like(s["table"]), ctx_out=torch.empty_like(s["ctx_len"]), missing=torch.empty(1, dtype=torch.int32, device=dev))
    _pools(s, case["layers"], n_pages, g, normal, dev)
    return s


def _prepare_beam(case, g, normal, uniform, dev):
    groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
    rows, pitch = groups * beams, -(-vocab // 8) * 8
    logits = 2.2 * normal(rows, pitch)
    # a few tokens stand out, the same ones in part for the beams of a group
    for count, by in ((12, 6.0), (200, 3.0)):
        like = (uniform(groups, 1, count) * vocab).long().expand(-1, beams, -1).reshape(rows, count)
        other = (uniform(rows, count) * vocab).long()
        logits.scatter_add_(1, torch.where(uniform(rows, count) < 0.5, like, other), by * uniform(rows, count))
    if case["barred"]:
        logits.masked_fill_(uniform(rows, pitch) < case["barred"], -math.inf)
    score = -40.0 * uniform(groups, beams)
    if case["first"]:
        score[:, 1:] = -math.inf                                    # beams that have not begun
    last = (uniform(rows) * (vocab - 1)).int() + 1
    last.view(groups, beams)[:, :case["done"]] = 0
    return dict(case=case, logits=logits.bfloat16(), score=score.view(-1).contiguous(), last=last, eos=0,
                parent=torch.empty(groups * case["n_out"], dtype=torch.int32, device=dev), token=torch.empty(groups * case["n_out"], dtype=torch.int32, device=dev),
                score_out=torch.empty(groups * case["n_out"], dtype=torch.float32, device=dev))


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
    x = s[name][0][page, :, row]
    if s["case"]["cache"] == "bf16":
        return x.float()
    return x.view(CACHES[s["case"]["cache"]][1]).float() * _power(s[name + "_scale"][0][page, :, row].int() - 127)[..., None]


def _pool_values(s):
    """The pools, FP8 codes and powers of two as the values they stand for."""
    if s["case"]["cache"] == "bf16":
        return s["k"], s["v"]
    kind = CACHES[s["case"]["cache"]][1]
    return s["k"].view(kind), s["v"].view(kind), s["k_scale"].view(torch.float8_e8m0fnu), s["v_scale"].view(torch.float8_e8m0fnu)


def _tree_plain(s):
    c = s["case"]
    seqs, n_q, n_kv, dim = c["seqs"], c["n_q"], c["n_kv"], c["dim"]
    group, dev = n_q // n_kv, s["q"].device
    key = torch.arange(s["max_ctx"], device=dev, dtype=torch.int32)
    page, row = _slots(s, torch.arange(seqs, device=dev)[:, None], key.expand(seqs, -1))
    keys = _values(s, "k", page, row).permute(0, 2, 3, 1).contiguous()                 # [seq][kv head][dim][key]
    # each sequence's new tokens, the heads of a kv head side by side: [seq][kv head][token x head][dim]
    new = s["seq_start"][1:] - s["seq_start"][:-1]
    index = torch.arange(s["max_new"], device=dev, dtype=torch.int32)
    at = (s["seq_start"][:-1, None] + index).clamp(max=s["tokens"] - 1).long()
    q = s["q"][at].float().view(seqs, -1, n_kv, group, dim).transpose(1, 2).reshape(seqs, n_kv, -1, dim)
    score = torch.matmul(q, keys).mul_(1.0 / math.sqrt(dim)).view(seqs, n_kv, -1, group, s["max_ctx"])
    del keys, q
    named = (s["seen"][at][..., None] >> torch.arange(64, device=dev) & 1).bool().flatten(2)           # [seq][token][new token]
    first = (s["ctx_len"] - new)[:, None]
    j = (key - first).long()                                                            # [seq][key]
    seen = torch.gather(named, 2, j.clamp(0, named.shape[2] - 1)[:, None].expand(-1, s["max_new"], -1)) & (j < new[:, None])[:, None]
    before = (j < 0)[:, None]
    if c["window"]:
        pos = first + (named & (torch.arange(named.shape[2], device=dev) < new[:, None])[:, None]).sum(-1) - 1
        before = before & ((key > pos[..., None] - c["window"]) | (key < c["sinks"]))
    seen = torch.where((j < 0)[:, None], before, seen)
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    score.div_(score.sum(-1, keepdim=True))
    values = _values(s, "v", page, row).permute(0, 2, 1, 3).contiguous()               # [seq][kv head][key][dim]
    y = torch.matmul(score.view(seqs, n_kv, -1, s["max_ctx"]), values).view(seqs, n_kv, -1, group, dim).transpose(1, 2).reshape(seqs, -1, n_q, dim)
    seq, index, _ = _tokens(s)
    return y[seq, index.long()].bfloat16()


def _append_plain(s):
    c = s["case"]
    n_q, n_kv, dim = c["n_q"], c["n_kv"], c["dim"]
    seq, _, pos = _tokens(s)
    page, row = _slots(s, seq, pos)
    x = s["qkv"].view(s["tokens"], n_q + 2 * n_kv, dim)
    pair = torch.arange(dim // 2, device=x.device)
    at = s["positions"][torch.zeros_like(pair) if s["axis"] is None else s["axis"].long()].t().long()   # [token][pair]
    cos, sin = s["cos"][at, pair].float()[:, None], s["sin"][at, pair].float()[:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.float()
        lo, hi = x[..., :dim // 2], x[..., dim // 2:]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    s["q_out"].copy_(turned(x[:, :n_q], s["norm_w"][0]))
    for name, rows in (("k", turned(x[:, n_q:n_q + n_kv], s["norm_w"][1])), ("v", x[:, n_q + n_kv:])):
        if c["cache"] == "bf16":
            s[name][0][page, :, row] = rows.bfloat16()
        else:
            s[name][0][page, :, row], s[name + "_scale"][0][page, :, row] = _quantized(rows, c["cache"])
    return (s["q_out"],) + _pool_values(s)


def _keep_plain(s):
    seq, index, _ = _tokens(s)
    first = s["ctx_len"] - (s["seq_start"][1:] - s["seq_start"][:-1])
    moves = torch.nonzero((index < s["n_keep"][seq]) & (s["keep"] != index))[:, 0]
    seq = seq[moves]
    page, row = _slots(s, seq, first[seq] + s["keep"][moves])
    to_page, to_row = _slots(s, seq, first[seq] + index[moves])
    for name in ("k", "v", "k_scale", "v_scale"):
        if s[name] is not None:
            s[name][:, to_page, :, to_row] = s[name][:, page, :, row]
    torch.add(first, s["n_keep"], out=s["ctx_out"])
    return (s["ctx_out"],) + _pool_values(s)


def _fork_plain(s):
    page, n_pages = s["case"]["page"], s["n_pages"]
    dev, (n_seqs, stride) = s["table"].device, s["table"].shape
    has = (s["parent"] >= 0) & (s["parent"] < n_seqs)
    source = s["parent"].clamp(0, n_seqs - 1).long()
    rows = torch.where(has, s["ctx_len"][source], 0)
    total = (rows + s["grow"]).clamp(max=stride * page)
    at = torch.arange(stride, device=dev, dtype=torch.int32)
    old = s["table"][source]
    there = (old >= 0) & (old < n_pages)
    full = (at < (rows // page)[:, None]) & there
    last = (at == (rows // page)[:, None]) & (rows % page > 0)[:, None] & there
    # who holds a page: as a whole (0), or as a last one, partly filled (its number + 1)
    me = torch.arange(len(rows), device=dev, dtype=torch.int32)[:, None] + 1
    holder = torch.where(s["reserved"] > 0, 0, NOBODY).int()
    claim = torch.where(full, 0, torch.where(last, me.expand_as(old), NOBODY)).int()
    holder = holder.scatter_reduce(0, old.clamp(0, n_pages - 1).long().flatten(), claim.flatten(), "amin")
    copied = last & (holder[old.clamp(0, n_pages - 1).long()] != me)
    need = copied | ((at >= ((rows + page - 1) // page)[:, None]) & (at < ((total + page - 1) // page)[:, None]))
    free = holder == NOBODY
    place = torch.where(free, free.cumsum(0) - 1, n_pages)
    pages = torch.full((n_pages + 1,), -1, dtype=torch.int32, device=dev).scatter_(0, place, torch.arange(n_pages, device=dev, dtype=torch.int32))
    pages[n_pages] = -1
    turn = need.flatten().cumsum(0).view_as(need) - 1
    got = pages[torch.where(need, turn, n_pages).clamp(max=n_pages)]
    s["table_out"].copy_(torch.where(need, got, torch.where(full | last, old, -1)))
    s["ctx_out"].copy_(total)
    s["missing"].copy_((need & (got < 0)).sum())
    # the rows of the last pages that were not anybody's own
    who = torch.nonzero(copied & (got >= 0))
    src, dst = old[who[:, 0], who[:, 1]].long(), got[who[:, 0], who[:, 1]].long()
    mine = torch.arange(page, device=dev) < (rows % page)[who[:, 0], None]             # [copy][row]
    for name in ("k", "v", "k_scale", "v_scale"):
        if s[name] is not None:
            m = mine[:, None].view(1, len(who), 1, page, *[1] * (s[name].dim() - 4))
            s[name][:, dst] = torch.where(m, s[name][:, src], s[name][:, dst])
    return (s["table_out"], s["ctx_out"], s["missing"]) + _pool_values(s)


def _beam_plain(s):
    c = s["case"]
    groups, beams, vocab, n_out = c["groups"], c["beams"], c["vocab"], c["n_out"]
    x = s["logits"][:, :vocab].float()
    dead, done = ~torch.isfinite(s["score"]), s["last"] == s["eos"]
    # sums in 64 bits: scores next to each other decide
    log_sum = torch.logsumexp(x.double(), 1) if not c["barred"] else (x.double() - x.amax(1, keepdim=True)).exp().sum(1).log() + x.amax(1)
    # the best of a row by its logits, equal ones by their index: a logit's order in the upper, its place from behind in the lower half of a whole number
    bits = (x + 0.0).bfloat16().view(torch.int16).long()                                 # -0 is 0
    order = torch.where(bits < 0, -32768 - bits, bits)
    low = -32768 - torch.tensor(-math.inf, dtype=torch.bfloat16).view(torch.int16).long().item()
    token = torch.arange(vocab, device=x.device)
    order = torch.where(done[:, None], torch.where(token == s["eos"], 0, low), torch.where(dead[:, None], low, order))
    best = torch.topk(order * (1 << 32) + (vocab - 1 - token), min(n_out, vocab), dim=1).values
    at = vocab - 1 - (best & 0xFFFFFFFF)
    total = s["score"].double()[:, None] + torch.where(done[:, None], torch.where(at == s["eos"], 0.0, -math.inf).double(), torch.gather(x, 1, at).double() - log_sum[:, None])
    total = torch.where(dead[:, None], -math.inf, total)
    total, pick = torch.sort(total.view(groups, -1), dim=1, descending=True, stable=True)
    pick = pick[:, :n_out]
    row = pick // best.shape[1] + beams * torch.arange(groups, device=x.device)[:, None]
    return row.int().flatten(), torch.gather(at.view(groups, -1), 1, pick).int().flatten(), total[:, :n_out].float().flatten()


# ------------------------------------------------------------------------------------------------- the library's operators

def _bound(s):
    """The call that a user's program keeps: descriptors, workspace and the rest of the arguments."""
    import importlib

    pkg = importlib.import_module("cccc-lite_amd")
    lib, c = pkg.library(), s["case"]
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    space = lambda n: torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")  # noqa: E731
    if c["kind"] == "beam":
        shape = (c["groups"], c["beams"], c["vocab"], c["n_out"])
        need = lib.beam_select_workspace_bytes(*shape)
        s["workspace"] = space(need)
        return lib.beam_select, (ptr(s["logits"]), s["logits"].stride(0), ptr(s["score"]), ptr(s["last"]), s["eos"], *shape, ptr(s["parent"]), ptr(s["token"]), ptr(s["score_out"]),
                                 ptr(s["workspace"]), need), (s["parent"], s["token"], s["score_out"])
    caches = [pkg.capi.make_paged_kv(CACHES[c["cache"]][0], c["dim"], c["n_kv"], c["page"], s["n_pages"], ptr(s["k"][i]), ptr(s["v"][i]), ptr(s["table"]), s["table"].shape[1], ptr(s["ctx_len"]),
                                     ptr(s["seq_start"]), len(s["ctx_len"]), k_scale=None if s["k_scale"] is None else ptr(s["k_scale"][i]),
                                     v_scale=None if s["v_scale"] is None else ptr(s["v_scale"][i])) for i in range(c.get("layers", 1))]
    if c["kind"] == "fork":
        layers = pkg.capi.paged_layers(caches)
        need = lib.kv_paged_fork_workspace_bytes(layers, len(caches), len(s["parent"]))
        s["workspace"] = space(need)
        return lib.kv_paged_fork, (layers, len(caches), len(s["parent"]), ptr(s["parent"]), None, ptr(s["grow"]), ptr(s["reserved"]), ptr(s["table_out"]), ptr(s["ctx_out"]), ptr(s["missing"]),
                                   ptr(s["workspace"]), need), (s["table_out"], s["ctx_out"], s["missing"]) + _pool_values(s)
    if c["kind"] == "keep":
        return lib.kv_paged_keep, (pkg.capi.paged_layers(caches), len(caches), ptr(s["keep"]), ptr(s["n_keep"]), s["tokens"], s["max_new"], ptr(s["ctx_out"])), (s["ctx_out"],) + _pool_values(s)
    cache, n_q, n_kv, dim = caches[0], c["n_q"], c["n_kv"], c["dim"]
    if c["kind"] == "append":
        ld, at = (n_q + 2 * n_kv) * dim, s["qkv"].data_ptr()
        return lib.qk_norm_rope_kv_paged_at, (cache, at, at + 2 * n_q * dim, at + 2 * (n_q + n_kv) * dim, ptr(s["norm_w"][0]), ptr(s["norm_w"][1]), ptr(s["cos"]), ptr(s["sin"]), s["cos"].shape[0],
                                              ptr(s["positions"]), c["axes"], s["positions"].stride(0), ptr(s["axis"]), ptr(s["q_out"]), n_q, s["tokens"], ld, ld, ld, EPS), (s["q_out"],) + _pool_values(s)
    need = lib.attention_paged_tree_workspace_bytes(cache, n_q, s["tokens"], s["max_new"], s["max_ctx"], c["window"], c["sinks"])
    s["workspace"] = space(need)
    ld = n_q * dim
    return lib.attention_paged_tree, (cache, ptr(s["q"]), ptr(s["y"]), ptr(s["seen"]), s["seen"].shape[1], ptr(s["workspace"]), need, n_q, s["tokens"], s["max_new"], s["max_ctx"],
                                      c["window"], c["sinks"], ld, ld), s["y"]


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _bound(state)
        entry, args, out = state["call"]
        status = entry(*args)
        if status:
            raise RuntimeError(f"{state['case']['kind']}: {status}")
        return out
    return {"tree": _tree_plain, "append": _append_plain, "keep": _keep_plain, "fork": _fork_plain, "beam": _beam_plain}[state["case"]["kind"]](state)


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


def _rows64(s, name, seq, n):
    """The first n rows of a sequence, [row][kv head][dim]."""
    page = s["case"]["page"]
    pos = torch.arange(n, device=s["table"].device)
    at = s["table"][seq].long()[pos // page]
    x = s[name][0][at, :, pos % page]
    if s["case"]["cache"] == "bf16":
        return x.double()
    return _table(s["case"]["cache"]).to(x.device)[x.long()] * _two(s[name + "_scale"][0][at, :, pos % page].long() - 127)[..., None]


def _codes64(x, cache):
    """Code values (not yet times their power of two) and powers of two of rows in 64 bits."""
    _, _, top, largest, bits, least = CACHES[cache]
    amax = x.abs().amax(-1)
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -140) / largest))
    e = torch.where(amax > largest * _two(e), e + 1, torch.where(amax <= largest * _two(e - 1), e - 1, e)).clamp(-100, 127 - top)
    y = x * _two(-e)[..., None]
    step = _two(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** least))).clamp(min=least) - bits)
    return (torch.round(y / step) * step).clamp(-largest, largest), _two(e)


def _append64(case, s):
    new, ctx = lengths(case)
    n_q, n_kv, dim, page, dev = case["n_q"], case["n_kv"], case["dim"], case["page"], s["table"].device
    fp8 = case["cache"] != "bf16"
    pools = {name: _table(case["cache"]).to(dev)[s[name].long()] if fp8 else s[name].double() for name in ("k", "v")}
    scales = {name: _two(s[name + "_scale"].long() - 127) if fp8 else None for name in ("k", "v")}
    q_out = torch.zeros(s["tokens"], n_q, dim, dtype=torch.float64, device=dev)
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    begin = 0
    for i, (n, c) in enumerate(zip(new, ctx)):
        x = s["qkv"][begin:begin + n].double().view(n, -1, dim)
        by = torch.empty(n, dim // 2, dtype=torch.complex128, device=dev)
        for a in range(case["axes"]):
            mine = torch.ones(dim // 2, dtype=torch.bool, device=dev) if s["axis"] is None else s["axis"] == a
            by[:, mine] = turn[s["positions"][a, begin:begin + n].long()][:, mine]
        turned = []
        for part, w in ((x[:, :n_q], s["norm_w"][0]), (x[:, n_q:n_q + n_kv], s["norm_w"][1])):
            if w is not None:
                part = part / torch.sqrt((part * part).sum(-1, keepdim=True) / dim + EPS) * w.double()
            z = torch.complex(part[..., :dim // 2], part[..., dim // 2:]) * by[:, None]
            turned.append(torch.cat([z.real, z.imag], -1))
        q_out[begin:begin + n] = turned[0]
        pos = torch.arange(c - n, c, device=dev)
        where = s["table"][i].long()[pos // page]
        for name, rows in (("k", turned[1]), ("v", x[:, n_q + n_kv:])):
            if fp8:
                pools[name][0][where, :, pos % page], scales[name][0][where, :, pos % page] = _codes64(rows, case["cache"])
            else:
                pools[name][0][where, :, pos % page] = rows
        begin += n
    return (q_out, pools["k"], pools["v"]) + ((scales["k"], scales["v"]) if fp8 else ())


def _tree64(case, s):
    new, ctx = lengths(case)
    n_q, dim, dev = case["n_q"], case["dim"], s["table"].device
    group = n_q // case["n_kv"]
    y = torch.zeros(s["tokens"], n_q, dim, dtype=torch.float64, device=dev)
    begin = 0
    for i, (n, c) in enumerate(zip(new, ctx)):
        behind = c - n
        words = s["seen"][begin:begin + n].cpu()
        hidden = torch.ones(n, c, dtype=torch.bool)
        for t in range(n):
            line = [j for j in range(n) if int(words[t, j // 64]) >> (j % 64) & 1]
            hidden[t, :behind] = False
            if case["window"]:
                hidden[t, min(case["sinks"], behind):max(min(case["sinks"], behind), behind + len(line) - 1 - case["window"] + 1)] = True
            hidden[t, [behind + j for j in line]] = False
        hidden = hidden.to(dev)
        k, v = (_rows64(s, name, i, c) for name in ("k", "v"))
        for h in range(n_q):
            score = s["q"][begin:begin + n, h].double() @ k[:, h // group].t().contiguous() / math.sqrt(dim)
            y[begin:begin + n, h] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v[:, h // group].contiguous()
        begin += n
    return y


def _beam64(case, s):
    groups, beams, vocab, n_out = (case[k] for k in ("groups", "beams", "vocab", "n_out"))
    out = torch.empty(groups, n_out, dtype=torch.float64, device=s["score"].device)
    for i in range(groups):
        mine = slice(i * beams, (i + 1) * beams)
        total = s["score"][mine].double()[:, None] + torch.log_softmax(s["logits"][mine, :vocab].double(), 1)
        for b in range(beams):
            if int(s["last"][i * beams + b]) == s["eos"]:
                total[b] = -math.inf
                total[b, s["eos"]] = s["score"][i * beams + b].double()
        out[i] = torch.sort(total.flatten(), descending=True).values[:n_out]
    return None, None, out.flatten()


def exact(case, seed):
    if case["kind"] in ("keep", "fork"):
        return None                                                 # rows are moved as they are
    return {"tree": _tree64, "append": _append64, "beam": _beam64}[case["kind"]](case, prepare(case, seed))
