"""Sequences that branch, in 64 bits or whole numbers, for the tests: trees of new tokens, kept rows, forked batches, beams."""
import copy
import math

import numpy as np

from paged_util import BF16, quantize, to_bf16


def trees(rng, new):
    """Per sequence which of its new tokens each sees: those that it descends from, and itself, [n][n]."""
    out = []
    for n in new:
        line = np.zeros((n, n), dtype=bool)
        for i in range(n):
            if i: line[i] = line[rng.integers(max(0, i - 5), i)]
            line[i, i] = True
        out.append(line)
    return out


def bits(seen, stride, rng=None):
    """Words of all tokens, [token][stride]; with rng the bits behind a sequence's number of new tokens hold anything."""
    tokens = sum(len(s) for s in seen)
    flat = np.zeros((tokens, 64 * stride), dtype=bool) if rng is None else rng.random((tokens, 64 * stride)) < 0.5
    at = 0
    for s in seen:
        flat[at:at + len(s), :len(s)] = s
        at += len(s)
    return np.packbits(flat, axis=1, bitorder="little").view(np.uint64).view(np.int64)


def tree_keys(n_rows, first, seen, window, n_sink):
    """Which rows of the cache a token sees whose bits are `seen`, the first new token at position `first`."""
    key = np.arange(n_rows)
    pos = first + max(int(seen.sum()) - 1, 0)
    in_front = (key < first) & ((key > pos - window) | (key < n_sink) if window else True)
    j = key - first
    return in_front | ((j >= 0) & (j < len(seen)) & seen[np.clip(j, 0, len(seen) - 1)])


def tree_attend(b, q, n_q, seen, window=0, n_sink=0, rows=None, lost=None):
    """y and what it may be off by: probabilities rounded to BF16 (half a step, 2^-8 of each), the result likewise, and the FP32 sums of the scores (dim + 4 roundings of 2^-24 of the sum of
    magnitudes, which move a probability and the sum of all by as much).  lost: rows without a page, per sequence."""
    group, dim = n_q // b.n_kv, b.dim
    y, bound = np.zeros((b.tokens, n_q, dim)), np.zeros((b.tokens, n_q, dim))
    for s in range(b.n_seqs):
        if not b.new[s]: continue
        first, t0 = b.ctx[s] - b.new[s], int(b.seq_start[s])
        k, v = (b.rows(name, s) if rows is None else rows[name][s] for name in ("k", "v"))
        for i in range(b.new[s]):
            see = tree_keys(b.ctx[s], first, seen[s][i], window, n_sink)
            if lost is not None: see &= ~lost[s]
            if first + i < 0 or not see.any(): continue
            for h in range(n_q):
                kk, vv = k[h // group][see], v[h // group][see]
                score = kk @ q[t0 + i, h] / math.sqrt(dim)
                w = np.exp(score - score.max())
                w /= w.sum()
                off = 2 * (dim + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[t0 + i, h])).max() / math.sqrt(dim) + 2.0 ** -20
                y[t0 + i, h] = w @ vv
                bound[t0 + i, h] = (2.0 ** -8 + off) * (w @ np.abs(vv)) + (2.0 ** -8 + off) * np.abs(y[t0 + i, h]) + 2.0 ** -126
    return y, bound


class Layers:
    """The caches of n layers: batch b's tables and lengths, pools of their own."""

    def __init__(self, b, n, torch, dev):
        self.b, self.batches = b, []
        for i in range(n):
            other = copy.copy(b)
            other.pool, other.scale = dict(b.pool), dict(b.scale)
            if i:
                for name in ("k", "v"):
                    x = b.rng.standard_normal(b.pool[name].shape)
                    if b.kind == BF16: other.pool[name] = to_bf16(x)
                    else: other.set_codes(name, *quantize(x, b.kind))
            other.upload(torch, dev)
            if i:
                for name in ("table", "ctx_len", "seq_start"): other.dev[name] = self.batches[0].dev[name]
            self.batches.append(other)
        b.dev = self.batches[0].dev

    def caches(self, pkg, **other):
        return pkg.capi.paged_layers([x.descriptor(pkg, **other) for x in self.batches])

    def pools(self):
        """Per layer {name: what lies in memory}."""
        names = ("k", "v") if self.b.kind == BF16 else ("k", "v", "k_scale", "v_scale")
        return [{name: x.download(name).copy() for name in names} for x in self.batches]


def fork(table, ctx, page, n_pages, parent, rows, grow, reserved):
    """(table, lengths, missing pages, copies as (page, new page, rows))."""
    n_seqs, stride = table.shape
    ok = lambda p: 0 <= p < n_pages  # noqa: E731
    plan, whole, last = [], set(np.flatnonzero(reserved).tolist()) if reserved is not None else set(), {}
    for s, p in enumerate(parent):
        have = min(max(int(ctx[p]), 0), stride * page) if 0 <= p < n_seqs else 0
        r = have if rows is None else min(max(int(rows[s]), 0), have)
        total = min(r + max(int(grow[s]), 0), stride * page)
        old = [int(x) if ok(x) else -1 for x in table[p, :-(-r // page)]] if r else []
        whole |= {x for x in old[:r // page] if x >= 0}
        if r % page and old[-1] >= 0: last.setdefault(old[-1], s)
        plan.append((r, total, old))
    held = whole | set(last)
    free = iter([x for x in range(n_pages) if x not in held])
    out, copies, missing = np.full((len(parent), stride), -1, dtype=np.int32), [], 0

    def take():
        nonlocal missing
        page = next(free, -1)
        missing += page < 0
        return page
    for s, (r, total, old) in enumerate(plan):
        mine = list(old)
        if r % page and old[-1] >= 0 and (old[-1] in whole or last[old[-1]] != s):
            mine[-1] = take()
            if mine[-1] >= 0: copies.append((old[-1], mine[-1], r % page))
        mine += [take() for _ in range(-(-total // page) - len(mine))]
        out[s, :len(mine)] = mine
    return out, np.array([t for _, t, _ in plan], dtype=np.int32), missing, copies


def beam(x, score, ended, eos, n_groups, n_beams, n_out):
    """(rows, tokens, totals) of the best, x [row][vocab] in 64 bits."""
    vocab = x.shape[1]
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    total, order = np.full(x.shape, -np.inf), np.zeros(x.shape)
    for r in range(len(x)):
        if not np.isfinite(score[r]): continue
        if ended[r]:
            if 0 <= eos < vocab: total[r, eos], order[r, eos] = score[r], 1
            continue
        m = x[r].max()
        order[r] = x[r]
        if m == -np.inf: continue
        with np.errstate(invalid="ignore"):
            d = np.where(x[r] == m, 0.0, x[r] - m)
        total[r] = score[r] + (d - np.log(np.exp(d).sum()))
    rows, tokens, totals = [], [], []
    for g in range(n_groups):
        t, o = (a[g * n_beams:(g + 1) * n_beams].ravel() for a in (total, order))
        best = np.lexsort((np.arange(t.size) % vocab, -o, np.arange(t.size) // vocab, -t))[:n_out]
        rows.append(g * n_beams + best // vocab)
        tokens.append(best % vocab)
        totals.append(t[best])
    return np.array(rows), np.array(tokens), np.array(totals)
