"""A small batch on a paged cache and its operators in 64 bits, for the tests."""
import math

import numpy as np

BF16, E4M3, E5M2 = 3, 4, 5
TOP = {E4M3: 8, E5M2: 15}               # exponent of the largest value, 1.75 * 2^TOP
BITS = {E4M3: 3, E5M2: 2}               # mantissa bits
LEAST = {E4M3: -6, E5M2: -14}           # exponent of the smallest normal value
EPS = 1e-6


def to_bf16(x):
    """Nearest-even BF16 bits of FP32 values."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(np.asarray(x, dtype=np.float32)), np.uint16(0x7FC0), r)


def from_bf16(b):
    return (np.ascontiguousarray(b).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def code_values(kind):
    """The value of each of the 256 codes."""
    code = np.arange(256)
    field, fraction = code % 128 >> BITS[kind], code % (1 << BITS[kind])
    value = np.where(field == 0, fraction * 2.0 ** (LEAST[kind] - BITS[kind]), (1 + fraction * 2.0 ** -BITS[kind]) * 2.0 ** (field - 1.0 + LEAST[kind]))
    if kind == E4M3:
        value[code % 128 == 127] = np.nan
    else:
        value[code % 128 == 124], value[code % 128 > 124] = np.inf, np.nan
    return np.where(code >= 128, -value, value)


def quantize(rows, kind):
    """Values of the codes (before their power of two) and exponents of rows in 64 bits."""
    finite = np.where(np.isfinite(rows), np.abs(rows), 0.0)
    amax = finite.max(-1)
    mantissa, exponent = np.frexp(amax)
    e = np.clip(np.where(amax > 0, exponent - 1 - TOP[kind] + (2 * mantissa > 1.75), -100), -100, 127 - TOP[kind])
    y = rows * 2.0 ** -e[..., None].astype(np.float64)
    size = np.where(np.isfinite(y), np.abs(y), 0.0)
    step = 2.0 ** (np.maximum(np.frexp(size)[1] - 1, LEAST[kind]) - BITS[kind])
    largest = 1.75 * 2.0 ** TOP[kind]
    with np.errstate(invalid="ignore"):
        codes = np.where(np.isfinite(y), np.clip(np.round(y / step) * step, -largest, largest), np.nan if kind == E4M3 else y)
    return codes, e


class Batch:
    """new[s] new tokens and ctx[s] rows of each sequence; pages of a pool in any order, `spare` of which belong to nobody."""

    def __init__(self, seed, kind, dim, n_kv, page, new, ctx, spare=3, stale=True, table_extra=2):
        rng = self.rng = np.random.default_rng(seed)
        self.kind, self.dim, self.n_kv, self.page, self.new, self.ctx = kind, dim, n_kv, page, list(new), list(ctx)
        self.n_seqs, self.tokens = len(new), sum(new)
        pages = [-(-c // page) for c in ctx]
        self.n_pages, self.table_stride = sum(pages) + spare, max(pages + [1]) + table_extra
        order = rng.permutation(self.n_pages)
        self.table = rng.integers(0, self.n_pages, (self.n_seqs, self.table_stride)).astype(np.int32)
        for s, n in enumerate(pages):
            self.table[s, :n] = order[sum(pages[:s]):sum(pages[:s]) + n]
        self.ctx_len = np.array(ctx, dtype=np.int32)
        self.seq_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        shape = (self.n_pages, n_kv, page, dim)
        rows = {"k": rng.standard_normal(shape) * (1 + 2 * (rng.random((n_kv, 1, dim)) < 0.05)), "v": rng.standard_normal(shape) * 0.7}
        self.pool, self.scale = {}, {"k": None, "v": None}
        for name, x in rows.items():
            if kind == BF16:
                self.pool[name] = to_bf16(x)
            else:
                self.set_codes(name, *quantize(x, kind))

    def set_codes(self, name, values, e):
        table = code_values(self.kind)
        order = np.argsort(table[:128][np.isfinite(table[:128])])
        known = table[:128][order]
        codes = order[np.searchsorted(known, np.abs(values))].astype(np.uint8) | np.where(np.signbit(values), 128, 0).astype(np.uint8)
        self.pool[name], self.scale[name] = codes, (e + 127).astype(np.uint8)

    def values(self, name):
        """The pool's values in 64 bits, [page][kv head][row][dim]."""
        if self.kind == BF16:
            return from_bf16(self.pool[name])
        return code_values(self.kind)[self.pool[name]] * 2.0 ** (self.scale[name].astype(np.float64) - 127)[..., None]

    def rows(self, name, s, n=None):
        """Rows 0 .. n - 1 of sequence s, [kv head][row][dim]."""
        pos = np.arange(self.ctx[s] if n is None else n)
        return self.values(name)[self.table[s, pos // self.page], :, pos % self.page].transpose(1, 0, 2)

    def slots(self):
        """(token, sequence, position) of every new token that has one."""
        return [(int(self.seq_start[s]) + i, s, self.ctx[s] - self.new[s] + i) for s in range(self.n_seqs) for i in range(self.new[s]) if self.ctx[s] - self.new[s] + i >= 0]

    # ---- on the device
    def upload(self, torch, dev):
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int16) if a.dtype == np.uint16 else np.ascontiguousarray(a)).to(dev)  # noqa: E731
        self.dev = {name: put(self.pool[name]) for name in ("k", "v")}
        for name in ("k", "v"):
            self.dev[name + "_scale"] = None if self.kind == BF16 else put(self.scale[name])
        for name in ("table", "ctx_len", "seq_start"):
            self.dev[name] = put(getattr(self, name))
        return self

    def descriptor(self, pkg, **other):
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        d = self.dev
        args = dict(type=self.kind, head_dim=self.dim, n_kv_heads=self.n_kv, page_size=self.page, n_pages=self.n_pages, k=p(d["k"]), v=p(d["v"]), page_table=p(d["table"]), table_stride=self.table_stride,
                    ctx_len=p(d["ctx_len"]), seq_start=p(d["seq_start"]), n_seqs=self.n_seqs, k_scale=p(d["k_scale"]), v_scale=p(d["v_scale"]))
        return pkg.capi.make_paged_kv(**(args | other))

    def download(self, name):
        out = self.dev[name].cpu().numpy()
        return out.view(np.uint16) if out.dtype == np.int16 else out


def norm_rope(x, w, cos, sin):
    """x [heads][dim] in 64 bits; w, cos, sin may be None."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w
    if cos is None:
        return x
    half = x.shape[-1] // 2
    lo, hi = x[..., :half], x[..., half:]
    return np.concatenate([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def seen_by(pos, n, window, n_sink):
    key = np.arange(n)
    return (key <= pos) & ((key > pos - window) | (key < n_sink) if window else True)


def attend(batch, q, n_q, window=0, n_sink=0, rows=None):
    """y, and what it may be off by: probabilities rounded to BF16 (half a step, 2^-8 of each), the result likewise, and the FP32 sums of the scores
    (dim + 4 roundings of 2^-24 of the sum of magnitudes, which move a probability and the sum of all by as much).  q [tokens][n_q][dim] in 64 bits."""
    group, dim = n_q // batch.n_kv, batch.dim
    y, bound = np.zeros((batch.tokens, n_q, dim)), np.zeros((batch.tokens, n_q, dim))
    for s in range(batch.n_seqs):
        if not batch.new[s]:
            continue
        k, v = (batch.rows(name, s) if rows is None else rows[name][s] for name in ("k", "v"))
        for t, of, pos in batch.slots():
            if of != s:
                continue
            seen = seen_by(pos, k.shape[1], window, n_sink)
            if not seen.any():
                continue
            for h in range(n_q):
                kk, vv = k[h // group][seen], v[h // group][seen]
                score = kk @ q[t, h] / math.sqrt(dim)
                w = np.exp(score - score.max())
                w /= w.sum()
                off = 2 * (dim + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[t, h])).max() / math.sqrt(dim) + 2.0 ** -20
                y[t, h] = w @ vv
                bound[t, h] = (2.0 ** -8 + off) * (w @ np.abs(vv)) + (2.0 ** -8 + off) * np.abs(y[t, h]) + 2.0 ** -126
    return y, bound
