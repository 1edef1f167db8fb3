"""Packed rows over a pool of pages, cache rows of 4 bits and attention over them as the interface defines them, in numpy."""
import numpy as np

from util import bf16_round

HD, BLOCK = 128, 32
BASE = 10000.0


def row_bytes(nkv):
    return -(-nkv * (HD // 2 + 2 * HD // BLOCK) // 16) * 16


def scales(x):
    """Of blocks [..., 32]: the smallest numbers of 5 significant bits that are not below the largest magnitude / 7."""
    x = np.abs(np.asarray(x, np.float64))
    amax = np.where(np.isnan(x).any(-1), np.inf, np.max(np.where(np.isnan(x), 0, x), -1))
    with np.errstate(invalid="ignore"):
        frac, e = np.frexp(amax / 7)
        s = np.ldexp(np.ceil(frac * 32) / 32, e)
    return np.where(amax < 2.0 ** -100, 0.0, np.where(amax < 2.0 ** 120, s, np.nan))


def pack(x):
    """f32 rows [n, nkv, 128] -> (bytes [n, row_bytes], the values that they stand for, f64)."""
    x = np.asarray(x, np.float32)
    n, nkv = x.shape[:2]
    b = x.reshape(n, nkv, HD // BLOCK, BLOCK)
    s = scales(b)
    with np.errstate(invalid="ignore", divide="ignore"):
        code = np.where(s[..., None] > 0, np.rint(b / s[..., None].astype(np.float32)), 0).astype(np.int64)
    assert np.abs(code).max(initial=0) <= 7
    u = (code + 8).astype(np.uint8).reshape(n, nkv * HD // 2, 2)
    out = np.zeros((n, row_bytes(nkv)), np.uint8)
    out[:, :nkv * HD // 2] = u[:, :, 0] | u[:, :, 1] << 4
    bits = (s.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    bits[np.isnan(s)] = 0x7FC0
    out[:, nkv * HD // 2:nkv * (HD // 2 + 8)] = bits.reshape(n, nkv * 4).view(np.uint8)
    return out, (code * s[..., None]).reshape(n, nkv, HD)


def tables(n_positions, base=BASE):
    """cos, sin f32 [n_positions, 64]."""
    a = np.arange(n_positions)[:, None] * base ** (-2.0 * np.arange(HD // 2) / HD)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def rotate(x, cos, sin):
    """f32 rows [n, heads, 128], neighbouring values a pair, each product and sum rounded to f32; cos, sin [n, 64]."""
    x0, x1 = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None], sin[:, None]
    out = np.empty_like(x)
    out[..., 0::2], out[..., 1::2] = x0 * c - x1 * s, x0 * s + x1 * c
    return out


def attend(q, k, v):
    """q [c, nh, 128] of the last c of the positions of k, v [n, nkv, 128]; returns (result, sum of the weights times the values' sizes) in 64 bits."""
    c, nh, _ = q.shape
    n, nkv, _ = k.shape
    qg = q.astype(np.float64).reshape(c, nkv, nh // nkv, HD).transpose(1, 0, 2, 3).reshape(nkv, -1, HD)
    k, v = (a.astype(np.float64).transpose(1, 0, 2) for a in (k, v))
    s = (qg @ k.transpose(0, 2, 1) / np.sqrt(HD)).reshape(nkv, c, nh // nkv, n)
    s = np.where((np.arange(n)[None] <= np.arange(n - c, n)[:, None])[None, :, None], s, -np.inf)
    e = np.exp(s - s.max(-1, keepdims=True))
    w = (e / e.sum(-1, keepdims=True)).reshape(nkv, -1, n)
    back = lambda a: a.reshape(nkv, c, nh // nkv, HD).transpose(1, 0, 2, 3).reshape(c, nh, HD)  # noqa: E731
    return back(w @ v), back(w @ np.abs(v))


class Sequences:
    """Sequences in a pool, `lens` positions each of which the last `counts` are packed rows; whatever is no row of theirs is NaN.
    `seqs`: their numbers in a larger pool."""

    def __init__(self, nh, nkv, P, lens, counts, seed, form, seqs=None, extra=3, k_size=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.P, self.form, self.lens, self.counts = nh, nkv, P, form, np.array(lens), np.array(counts)
        self.B, self.rows = len(lens), int(sum(counts))
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.order = np.arange(self.B) if seqs is None else np.array(seqs)
        self.n_seqs = int(self.order.max()) + 1
        held = -(-self.lens // P)
        self.ld = max(1, int(held.max(initial=0))) + 1
        self.n_pages = int(held.sum()) + extra
        free = rng.permutation(self.n_pages).tolist()
        self.tables = np.full((self.n_seqs, self.ld), -1, np.int32)
        self.lens_all = np.zeros(self.n_seqs, np.int32)
        for b, s in enumerate(self.order):
            self.tables[s, :held[b]] = [free.pop() for _ in range(held[b])]
            self.lens_all[s] = self.lens[b]
        self.refs = np.zeros(self.n_pages, np.int32)
        self.refs[self.tables[self.tables >= 0]] = 1
        self.q_bits, self.q = bf16_round((rng.standard_normal((self.rows, nh, HD)) * 1.5).astype(np.float32))
        # cache rows of all pages: raw (bf16 bits or bytes) and values
        self.raw, self.values = [], []
        held_rows = np.concatenate([self.places(b, range(n)) for b, n in enumerate(self.lens)]).astype(np.int64) if self.lens.sum() else np.zeros(0, np.int64)
        for size in (k_size, 1.0):
            x = (rng.standard_normal((len(held_rows), nkv, HD)) * size).astype(np.float32)
            if form == "q4":
                bits, val = pack(x)
                raw = np.full((self.n_pages * P, row_bytes(nkv)), 0xFF, np.uint8)
            else:
                bits, val = bf16_round(x)
                bits = bits.reshape(len(x), -1)
                raw = np.full((self.n_pages * P, nkv * HD), 0x7FC0, np.uint16)
            raw[held_rows] = bits
            values = np.full((self.n_pages * P, nkv, HD), np.nan)
            values[held_rows] = val
            self.raw.append(raw)
            self.values.append(values)

    def places(self, b, positions):
        pos = np.array(positions, np.int64)
        return self.tables[self.order[b], pos // self.P].astype(np.int64) * self.P + pos % self.P

    def new_places(self):
        return np.concatenate([self.places(b, range(n - c, n)) for b, (n, c) in enumerate(zip(self.lens, self.counts))]).astype(np.int64)

    def new_positions(self):
        return np.concatenate([np.arange(n - c, n) for n, c in zip(self.lens, self.counts)]).astype(np.int64)

    def put(self, dev, seqs=True):
        import tang_b200 as tb

        self.dev, self.tb = dev, tb
        self.state = [dev.upload(a, tb.I32) for a in (self.refs, self.tables, self.lens_all)]
        self.pool = tb.PagePool(dev, self.n_pages, self.P, self.n_seqs, self.ld, None, *self.state)
        dt = tb.U8 if self.form == "q4" else tb.BF16
        self.kb, self.vb = (dev.upload(a.reshape(-1), dt) for a in self.raw)
        self.qb = dev.upload(self.q_bits.reshape(-1), tb.BF16)
        self.seq_rows = dev.upload(self.starts, tb.I32) if not (self.counts == 1).all() else None
        self.seqs = dev.upload(self.order, tb.I32) if not np.array_equal(self.order, np.arange(self.B)) else None
        return self

    def prefill(self, max_len=None, out=None):
        return self.dev.gqa_prefill_paged(self.qb, self.kb, self.vb, self.pool, self.B, self.rows, self.nh, self.nkv, HD, max_len or max(1, int(self.lens.max())),
                                          seqs=self.seqs, seq_rows=self.seq_rows, out=out)

    def decode(self, max_len=None, out=None):
        return self.dev.gqa_decode_paged_q4(self.qb, self.kb, self.vb, self.pool, self.B, self.nh, self.nkv, HD, max_len or max(1, int(self.lens.max())),
                                            seqs=self.seqs, out=out)

    def reference(self):
        out, size = np.zeros((self.rows, self.nh, HD)), np.zeros((self.rows, self.nh, HD))
        for b, (n, c) in enumerate(zip(self.lens, self.counts)):
            if n and c:
                at, r = self.places(b, range(n)), slice(self.starts[b], self.starts[b + 1])
                out[r], size[r] = attend(self.q[r], self.values[0][at], self.values[1][at])
        return out, size


def widen(bits):
    return (np.asarray(bits).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def check_attention(got_bits, want, size, terms):
    """Scores: sums of 128 exact products in f32, and their exponentials, 2^-14 of the weights (as for the attention over pages of bf16).  Weights of one
    bf16 term are off by up to 2^-8 of themselves; divided by the sum of what they became, that is 2^-8 of |value - result| on the average, at
    most 2^-8 (size + |result|).  Two terms leave 2^-16.  The result's rounding to bf16 is 2^-8 of it."""
    got = widen(got_bits).reshape(want.shape)
    assert np.isfinite(got).all()
    off = 2.0 ** -14 * size + (2.0 ** -8 * (size + np.abs(want)) if terms == 1 else 2.0 ** -15 * size)
    tol = off + 2.0 ** -8 * (np.abs(want) + off) + 1e-30
    err = np.abs(got - want) / tol
    assert err.max(initial=0) <= 1, (err.max(), np.unravel_index(err.argmax(), err.shape))
