"""Log probabilities of given tokens, entropy and the most likely tokens (tq_token_logprobs) against 64 bits: every type, strides and slices,
vocabularies of one token to the largest, ties, rows without a logit, infinities and NaN, refusals."""
import numpy as np
import pytest

from util import bf16_round

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -24                      # half a step of f32, relative


@pytest.fixture(scope="module")
def dev():
    import tang_b200

    d = tang_b200.QuantComputeDevice(0)
    yield d
    d.close()


def reference(x, tokens, top):
    """x [rows, V] in 64 bits.  (log p of the tokens, entropy, ids, log p of the ids, how much of a row is not its largest logits)"""
    m = x.max(1, keepdims=True)
    d = x - m
    e = np.exp(d)
    lead = (d == 0).sum(1)
    rest = np.where(d == 0, 0, e).sum(1)
    log_s = np.log(lead) + np.log1p(rest / lead)
    with np.errstate(invalid="ignore"):
        h = log_s - np.where(e > 0, d * e, 0).sum(1) / (lead + rest)
    lp = d - log_s[:, None]
    with np.errstate(over="ignore"):
        lp[np.isneginf(lp.astype(np.float32))] = -np.inf      # (too far from zero for an f32)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return np.take_along_axis(lp, tokens, 1), h, ids, np.take_along_axis(lp, ids, 1), rest / (lead + rest)


def close(got, want, rest, V):
    """A log probability is (x - m) - log S: a rounding of each difference, and log S as exact as the sum of the other terms, in which a thread adds
    at most V / 64 terms one after the other, each with four roundings of its own.  An exponential below 2^-126, the smallest normal f32, counts as zero:
    V of them are less than V 2^-126."""
    tol = 4 * STEP * np.abs(want) + (V / 64 + 64) * STEP * rest[:, None] + V * 2.0 ** -126
    fin = np.isfinite(want)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    assert (np.abs(got - want)[fin] <= tol[fin]).all(), (np.abs(got - want)[fin] / tol[fin]).max()


def run(dev, x, tokens, top, slices=1, bf16=False, pad=0, entropy=True):
    """x [rows, V] f32, laid out [slices][rows][cols + pad] with NaN in the padding."""
    import tang_b200 as tb

    rows, V = x.shape
    cols = V // slices
    a = np.full((slices, rows, cols + pad), np.nan, np.float32)
    a[:, :, :cols] = x.reshape(rows, slices, cols).transpose(1, 0, 2)
    buf = dev.upload(bf16_round(a)[0], tb.BF16) if bf16 else dev.upload(a)
    if bf16 and pad:                   # (the conversion of NaN is not what this tests)
        raw = bf16_round(np.nan_to_num(a))[0].reshape(a.shape)
        raw[:, :, cols:] = 0x7FC0
        buf = dev.upload(raw, tb.BF16)
    got = dev.token_logprobs(buf, rows, cols, dev.upload(tokens.astype(np.int32), tb.I32), n_tokens=tokens.shape[1], top=top, slices=slices,
                             ld=cols + pad if pad else 0, entropy=entropy)
    dev.sync()
    return (got.logprobs.to_vec().reshape(rows, -1), got.entropy.to_vec() if entropy else None,
            got.top_ids.to_vec().reshape(rows, top) if top else np.zeros((rows, 0), int),
            got.top_logprobs.to_vec().reshape(rows, top) if top else np.zeros((rows, 0)))


def check(dev, x, tokens, top, **how):
    rows, V = x.shape
    x64 = (bf16_round(x)[1] if how.get("bf16") else x).astype(np.float64)
    lp, h, ids, top_lp = run(dev, x, tokens, top, **how)
    want_lp, want_h, want_ids, want_top, rest = reference(x64, tokens, top)
    close(lp, want_lp, rest, V)
    if h is not None:
        # every term of the entropy is positive: its relative error is that of the sums; and (m - x) exp(x - m) falls with m - x behind 1: the terms whose
        # exponential is below 2^-126, m - x > 87, and so counts as zero are below 88 * 2^-126 each
        assert (np.abs(h - want_h) <= (V / 64 + 64) * STEP * want_h + V * 88 * 2.0 ** -126).all()
    assert np.array_equal(ids, want_ids)
    close(top_lp, want_top, rest, V)


@pytest.mark.parametrize("rows,V,slices,pad,top,n_tokens", [
    (1, 1, 1, 0, 1, 1), (3, 2, 2, 0, 2, 2), (2, 7, 1, 0, 7, 3), (5, 64, 1, 0, 64, 1), (1, 1000, 1, 0, 5, 1), (4, 1003, 1, 5, 20, 2), (3, 4 * 251, 4, 0, 8, 1),
    (3, 4 * 251, 4, 3, 64, 1), (200, 517, 1, 0, 3, 1), (2, 32000, 1, 0, 20, 1), (150, 8013, 3, 0, 20, 1), (7, 128256, 1, 0, 20, 4), (1, 128256, 1, 0, 64, 1),
    (33, 128256, 8, 0, 1, 1), (400, 3000, 2, 1, 0, 1), (1, 262147, 1, 0, 40, 1), (2, 128256, 4, 0, 0, 1)])
@pytest.mark.parametrize("bf16", [False, True])
def test_against_64_bits(dev, rows, V, slices, pad, top, n_tokens, bf16):
    rng = np.random.default_rng(rows * 31 + V)
    x = (rng.standard_normal((rows, V)) * 2.5).astype(np.float32)
    x[np.arange(rows), rng.integers(0, V, rows)] = rng.uniform(0, 25, rows)
    check(dev, x, rng.integers(0, V, (rows, n_tokens)), top, slices=slices, bf16=bf16, pad=pad)


@pytest.mark.parametrize("kind", ["equal", "two values", "ascending", "descending", "one finite", "few finite", "far apart", "large", "signed zeros", "sure", "blocks", "lowest", "mostly lowest", "millions", "huge"])
@pytest.mark.parametrize("V,slices", [(90, 1), (5000, 1), (4 * 5003, 4), (128256, 1)])
def test_rows_that_are_hard_to_order_or_to_add(dev, kind, V, slices):
    rng = np.random.default_rng(V)
    rows, top = 5, 20
    x = rng.standard_normal((rows, V)).astype(np.float32)
    if kind == "equal":
        x[:] = 1.25
    elif kind == "two values":
        x[:] = np.where(rng.random((rows, V)) < 0.3, 2.0, 1.0)
    elif kind == "ascending":
        x[:] = np.linspace(-3, 3, V)
    elif kind == "descending":
        x[:] = np.linspace(3, -3, V)
    elif kind == "one finite":
        x[:] = -np.inf
        x[np.arange(rows), rng.integers(0, V, rows)] = 3
    elif kind == "few finite":
        x[rng.random((rows, V)) < 1 - 12 / V] = -np.inf
        x[:, V // 2] = 1
    elif kind == "far apart":
        x *= 1000
    elif kind == "large":
        x = (x + 30000).astype(np.float32)
    elif kind == "signed zeros":
        x[:] = np.where(rng.random((rows, V)) < 0.5, 0.0, -0.0)
    elif kind == "sure":
        x[np.arange(rows), rng.integers(0, V, rows)] = 40
    elif kind == "lowest":             # what masks are made of
        x[:] = np.finfo(np.float32).min
        x[1, :V // 2] = -np.inf
        x[2, 1::2] = 2e30
    elif kind == "mostly lowest":
        x[rng.random((rows, V)) < 1 - 12 / V] = np.finfo(np.float32).min
        x[0, V // 2] = np.finfo(np.float32).max
        x[3, V // 3:] = -np.inf
    elif kind == "millions":           # steps of 1/8 between neighbours
        x += np.array([2 ** 20 - 2, 2 ** 20 + 5, -2 ** 20, -2 ** 20 - 3, 2 ** 23])[:, None]
    elif kind == "huge":
        x *= 1e37
    elif kind == "blocks":             # the largest ones side by side, over and over the same
        x[:, V // 3:V // 3 + min(3000, V // 3)] = 7.5
        x[:, V - 2] = 7.5
    check(dev, x, rng.integers(0, V, (rows, 3)), top, slices=slices)


def test_tokens_that_are_none_and_rows_without_numbers(dev):
    V = 700
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, V)).astype(np.float32)
    x[1] = -np.inf
    x[2, 33] = np.nan
    x[3, 5] = np.inf
    x[4] = np.nan
    x[5, 10:] = np.nan
    tokens = np.array([[3, -1, V, 2 ** 31 - 1, -2 ** 31]] * 6)
    lp, h, ids, top_lp = run(dev, x, tokens, 12)
    assert (lp[:, [1, 4]] == 0).all() and np.isnan(lp[:, [2, 3]]).all()
    want = reference(x[:1].astype(np.float64), tokens[:1, :1], 12)
    assert abs(lp[0, 0] - want[0][0, 0]) < 1e-5 and np.array_equal(ids[0], want[2][0])
    assert lp[1, 0] == -np.inf and h[1] == 0 and np.array_equal(ids[1], np.arange(12)) and (top_lp[1] == -np.inf).all()
    assert np.isnan(lp[2:, 0]).all() and np.isnan(h[2:]).all() and np.isnan(top_lp[2:]).all()
    assert np.array_equal(ids[2], np.argsort(-np.where(np.isnan(x[2]), -np.inf, x[2]), kind="stable")[:12])
    assert ids[3, 0] == 5 and (ids[4] == -1).all()
    assert np.array_equal(ids[5, :10], np.argsort(-x[5, :10], kind="stable")) and (ids[5, 10:] == -1).all()


def test_any_alignment_and_rows_behind_the_last(dev):
    """Logits that start at any element of a larger buffer; results behind the last row stay as they were."""
    import tang_b200 as tb

    rng = np.random.default_rng(2)
    V, rows = 4099, 3
    x = rng.standard_normal((rows, V)).astype(np.float32)
    want = reference(x.astype(np.float64), np.zeros((rows, 1), int), 9)
    for bf16 in (False, True):
        size = 2 if bf16 else 4
        ref = reference(bf16_round(x)[1].astype(np.float64), np.zeros((rows, 1), int), 9) if bf16 else want
        for off in range(9):
            a = np.full(off + rows * V, 50.0, np.float32)
            a[off:] = x.reshape(-1)
            whole = dev.upload(bf16_round(a)[0], tb.BF16) if bf16 else dev.upload(a)
            part = tb.Buffer(dev, whole.ptr + off * size, rows * V, whole.dtype, owns=False)
            out = tb.TokenLogprobs(*(dev.upload(np.full(n, -7, np.float32 if i != 2 else np.int32), tb.F32 if i != 2 else tb.I32)
                                     for i, n in enumerate((rows + 2, rows + 2, rows * 9 + 2, rows * 9 + 2))))
            dev.token_logprobs(part, rows, V, dev.upload(np.zeros(rows, np.int32), tb.I32), top=9, out=out)
            dev.sync()
            got = [b.to_vec() for b in (out.logprobs, out.entropy, out.top_ids, out.top_logprobs)]
            assert all((g[-2:] == -7).all() for g in got)
            close(got[0][:rows, None], ref[0], ref[4], V)
            assert np.array_equal(got[2][:-2].reshape(rows, 9), ref[2])


def test_the_same_bits_again_and_from_a_graph(dev):
    import tang_b200 as tb

    rng = np.random.default_rng(3)
    rows, V = 9, 50001
    x = [rng.standard_normal((rows, V)).astype(np.float32) * 3 for _ in range(2)]
    tokens = dev.upload(rng.integers(0, V, rows).astype(np.int32), tb.I32)
    buf = dev.upload(x[0])
    read = lambda o: [b.to_vec() for b in (o.logprobs, o.entropy, o.top_ids, o.top_logprobs)]
    out = dev.token_logprobs(buf, rows, V, tokens, top=20)
    first = read(out)
    dev.begin_capture()
    dev.token_logprobs(buf, rows, V, tokens, top=20, out=out)
    g = dev.end_capture()
    dev.upload_into(buf, x[1])
    g.launch()
    dev.sync()
    second = read(out)
    dev.upload_into(buf, x[0])
    g.launch()
    dev.sync()
    assert all(np.array_equal(a, b) for a, b in zip(first, read(out)))
    g.free()
    fresh = dev.token_logprobs(dev.upload(x[1]), rows, V, tokens, top=20)
    dev.sync()
    assert all(np.array_equal(a, b) for a, b in zip(second, read(fresh)))


def test_two_handles_with_streams_of_their_own(dev):
    import tang_b200 as tb

    other = tb.QuantComputeDevice(0)
    rng = np.random.default_rng(4)
    x = rng.standard_normal((2, 64, 9001)).astype(np.float32)
    bufs = [d.upload(a) for d, a in zip((dev, other), x)]
    outs = [d.token_logprobs(b, 64, 9001, top=5) for _ in range(5) for d, b in zip((dev, other), bufs)]
    dev.sync()
    other.sync()
    for i, o in enumerate(outs):
        assert np.array_equal(o.top_ids.to_vec().reshape(64, 5), np.argsort(-x[i % 2], axis=1, kind="stable")[:, :5])
    del outs, bufs
    other.close()


def test_refusals(dev):
    import ctypes as C

    import tang_b200 as tb

    x, tok = dev.upload(np.zeros(100, np.float32)), dev.upload(np.zeros(10, np.int32), tb.I32)
    for kw in ({"rows": 11, "cols": 10}, {"rows": 10, "cols": 10, "tokens": tok, "n_tokens": 2}, {"rows": 1, "cols": 100, "top": 65}, {"rows": 10, "cols": 10, "top": 11},
               {"rows": 1, "cols": 0}, {"rows": 2, "cols": 10, "ld": 9}, {"rows": 1, "cols": 10, "slices": 0}):
        with pytest.raises(tb.TangqError):
            dev.token_logprobs(x, **kw)
    with pytest.raises(tb.TangqError):
        dev.token_logprobs(tok, 1, 10)                       # ints are no logits
    with pytest.raises(tb.TangqError):
        dev.token_logprobs(tb.Buffer(dev, x.ptr + 2, 10, tb.F32, owns=False), 1, 10)
    L = dev._L
    assert L.tq_token_logprobs(dev._ctx, C.c_void_p(x.ptr), tb.F32, 0, 1, 1, 10, None, 1, 0, None, None, None, None) == tb._lib.TQ_EINVAL
    assert L.tq_token_logprobs(dev._ctx, C.c_void_p(x.ptr), tb.F32, 0, 1, 1, 10, None, 0, 1, None, None, None, None) == tb._lib.TQ_EINVAL
    assert L.tq_token_logprobs(dev._ctx, None, tb.F32, 0, 1, 0, 10, None, 0, 0, None, None, None, None) == tb._lib.TQ_OK     # no rows
    dev.sync()


def test_vocabularies_whose_places_pass_32_bits_are_refused(dev):
    """Before anything is launched: there is no such row here."""
    import ctypes as C

    import tang_b200 as tb

    x, out = dev.upload(np.zeros(16, np.float32)), dev.alloc(1)
    for slices, cols in ((1, 2 ** 31 - 1), (1, 2 ** 31 - 2 ** 16 + 1), (2, 2 ** 30), (3, 715806038), (65535, 32768), (1, 2 ** 31), (2 ** 16, 1)):
        assert slices * cols > 2 ** 31 - 2 ** 16 or slices == 2 ** 16
        assert dev._L.tq_token_logprobs(dev._ctx, C.c_void_p(x.ptr), tb.BF16, 0, slices, 1, cols, None, 0, 0, None, C.c_void_p(out.ptr), None, None) == tb._lib.TQ_EINVAL
    dev.sync()
