"""Prompts of different lengths over pages: packed rows appended to bf16 and 4-bit pages (tq_kv_append_paged) and read back (tq_kv_read_paged), causal
attention of packed rows (tq_gqa_prefill_paged) and decode attention over 4 bits (tq_gqa_decode_paged_q4), against 64 bits."""
import numpy as np
import pytest

from packed_util import HD, Sequences, check_attention, pack, rotate, row_bytes, tables, widen
from util import bf16_round

pytestmark = pytest.mark.gpu

# query heads, KV heads, page rows, lengths, new rows
ROWS = {
    "one token": (32, 8, 16, [1], [1]),
    "a page's end": (8, 2, 16, [16, 17, 32], [1, 1, 1]),
    "prompts": (16, 4, 32, [33, 7, 100, 1], [33, 7, 60, 1]),
    "nothing new of some": (8, 8, 16, [5, 40, 0, 18], [0, 40, 0, 3]),
    "odd heads": (15, 3, 64, [70, 130], [70, 5]),
    "one KV head": (8, 1, 128, [300], [171]),
    "many rows": (32, 8, 64, [700, 350, 129], [700, 350, 64]),
}


@pytest.fixture(scope="module")
def dev():
    import tang_b200

    d = tang_b200.QuantComputeDevice(0)
    yield d
    d.close()


def appended(s, dev, x, dtype, n_positions, seq_rows=True, rows=None, **kw):
    import tang_b200 as tb

    cos, sin = tables(n_positions)
    xb = dev.upload(x.reshape(-1), dtype)
    rows = s.rows if rows is None else rows
    return dev.kv_append_paged(xb, dev.upload(cos, tb.F32), dev.upload(sin, tb.F32), s.pool, s.kb, s.vb, s.B, rows, s.nh, s.nkv, HD, seqs=s.seqs,
                               seq_rows=s.seq_rows if seq_rows else None, **kw), cos, sin


@pytest.mark.parametrize("name", list(ROWS))
@pytest.mark.parametrize("form", ["bf16", "q4"])
@pytest.mark.parametrize("bf16", [False, True])
def test_append(dev, name, form, bf16):
    """Bit for bit: products and sums of the rotation are rounded one by one, and so is the integer of a value."""
    import tang_b200 as tb

    nh, nkv, P, lens, counts = ROWS[name]
    s = Sequences(nh, nkv, P, lens, counts, 1, form, seqs=[3, 0, 5, 1][:len(lens)] if len(lens) > 1 else None).put(dev)
    x = s.rng.standard_normal((s.rows, nh + 2 * nkv, HD)).astype(np.float32) * 2
    bits, rounded = bf16_round(x)
    q, cos, sin = appended(s, dev, bits if bf16 else x, tb.BF16 if bf16 else tb.F32, max(lens) + 1)
    x = rounded if bf16 else x
    pos, at = s.new_positions(), s.new_places()
    turned = rotate(x[:, :nh + nkv], cos[pos], sin[pos])
    assert np.array_equal(q.to_vec().reshape(s.rows, nh, HD), bf16_round(turned[:, :nh])[0].reshape(s.rows, nh, HD))
    for buf, raw, new in ((s.kb, s.raw[0], turned[:, nh:]), (s.vb, s.raw[1], x[:, nh + nkv:])):
        want = raw.copy()
        want[at] = pack(new)[0] if form == "q4" else bf16_round(np.ascontiguousarray(new))[0].reshape(s.rows, -1)
        got = buf.to_vec().reshape(want.shape)
        assert np.array_equal(got[at], want[at])
        rest = np.ones(len(want), bool)
        rest[at] = False
        assert np.array_equal(got[rest], want[rest])
    dev.sync()


@pytest.mark.parametrize("name", list(ROWS))
@pytest.mark.parametrize("form", ["bf16", "q4"])
def test_read(dev, name, form):
    nh, nkv, P, lens, counts = ROWS[name]
    s = Sequences(nh, nkv, P, lens, counts, 2, form).put(dev)
    k, v = dev.kv_read_paged(s.kb, s.vb, s.pool, s.B, s.rows, nkv, HD, seq_rows=s.seq_rows)
    at = s.new_places()
    for buf, values in ((k, s.values[0]), (v, s.values[1])):
        assert np.array_equal(widen(buf.to_vec()).reshape(s.rows, nkv, HD), values[at])
    dev.sync()


def test_four_bits_of_what_is_no_ordinary_number(dev):
    """Zeros, tiny, huge and infinite values, NaN: block by block; ties go to the even integer."""
    import tang_b200 as tb

    s = Sequences(2, 2, 16, [16], [16], 3, "q4").put(dev)
    x = np.zeros((16, 6, HD), np.float32)
    v = x[:, 4:].reshape(16, 8, 32)
    v[0, 0] = 0.0
    v[0, 1, 3], v[0, 2, 5], v[0, 3, 31] = np.inf, -np.inf, np.nan
    v[1, 0, :4], v[1, 1, :2] = [7, 0.5, 1.5, -2.5], [-7, 3.4999]
    v[2, 0, 0], v[2, 1, 0], v[2, 2, 0] = 2.0 ** 120, np.float32(2.0 ** 120) * np.float32(1 - 2.0 ** -24), 3e38
    v[3, 0, 7], v[3, 1, 7], v[3, 2, 7] = 2.0 ** -100, np.float32(2.0 ** -100) * np.float32(1 - 2.0 ** -24), 1e-44
    v[4, :, :] = np.arange(-16, 16)
    v[5, 0, :3], v[5, 1, 9] = [7 * 17 / 16, 17 / 32, 17 / 16], -7 * 33 / 32
    appended(s, dev, x, tb.F32, 16)
    got = s.vb.to_vec().reshape(s.raw[1].shape)[s.new_places()]
    bits, values = pack(x[:, 4:])
    assert np.array_equal(got, bits)
    k, w = dev.kv_read_paged(s.kb, s.vb, s.pool, 1, 16, 2, HD, seq_rows=s.seq_rows)
    w = widen(w.to_vec()).reshape(16, 2, HD)
    assert np.array_equal(np.isnan(w), np.isnan(values)) and np.array_equal(w[~np.isnan(w)], values[~np.isnan(values)])
    assert np.isnan(w).sum() == 5 * 32 and list(w[1, 0, :4]) == [7, 0, 2, -2]
    dev.sync()


def test_rows_behind_the_last_sequence_are_left(dev):
    import tang_b200 as tb

    for form in ("bf16", "q4"):
        s = Sequences(4, 2, 16, [20, 9], [4, 9], 4, form).put(dev)
        rows = 21
        x = s.rng.standard_normal((rows, 8, HD)).astype(np.float32)
        q = dev.upload(np.full(rows * 4 * HD, 0x1234, np.uint16), tb.BF16)
        before = s.kb.to_vec()
        appended(s, dev, x, tb.F32, 20, rows=rows, q_out=q)
        left = q.to_vec().reshape(rows, -1)[13:]
        assert (left == 0x1234).all()
        changed = (s.kb.to_vec() != before).reshape(s.raw[0].shape).any(1)
        assert set(np.nonzero(changed)[0]) <= set(s.new_places())
        out = dev.upload(np.full(rows * 4 * HD, 0x1234, np.uint16), tb.BF16)
        s.qb = dev.upload(np.concatenate([s.q_bits.reshape(-1), np.zeros((rows - 13) * 4 * HD, np.uint16)]), tb.BF16)
        dev.gqa_prefill_paged(s.qb, s.kb, s.vb, s.pool, 2, rows, 4, 2, HD, 20, seq_rows=s.seq_rows, out=out)
        ko, vo = (dev.upload(np.full(rows * 2 * HD, 0x1234, np.uint16), tb.BF16) for _ in range(2))
        dev.kv_read_paged(s.kb, s.vb, s.pool, 2, rows, 2, HD, seq_rows=s.seq_rows, k_out=ko, v_out=vo)
        for b in (out, ko, vo):
            got = b.to_vec().reshape(rows, -1)
            assert (got[13:] == 0x1234).all() and (got[:13] != 0x1234).any(1).all()
        dev.sync()


def test_strided_rows(dev):
    import tang_b200 as tb

    s = Sequences(4, 2, 16, [3, 40], [3, 10], 5, "bf16").put(dev)
    ld = 8 * HD + 12
    x = s.rng.standard_normal((s.rows, ld)).astype(np.float32)
    q, cos, sin = appended(s, dev, x, tb.F32, 40, ldx=ld)
    turned = rotate(np.ascontiguousarray(x[:, :6 * HD]).reshape(s.rows, 6, HD), cos[s.new_positions()], sin[s.new_positions()])
    assert np.array_equal(q.to_vec(), bf16_round(np.ascontiguousarray(turned[:, :4]))[0].reshape(-1))
    dev.sync()


def test_what_is_not_the_sequences_to_write_is_left(dev):
    """A shared page, a refused extension, a sequence twice, no page, a position behind the tables, more rows than positions: reported, nothing written for it,
    the others' rows are."""
    import tang_b200 as tb

    def case(change, ok, n_positions=64, seqs=None, counts=(3, 3, 3)):
        s = Sequences(4, 2, 16, [20, 30, 40], list(counts), 6, "bf16")
        change(s)
        s.put(dev)
        if seqs is not None:
            s.seqs = dev.upload(np.array(seqs, np.int32), tb.I32)
        x = s.rng.standard_normal((s.rows, 8, HD)).astype(np.float32)
        before = s.kb.to_vec().reshape(s.raw[0].shape)
        appended(s, dev, x, tb.F32, n_positions)
        with pytest.raises(tb.TangqError):
            dev.sync()
        changed = set(np.nonzero((s.kb.to_vec().reshape(before.shape) != before).any(1))[0])
        want = set()
        for b in ok:
            n, c = s.lens[b], counts[b]
            want |= set(s.places(b, range(n - c, n)).tolist())
        assert changed == want

    def share(s):
        s.refs[s.tables[1, 1]] = 2

    def no_page(s):
        s.tables[1, 1] = s.n_pages

    def short(s):
        s.lens_all[1] = 2

    case(share, [0, 2])
    case(no_page, [0, 2])
    case(short, [0, 2])
    case(lambda s: None, [0, 1], n_positions=37)
    case(lambda s: None, [2], seqs=[0, 0, 2])
    case(lambda s: None, [0, 2], seqs=[0, 7, 2])
    case(lambda s: None, [0, 2], seqs=[0, -1, 2])
    # a refused extension: the pool has no pages left
    s = Sequences(4, 2, 16, [16, 16], [1, 1], 7, "bf16", extra=1).put(dev)
    s.pool.set_arrays([s.kb, s.vb])
    s.pool.extend([0, 1])
    before = s.kb.to_vec()
    with pytest.raises(tb.TangqError):
        dev.sync()
    appended(s, dev, np.ones((2, 8, HD), np.float32), tb.F32, 64)
    with pytest.raises(tb.TangqError):
        dev.sync()
    assert np.array_equal(before, s.kb.to_vec())


# query heads, KV heads, page rows, lengths, new rows
PREFILL = {
    "one token": (32, 8, 16, [1], [1]),
    "one tile": (8, 2, 64, [128], [128]),
    "a tile and one": (8, 2, 64, [129], [129]),
    "packed": (32, 8, 32, [300, 1, 77, 513, 2], [300, 1, 77, 513, 2]),
    "behind cached ones": (16, 4, 16, [700, 45, 131], [100, 1, 3]),
    "one query head each": (4, 4, 128, [260, 31], [260, 31]),
    "two": (6, 3, 16, [150, 140], [150, 12]),
    "three": (9, 3, 32, [200, 64], [200, 64]),
    "five": (15, 3, 64, [129, 100], [129, 30]),
    "six": (6, 1, 16, [99], [99]),
    "seven": (14, 2, 16, [270, 17], [50, 17]),
    "eight": (8, 1, 256, [600], [600]),
    "nothing new of some": (8, 2, 16, [5, 40, 0, 18], [0, 40, 0, 3]),
    "large pages": (8, 2, 1024, [1500, 900], [600, 900]),
    "few rows, many keys": (8, 2, 64, [5000, 4097], [2, 33]),
    "one row each": (8, 2, 32, [900, 64, 1, 2500], [1, 1, 1, 1]),
    "many sequences": (4, 2, 16, [(7 * i) % 90 + 1 for i in range(150)], [min((7 * i) % 90 + 1, 1 + (5 * i) % 40) for i in range(150)]),
}


@pytest.mark.parametrize("name", list(PREFILL))
@pytest.mark.parametrize("form", ["bf16", "q4"])
def test_prefill(dev, name, form):
    s = Sequences(*PREFILL[name], 10 + len(name), form).put(dev)
    got = s.prefill().to_vec()
    dev.sync()
    check_attention(got, *s.reference(), terms=1)


def test_prefill_of_listed_sequences_and_a_loose_bound(dev):
    for form in ("bf16", "q4"):
        s = Sequences(8, 2, 32, [60, 200, 33], [60, 7, 33], 30, form, seqs=[4, 1, 6]).put(dev)
        a = s.prefill().to_vec()
        b = s.prefill(max_len=1 << 20).to_vec()
        dev.sync()
        want = s.reference()
        check_attention(a, *want, terms=1)
        check_attention(b, *want, terms=1)


def test_prefill_bounded(dev):
    """Keys at max_len and behind are not attended."""
    s = Sequences(8, 2, 16, [300, 40], [20, 40], 31, "bf16").put(dev)
    got = widen(s.prefill(max_len=150).to_vec()).reshape(60, 8, HD)
    dev.sync()
    at = s.places(0, range(150))
    from packed_util import attend

    for r in range(20):
        want, size = attend(s.q[r:r + 1], s.values[0][at], s.values[1][at])
        assert (np.abs(got[r:r + 1] - want) <= 2.0 ** -6 * size).all()


@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_prefill_values_that_earlier_rows_do_not_see(dev, bad):
    """A value that is no number in a later position of the same tile: the rows before it are finite."""
    for P, at_pos, c in ((16, 150, 200), (64, 199, 200), (32, 128, 129)):
        s = Sequences(8, 2, P, [200], [c if c <= 200 else 200], 32, "bf16")
        place = s.places(0, [at_pos])[0]
        s.raw[1][place, 5] = 0x7F80 if np.isinf(bad) else 0x7FC0
        s.put(dev)
        got = widen(s.prefill().to_vec()).reshape(s.rows, 8, HD)
        dev.sync()
        want, size = s.reference()
        first = 200 - s.rows
        before = np.arange(s.rows) + first < at_pos
        ok = np.ones((8, HD), bool)
        ok[:4, 5] = False
        assert np.isfinite(got[before]).all() and np.isfinite(got[~before][:, ok]).all() and not np.isfinite(got[~before][:, ~ok]).any()
        tol = 2.0 ** -14 * size + 2.0 ** -7 * (size + np.abs(want))
        assert (np.abs(got - want)[before] <= tol[before]).all() and (np.abs(got - want)[~before][:, ok] <= tol[~before][:, ok]).all()


@pytest.mark.parametrize("form", ["bf16", "q4"])
def test_prefill_keys_that_are_no_number(dev, form):
    """Rows that see such a key are NaN, in its KV head; those before it are what they were."""
    for at_pos in (0, 3, 130, 131, 170, 199):
        s = Sequences(8, 2, 32, [200], [200], 34, form)
        place = s.places(0, [at_pos])[0]
        if form == "q4":
            s.raw[0][place, 2 * 64:].view(np.uint16)[5] = 0x7FC0
        else:
            s.raw[0][place, HD + 40] = 0x7FC0
        s.put(dev)
        got = widen(s.prefill().to_vec()).reshape(s.rows, 8, HD)
        dev.sync()
        want, size = s.reference()
        bad = np.zeros((200, 8), bool)
        bad[at_pos:, 4:] = True
        assert np.isnan(got[bad]).all()
        tol = 2.0 ** -14 * size + 2.0 ** -7 * (size + np.abs(want))
        assert (np.abs(got - want)[~bad] <= tol[~bad]).all()


def test_prefill_scores_that_grow(dev):
    """Keys in ascending order of their scores, far apart: the reference has to follow."""
    s = Sequences(8, 2, 32, [640], [640], 33, "bf16")
    at = s.places(0, range(640))
    grow = np.linspace(0.01, 40.0, 640)[:, None, None] * np.sign(s.q[-1, 0])[None, None]
    bits, val = bf16_round(np.broadcast_to(grow, (640, 2, HD)).astype(np.float32).copy())
    s.raw[0][at], s.values[0][at] = bits.reshape(640, -1), val
    s.put(dev)
    got = s.prefill().to_vec()
    dev.sync()
    want, size = s.reference()
    got = widen(got).reshape(want.shape)
    # (scores of up to 2^11, sums in f32: 2^-24 * 128 of their parts, 2^-6 of the weights where several are near)
    assert np.isfinite(got).all() and (np.abs(got - want) <= 2.0 ** -4 * size + 1e-6).all()


DECODE = {
    "one position": (32, 8, 16, [1]),
    "none": (8, 2, 16, [0, 5, 0]),
    "a chunk's ends": (8, 2, 16, [31, 32, 33, 64, 65]),
    "a small model": (16, 4, 64, [700, 3, 129]),
    "one query head each": (4, 4, 32, [300, 40]),
    "two": (6, 3, 16, [150, 1000]),
    "three": (9, 3, 32, [200, 64]),
    "five": (15, 3, 64, [129, 100, 2000]),
    "six": (6, 1, 16, [99]),
    "seven": (14, 2, 128, [270, 17]),
    "eight": (8, 1, 256, [600, 5000]),
    "long": (8, 2, 1024, [20000]),
    "many": (8, 8, 16, [(37 * i) % 400 for i in range(300)]),
}


@pytest.mark.parametrize("name", list(DECODE))
def test_decode_over_four_bits(dev, name):
    nh, nkv, P, lens = DECODE[name]
    s = Sequences(nh, nkv, P, lens, [1] * len(lens), 50 + len(name), "q4", k_size=1.5).put(dev)
    a = s.decode().to_vec()
    b = s.decode(max_len=1 << 20).to_vec()
    dev.sync()
    want = s.reference()
    check_attention(a, *want, terms=2)
    check_attention(b, *want, terms=2)


def test_decode_over_four_bits_of_listed_sequences_and_bounded(dev):
    s = Sequences(8, 2, 32, [60, 200, 33], [1, 1, 1], 60, "q4", seqs=[4, 1, 6]).put(dev)
    got = s.decode().to_vec()
    cut = widen(s.decode(max_len=50).to_vec()).reshape(3, 8, HD)
    dev.sync()
    check_attention(got, *s.reference(), terms=2)
    from packed_util import attend

    at = s.places(1, range(50))
    want, size = attend(s.q[1:2], s.values[0][at], s.values[1][at])
    assert (np.abs(cut[1:2] - want) <= 2.0 ** -7 * size).all()


def test_decode_over_four_bits_scores_that_grow(dev):
    s = Sequences(8, 2, 32, [900], [1], 61, "q4")
    at = s.places(0, range(900))
    grow = np.linspace(0.01, 40.0, 900)[:, None, None] * np.sign(s.q[0, 0])[None, None]
    bits, val = pack(np.broadcast_to(grow, (900, 2, HD)).astype(np.float32).copy())
    s.raw[0][at], s.values[0][at] = bits, val
    s.put(dev)
    got = widen(s.decode().to_vec()).reshape(1, 8, HD)
    dev.sync()
    want, size = s.reference()
    assert np.isfinite(got).all() and (np.abs(got - want) <= 2.0 ** -4 * size + 1e-6).all()


def test_decode_over_four_bits_with_values_that_are_no_number(dev):
    """A block that is NaN: in values it is that block's results of its KV head, in keys all of that KV head's; the others' are what they were."""
    s = Sequences(8, 2, 16, [200, 300], [1, 1], 62, "q4")
    for which in (0, 1):
        t = Sequences(8, 2, 16, [200, 300], [1, 1], 62, "q4")
        place = t.places(0, [77])[0]
        scale = t.raw[which][place, 2 * 64:].view(np.uint16)
        scale[1 * 4 + 2] = 0x7FC0      # KV head 1, values 64 .. 95
        t.put(dev)
        got = widen(t.decode().to_vec()).reshape(2, 8, HD)
        dev.sync()
        bad = np.zeros((2, 8, HD), bool)
        bad[0, 4:, slice(64, 96) if which else slice(None)] = True
        assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
        s.put(dev)
        ok = widen(s.decode().to_vec()).reshape(2, 8, HD)
        dev.sync()
        assert np.array_equal(got[~bad], ok[~bad])


@pytest.mark.parametrize("form", ["bf16", "q4"])
def test_the_largest_batch(dev, form):
    """1024 sequences in an order of their own: one row each, and several, some none."""
    import tang_b200 as tb

    rng = np.random.default_rng(7)
    order = rng.permutation(1100)[:1024]
    for most in (1, 9):
        lens = rng.integers(1, 60, 1024)
        counts = np.minimum(lens, rng.integers(0 if most > 1 else 1, most + 1, 1024))
        s = Sequences(4, 2, 16, lens, counts, 8, form, seqs=order).put(dev)
        x = s.rng.standard_normal((s.rows, 8, HD)).astype(np.float32)
        at = s.new_places()
        k, v = dev.kv_read_paged(s.kb, s.vb, s.pool, 1024, s.rows, 2, HD, seqs=s.seqs, seq_rows=s.seq_rows)
        assert np.array_equal(widen(k.to_vec()).reshape(s.rows, 2, HD), s.values[0][at]) and np.array_equal(widen(v.to_vec()).reshape(s.rows, 2, HD), s.values[1][at])
        got = s.prefill().to_vec()
        want = s.reference()
        check_attention(got, *want, terms=1)
        if form == "q4" and most == 1:
            check_attention(s.decode().to_vec(), *want, terms=2)
        appended(s, dev, x, tb.F32, 64)
        new = s.kb.to_vec().reshape(s.raw[0].shape)
        cos, sin = tables(64)
        turned = rotate(x[:, 4:6], cos[s.new_positions()], sin[s.new_positions()])
        assert np.array_equal(new[at], pack(turned)[0] if form == "q4" else bf16_round(np.ascontiguousarray(turned))[0].reshape(s.rows, -1))
        dev.sync()


@pytest.mark.parametrize("form", ["bf16", "q4"])
def test_starts_that_do_not_ascend(dev, form):
    """Reported; rows of the sequences whose starts are sound are what they are without the others."""
    import tang_b200 as tb

    for starts, sound in (([0, 20, 10, 30], [(0, 0, 10)]), ([0, 10, 40, 30], [(0, 0, 10)]), ([-3, 10, 20, 30], [(1, 10, 10), (2, 20, 10)])):
        s = Sequences(4, 2, 16, [50, 60, 70], [10, 10, 10], 9, form).put(dev)
        want, size = s.reference()
        s.seq_rows = dev.upload(np.array(starts, np.int32), tb.I32)
        out = dev.upload(np.zeros(30 * 4 * HD, np.uint16), tb.BF16)
        got = s.prefill(out=out).to_vec().reshape(30, 4, HD)
        with pytest.raises(tb.TangqError):
            dev.sync()
        if starts[1] == 10 and starts[0] == 0 or starts[0] < 0:
            for i, first, n in sound:
                check_attention(got[first:first + n], want[first:first + n], size[first:first + n], terms=1)
        before = s.kb.to_vec()
        x = s.rng.standard_normal((30, 8, HD)).astype(np.float32)
        appended(s, dev, x, tb.F32, 80)
        with pytest.raises(tb.TangqError):
            dev.sync()
        changed = set(np.nonzero((s.kb.to_vec() != before).reshape(s.raw[0].shape).any(1))[0])
        allowed = set()
        for b in range(3):
            allowed |= set(s.places(b, range(s.lens[b])).tolist())
        assert changed <= allowed


@pytest.mark.parametrize("form", ["bf16", "q4"])
@pytest.mark.parametrize("what", ["page", "sequence", "length"])
def test_what_does_not_exist_is_reported(dev, form, what):
    """A page, a sequence, more rows than positions: the other sequences' results are what they are."""
    import tang_b200 as tb

    for counts in ([10, 1, 30], [1, 1, 1]):
        s = Sequences(8, 2, 16, [100, 40, 90], counts, 11, form, seqs=[2, 0, 1])
        want, size = s.reference()
        if what == "page":
            s.tables[0, 1] = -5
        elif what == "sequence":
            s.order = np.array([2, 99, 1])
        else:
            s.lens_all[0] = -1 if counts[1] == 1 else 0
        s.put(dev)
        calls = [lambda: s.prefill(), lambda: dev.kv_read_paged(s.kb, s.vb, s.pool, 3, s.rows, 2, HD, seqs=s.seqs, seq_rows=s.seq_rows)[0]]
        if form == "q4" and counts[0] == 1 and what != "length":
            calls.append(lambda: s.decode())
        for i, call in enumerate(calls):
            got = call().to_vec()
            reads_it = what != "page" or i != 1 or counts[1] > 24       # (the page holds positions 16 to 31, the new rows are behind it)
            if reads_it:
                with pytest.raises(tb.TangqError):
                    dev.sync()
            else:
                dev.sync()
            if i != 1:
                ok = np.ones(s.rows, bool)
                ok[s.starts[1]:s.starts[2]] = False
                check_attention(got.reshape(want.shape)[ok], want[ok], size[ok], terms=1 if i == 0 else 2)
