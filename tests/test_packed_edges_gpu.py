"""Packed rows over pages at their edges: lists of starts that are not what they should be, values and keys that are no number where a tile's keys are cut
into parts or the context is long, values near the end of what f32 holds, bounds on the length."""
import numpy as np
import pytest

from packed_util import HD, Sequences, attend, check_attention, pack, rotate, tables, widen
from util import bf16_round

pytestmark = pytest.mark.gpu
FILLER = 0x1234


@pytest.fixture(scope="module")
def dev():
    import tang_b200

    d = tang_b200.QuantComputeDevice(0)
    yield d
    d.close()


def sound(starts, rows):
    """(sequence, first row, rows) of those whose rows are theirs: no start before is larger, the first is 0, the end neither before nor behind what there is."""
    return [(i, a, b - a) for i, (a, b) in enumerate(zip(starts, starts[1:])) if a == max(starts[:i + 1]) and a >= 0 and (i or a == 0) and a <= b <= rows]


def many(n, at, value):
    starts = [2 * i for i in range(n + 1)]
    starts[at] = value
    return starts


STARTS = {
    "behind 0": [5, 30, 40, 40],
    "all behind 0": [7, 7, 7, 7],
    "nobody's before": [3, 3, 9, 40],
    "below 0": [-3, 10, 20, 30],
    "back into the first": [0, 20, 10, 30],
    "back into the first, then on": [0, 30, 10, 40],
    "an end behind the rows": [0, 10, 60, 40],
    "the last one back": [0, 20, 20, 10],
    "one of many back": many(150, 140, 10),
    "one of many ahead": many(150, 40, 200),
    "the last of many back": many(150, 150, 7),
}


@pytest.mark.parametrize("form", ["bf16", "q4"])
@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("name", list(STARTS))
def test_starts_that_are_not_what_they_should_be(dev, form, long, name):
    """Reported by every call.  Rows that are a sequence's by the rule are appended, read and attended, all others are left as they were: whether a tile's keys
    are cut into parts (long) or not."""
    import tang_b200 as tb

    starts = STARTS[name]
    B = len(starts) - 1
    rows = 40 if B == 3 else 2 * B
    lens = ([1450, 1360, 1270] if long else [50, 60, 70]) if B == 3 else [(1100 if long and i == 3 else 320) - i % 7 for i in range(B)]
    s = Sequences(4, 2, 16, lens, [rows // B] * (B - 1) + [rows - rows // B * (B - 1)], 3, form).put(dev)
    s.seq_rows = dev.upload(np.array(starts, np.int32), tb.I32)
    ok = sound(starts, rows)
    theirs = np.zeros(rows, bool)
    for _, a, n in ok:
        theirs[a:a + n] = True
    filled = lambda width: dev.upload(np.full(rows * width * HD, FILLER, np.uint16), tb.BF16)  # noqa: E731

    def reported():
        with pytest.raises(tb.TangqError):
            dev.sync()

    out = filled(4)
    got = s.prefill(out=out).to_vec().reshape(rows, 4, HD)
    reported()
    assert (got[~theirs] == FILLER).all()
    for i, a, n in ok:
        if n:
            at = s.places(i, range(lens[i]))
            check_attention(got[a:a + n], *attend(s.q[a:a + n], s.values[0][at], s.values[1][at]), terms=1)
    places = {i: s.places(i, range(lens[i] - n, lens[i])) for i, _, n in ok}
    k, v = dev.kv_read_paged(s.kb, s.vb, s.pool, B, rows, 2, HD, seq_rows=s.seq_rows, k_out=filled(2), v_out=filled(2))
    reported()
    for buf, values in ((k, s.values[0]), (v, s.values[1])):
        got = buf.to_vec().reshape(rows, 2, HD)
        assert (got[~theirs] == FILLER).all()
        for i, a, n in ok:
            assert np.array_equal(widen(got[a:a + n]), values[places[i]])
    x = s.rng.standard_normal((rows, 8, HD)).astype(np.float32)
    cos, sin = tables(1500)
    q = dev.kv_append_paged(dev.upload(x), dev.upload(cos), dev.upload(sin), s.pool, s.kb, s.vb, B, rows, 4, 2, HD, seq_rows=s.seq_rows, q_out=filled(4))
    reported()
    assert (q.to_vec().reshape(rows, -1)[~theirs] == FILLER).all()
    stored = lambda a: pack(a)[0] if form == "q4" else bf16_round(np.ascontiguousarray(a))[0].reshape(len(a), -1)  # noqa: E731
    wants = [raw.copy() for raw in s.raw]
    for i, a, n in ok:
        pos = np.arange(lens[i] - n, lens[i])
        turned = rotate(x[a:a + n, :6], cos[pos], sin[pos])
        if n:
            wants[0][places[i]], wants[1][places[i]] = stored(turned[:, 4:]), stored(x[a:a + n, 6:])
            assert np.array_equal(q.to_vec().reshape(rows, 4, HD)[a:a + n], bf16_round(np.ascontiguousarray(turned[:, :4]))[0].reshape(n, 4, HD))
    for buf, want in ((s.kb, wants[0]), (s.vb, wants[1])):
        assert np.array_equal(buf.to_vec().reshape(want.shape), want)


def spoil(s, which, place, form):
    """Makes a value of a cache row no number (an infinity or NaN, a block's scale in 4 bits); the columns of the results that it reaches, [heads, 128]."""
    hit = np.zeros((s.nh, HD), bool)
    group = s.nh // s.nkv
    if form == "q4":
        s.raw[which][place, s.nkv * 64:].view(np.uint16)[4 + 2] = 0x7FC0      # KV head 1, values 64 .. 95
        hit[group:2 * group, slice(64, 96) if which else slice(None)] = True
    else:
        s.raw[which][place, HD + 40] = 0x7F80 if place % 2 else 0x7FC0
        hit[group:2 * group, 40 if which else slice(None)] = True
    return hit


def near(got, want, size):
    return (np.abs(got - want) <= 2.0 ** -14 * size + 2.0 ** -8 * (size + np.abs(want)) + 2.0 ** -8 * (np.abs(want) + 2.0 ** -7 * size)).all()


@pytest.mark.parametrize("form", ["bf16", "q4"])
@pytest.mark.parametrize("which", ["keys", "values"])
@pytest.mark.parametrize("at", [[1999], [1990], [1965], [1960], [1959], [700], [1992, 3], [1963, 1980, 1995]])
def test_what_is_no_number_where_keys_are_cut_into_parts(dev, form, which, at):
    """One sequence of 2000 positions, 40 rows, 2 KV heads: two tiles, seven parts each.  Rows that see such a key or value are no numbers where it reaches them
    (an infinite key that a query makes a score of minus infinity has no weight, and is not missed); the others are what they are."""
    s = Sequences(8, 2, 32, [2000], [40], 40, form)
    want, size = s.reference()
    bad = np.zeros((40, 8, HD), bool)
    for pos in at:
        place = s.places(0, [pos])[0]
        hit = spoil(s, which == "values", place, form)
        bad[max(pos - 1960, 0):] |= hit
        if which == "keys":
            s.values[0][place, 1] = np.nan if form == "q4" else np.where(np.arange(HD) == 40, np.inf if place % 2 else np.nan, s.values[0][place, 1])
    if which == "keys":
        with np.errstate(invalid="ignore"):
            want, size = s.reference()
        assert np.isnan(want[bad]).any() and np.isfinite(want[~bad]).all()
        bad = np.isnan(want)
    s.put(dev)
    got = widen(s.prefill().to_vec()).reshape(want.shape)
    dev.sync()
    assert not np.isfinite(got[bad]).any() and near(got[~bad], want[~bad], size[~bad])


@pytest.mark.parametrize("form", ["bf16", "q4"])
@pytest.mark.parametrize("nh,nkv", [(4, 4), (15, 3), (8, 2), (8, 1)])
def test_values_that_are_no_number_in_every_position(dev, form, nh, nkv):
    """Nothing but NaN: every row sees one, in as many tiles as there are, and the heads beside them are what they are."""
    s = Sequences(nh, nkv, 16, [700, 130, 1], [700, 40, 1], 41, form)
    want, size = s.reference()
    bad = np.zeros((nh, HD), bool)
    for b, n in enumerate(s.lens):
        at = s.places(b, range(n))
        if form == "q4":
            s.raw[1][at, nkv * 64:nkv * 64 + 2] = np.array([0xC0, 0x7F], np.uint8)
            bad[:nh // nkv, :32] = True
        else:
            s.raw[1][at, :HD] = 0x7FC0
            bad[:nh // nkv] = True
    s.put(dev)
    got = widen(s.prefill().to_vec()).reshape(want.shape)
    dev.sync()
    assert np.isnan(got[:, bad]).all() and near(got[:, ~bad], want[:, ~bad], size[:, ~bad])


def test_infinite_values_stay_infinite(dev):
    """One is an infinity from its position on; two of different signs are NaN from the second one's on.  Rows before them are finite."""
    for nh, nkv, c in ((8, 2, 200), (4, 4, 200), (7, 1, 60), (9, 3, 33)):
        s = Sequences(nh, nkv, 16, [200], [c], 42, "bf16")
        want, size = s.reference()
        first = 200 - c
        up, down = first + c // 3, first + c // 3 + 9
        for pos, bits in ((up, 0x7F80), (down, 0xFF80)):
            s.raw[1][s.places(0, [pos])[0], 17] = bits
        s.put(dev)
        got = widen(s.prefill().to_vec()).reshape(want.shape)
        dev.sync()
        group, column = nh // nkv, got[:, :nh // nkv, 17]
        assert np.isfinite(column[:up - first]).all() and (column[up - first:down - first] == np.inf).all() and np.isnan(column[down - first:]).all()
        rest = np.ones(got.shape, bool)
        rest[up - first:, :group, 17] = False
        assert near(got[rest], want[rest], size[rest])


@pytest.mark.parametrize("form", ["bf16", "q4"])
def test_values_that_are_no_number_behind_a_long_context(dev, form):
    """100003 positions and as many new rows as leave a tile's keys in one part: what rows cost that do not see such a value does not grow with the context."""
    n, c = 100003, 4800
    s = Sequences(8, 2, 64, [n], [c], 43, form)
    places = {pos: s.places(0, [pos])[0] for pos in (n - 1, n - 40, n - 3000, n - c + 1)}
    for place in places.values():
        hit = spoil(s, 1, place, form)
    s.put(dev)
    got = widen(s.prefill().to_vec()).reshape(c, 8, HD)
    dev.sync()
    seen = n - c + np.arange(c) >= n - c + 1
    assert np.isfinite(got[~seen]).all() and np.isfinite(got[:, ~hit]).all() and not np.isfinite(got[seen][:, hit]).any()
    at = s.places(0, range(n))
    k, v = s.values[0][at], s.values[1][at]
    for r in (0, 1, 30, c - 3000, c - 40, c - 1):
        want, size = attend(s.q[r:r + 1], k[:n - c + r + 1], v[:n - c + r + 1])
        ok = slice(None) if r == 0 else ~hit
        assert near(got[r][ok], want[0][ok], size[0][ok])


@pytest.mark.parametrize("form", ["bf16", "q4"])
def test_a_value_that_is_no_number_at_the_end_of_a_long_context(dev, form):
    """The same where only the last row sees it: all rows before it are finite."""
    n, c = 60001, 4800
    s = Sequences(8, 2, 64, [n], [c], 44, form)
    hit = spoil(s, 1, s.places(0, [n - 1])[0], form)
    s.put(dev)
    got = widen(s.prefill().to_vec()).reshape(c, 8, HD)
    dev.sync()
    assert np.isfinite(got[:-1]).all() and np.isfinite(got[-1, ~hit]).all() and not np.isfinite(got[-1, hit]).any()
    at = s.places(0, range(n))
    k, v = s.values[0][at], s.values[1][at]
    for r in (c - 2, c - 31):
        want, size = attend(s.q[r:r + 1], k[:n - c + r + 1], v[:n - c + r + 1])
        assert near(got[r], want[0], size[0])


def scored(s, high, values, seed=5):
    """All queries are one vector, keys are noise beside it, those that `high` names score 2^7.2 times the weight of the others; values are positive, `values` large."""
    rng = np.random.default_rng(seed)
    u = (rng.standard_normal(HD) * 1.5).astype(np.float32)
    s.q_bits, s.q = bf16_round(np.broadcast_to(u, s.q.shape).copy())
    u = s.q[0, 0].astype(np.float64)
    for b, n in enumerate(s.lens):
        at, up = s.places(b, range(n)), high(np.arange(n))
        k = rng.standard_normal((n, s.nkv, HD)) * 0.1
        k += (up * 7.2 * np.log(2) * np.sqrt(HD))[:, None, None] * u / (u @ u)
        for i, x in enumerate((k, np.minimum(np.abs(rng.standard_normal((n, s.nkv, HD))), 4) * values)):
            x = np.ascontiguousarray(x, np.float32)
            if s.form == "q4":
                s.raw[i][at], s.values[i][at] = pack(x)
            else:
                bits, s.values[i][at] = bf16_round(x)
                s.raw[i][at] = bits.reshape(n, -1)
    return s


@pytest.mark.parametrize("form,values", [("bf16", 2.0 ** 120), ("q4", 2.0 ** 117)])
@pytest.mark.parametrize("lens,counts", [([640], [640]), ([2000], [40]), ([900, 130], [30, 130])])
def test_prefill_sums_near_the_end_of_f32(dev, form, values, lens, counts):
    """Values so large that 2^8 times their sum is no f32 number, whose sum with weights of at most 1 is one: a row's reference may lag, and is not felt.  (bf16: 8 of
    320 keys at a time are high, 4 bits: 64; the sums are below 2^126.)"""
    some = 8 if form == "bf16" else 64
    s = scored(Sequences(8, 2, 32, lens, counts, 45, form), lambda pos: (pos // 64 % 5 == 1) & (pos % 64 < some), values).put(dev)
    got = widen(s.prefill().to_vec())
    dev.sync()
    want, size = s.reference()
    assert np.isfinite(got).all() and near(got.reshape(want.shape), want, size)


def test_decode_over_four_bits_sums_near_the_end_of_f32(dev):
    """As above; as many heads and positions as give a warp several chunks of 32 keys, every second of which is high."""
    s = scored(Sequences(32, 32, 16, [900, 700, 33, 64, 800, 1000], [1] * 6, 46, "q4"), lambda pos: pos // 32 % 2 == 1, 2.0 ** 117).put(dev)
    got = s.decode().to_vec()
    dev.sync()
    check_attention(got, *s.reference(), terms=2)


@pytest.mark.parametrize("form", ["bf16", "q4"])
def test_values_near_the_other_end_of_f32(dev, form):
    """Values of 2^-100: neither attention takes them for zeros."""
    s = scored(Sequences(8, 2, 32, [640], [640 if form == "bf16" else 1], 47, form), lambda pos: pos // 64 % 5 == 1, 2.0 ** -98).put(dev)
    got = s.prefill().to_vec()
    want = s.reference()
    # (the allowance of check_attention for results of zero is larger than these)
    for out, terms in ((got, 1), *([(s.decode().to_vec(), 2)] if form == "q4" else [])):
        check_attention(((widen(out) * 2.0 ** 98).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16), want[0] * 2.0 ** 98, want[1] * 2.0 ** 98, terms)
    dev.sync()


def test_results_that_share_memory_with_what_is_read_are_refused(dev):
    """Queries of an append beside, within and into the rows it reads; results of the attention the same; next to them is another buffer."""
    import tang_b200 as tb

    s = Sequences(4, 2, 16, [20, 9], [4, 9], 48, "bf16").put(dev)
    rows, width, nq = s.rows, 8 * HD, 4 * HD
    cos, sin = (dev.upload(a) for a in tables(32))
    whole = dev.upload(np.zeros(rows * width + 2 * rows * nq, np.uint16), tb.BF16)
    part = lambda first, n: tb.Buffer(dev, whole.ptr + 2 * first, n, tb.BF16, owns=False)  # noqa: E731
    x = part(rows * nq, rows * width)
    append = lambda out: dev.kv_append_paged(x, cos, sin, s.pool, s.kb, s.vb, 2, rows, 4, 2, HD, seq_rows=s.seq_rows, q_out=out)  # noqa: E731
    for first in (8, rows * nq, rows * nq + nq, rows * nq + rows * width - 8):
        with pytest.raises(tb.TangqError):
            append(part(first, rows * nq))
    for first in (0, rows * nq + rows * width):
        append(part(first, rows * nq))
    dev.sync()
    q = part(rows * nq, rows * nq)
    attend_to = lambda out: dev.gqa_prefill_paged(q, s.kb, s.vb, s.pool, 2, rows, 4, 2, HD, 20, seq_rows=s.seq_rows, out=out)  # noqa: E731
    for first in (8, rows * nq - 8, rows * nq, rows * nq + nq, 2 * rows * nq - 8):
        with pytest.raises(tb.TangqError):
            attend_to(part(first, rows * nq))
    for first in (0, 2 * rows * nq):
        attend_to(part(first, rows * nq))
    dev.sync()


@pytest.mark.parametrize("form", ["bf16", "q4"])
def test_as_many_parts_as_there_may_be(dev, form):
    """A tile's keys in 32 parts, 31 of 10 or 11 blocks, and two sequences of which one has fewer blocks than parts."""
    for lens, counts in (([20011], [3]), ([9000, 40], [2, 5])):
        s = Sequences(4, 1, 64, lens, counts, 49, form).put(dev)
        got = s.prefill().to_vec()
        dev.sync()
        check_attention(got, *s.reference(), terms=1)
