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
