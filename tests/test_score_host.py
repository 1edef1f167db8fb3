"""``Engine.score`` without a GPU: which rows' logits are taken, which token each is rated for, and in what portions."""
import numpy as np
import pytest

from test_tofazen_host import _FakeDevice, _FakeModel


class _RatingDevice(_FakeDevice):
    """'Log probability' of token t under the row [token, position, slot]: 100 t + 10 position + token; the likeliest token is the slot."""

    def upload(self, data, dtype):
        buf = self.alloc(len(data), dtype)
        self.upload_into(buf, data)
        return buf

    def token_logprobs(self, logits, rows, cols, tokens, top=0, entropy=True):
        import tang_b200 as tb

        x, t = self._at(logits).reshape(rows, cols), self._at(tokens)
        assert cols == 3 and len(t) == rows and not entropy
        wrap = lambda v, n, d: _Answer(np.asarray(v))
        return tb.TokenLogprobs(wrap(100 * t + 10 * x[:, 1] + x[:, 0], rows, tb.F32), None, wrap(np.repeat(x[:, 2:], top, 1).reshape(-1), rows, tb.I32),
                                wrap(np.zeros(rows * top), rows, tb.F32))


class _Answer:
    def __init__(self, v):
        self.v = v

    def to_vec(self):
        return self.v


@pytest.mark.parametrize("score_rows", [1, 2, 3, 64])
def test_every_token_but_the_first_is_rated(score_rows):
    from tang_b200 import Engine

    m = _FakeModel()
    m.dev = _RatingDevice()
    e = Engine(m)
    assert e.score_rows == (1 << 28) // 3
    e.score_rows = score_rows
    a, b, c = e.score([("a", [2, 1, 0, 2, 1]), ("b", [1]), ("c", [0, 2, 2])], top=2)
    assert a["logprobs"].tolist() == [102, 11, 220, 132] and a["top_ids"].tolist() == [[e.pool.slot["a"]] * 2] * 4
    assert b["logprobs"].shape == (0,) and b["top_ids"].shape == (0, 2)
    assert c["logprobs"].tolist() == [200, 212] and c["top_logprobs"].shape == (2, 2)
    assert max(m.steps) <= score_rows and sum(m.steps) == 9
    # what a request holds already comes before
    assert e.score([("a", [0, 2])])[0]["logprobs"].tolist() == [250] and e.pool.length["a"] == 7
    assert e.step([("b", [2], [0])]).tolist() == [[2, 1, e.pool.slot["b"]]]


def test_bad_scores_are_refused():
    from tang_b200 import Engine, TangqError

    e = Engine(_FakeModel())
    for bad, top in (([("a", [3, 0])], 0), ([("a", [])], 0), ([("a", [1]), ("a", [1])], 0), ([("a", [1] * 65)], 0), ([("a", [1, 1])], 4), ([("a", [1, 1])], -1)):
        with pytest.raises(TangqError):
            e.score(bad, top)
    assert not e.pool.slot
