"""What the page pool, the paged attention and the log probabilities refuse before a GPU is asked, and the pages' definition in plain Python."""
import ctypes as C

import numpy as np
import pytest

from pages_util import Pool, Refused


@pytest.fixture(scope="module")
def tb():
    import tang_b200
    from tang_b200 import _build

    _build.build_library()
    tang_b200.load()
    return tang_b200


class NoDevice:
    """Stands in for a device handle: whoever reaches the library fails."""

    def __getattr__(self, name):
        raise AssertionError(f"the library was called: {name}")


def test_null_handles(tb):
    L = tb.load()
    z = C.c_void_p()
    bad = tb._lib.TQ_EINVAL
    assert L.tq_pages_extend(z, z, z, 1) == bad and L.tq_pages_fork(z, z, z, z, 1) == bad and L.tq_pages_free(z, z, 1) == bad
    assert L.tq_pages_compact(z, z) == bad and L.tq_pages_destroy(z) == tb._lib.TQ_OK
    assert L.tq_pages_create(z, 1, 16, 1, 1, z, z, z, C.byref(z)) == bad
    assert L.tq_gqa_decode_paged(z, z, z, z, z, z, 1, z, z, 0, 0, 8, 2, 128, 1, z, 0) == bad
    assert L.tq_token_logprobs(z, z, 0, 0, 1, 1, 1, z, 0, 0, z, z, z, z) == bad


def test_sizes_are_checked_before_the_call(tb):
    dev = tb.QuantComputeDevice.__new__(tb.QuantComputeDevice)
    dev._ctx = None
    dev.alloc = dev.upload = NoDevice
    buf = lambda n, dt=tb.I32: tb.Buffer(dev, 64, n, dt, owns=False)
    for kw in ({"refs": buf(5)}, {"tables": buf(7)}, {"lens": buf(3)}, {"refs": buf(4, tb.F32)}):
        with pytest.raises(tb.TangqError):
            tb.PagePool(dev, 4, 16, 2, 3, **kw)
    with pytest.raises(tb.TangqError):
        dev.token_logprobs(buf(10, tb.F32), 2, 6)
    with pytest.raises(tb.TangqError):
        dev.token_logprobs(buf(12, tb.F32), 2, 6, tokens=buf(3), n_tokens=2)
    with pytest.raises(tb.TangqError):
        dev.token_logprobs(buf(12, tb.F32), 2, 6, top=3, out=tb.TokenLogprobs(entropy=buf(2, tb.F32), top_ids=buf(5), top_logprobs=buf(6, tb.F32)))
    pool = tb.PagePool.__new__(tb.PagePool)
    pool.dev, pool.n_pages, pool.page_rows, pool.handle = dev, 2, 16, 0
    ok = dict(q=buf(8 * 128, tb.BF16), k_pages=buf(2 * 16 * 256, tb.BF16), v_pages=buf(2 * 16 * 256, tb.BF16), pool=pool, batch=1, n_heads=8, n_kv_heads=2, head_dim=128,
              max_len=5)
    for kw in ({"q": buf(7 * 128, tb.BF16)}, {"k_pages": buf(16, tb.BF16)}, {"v_pages": buf(16, tb.BF16)}, {"batch": 2}, {"seqs": buf(0)}, {"group_starts": buf(1), "n_groups": 1},
               {"group_starts": buf(1), "shared": buf(1), "n_groups": 2}, {"out": buf(9, tb.BF16)}):
        with pytest.raises(tb.TangqError):
            dev.gqa_decode_paged(**{**ok, **kw})


def test_the_definition_keeps_its_counts():
    rng = np.random.default_rng(0)
    for _ in range(40):
        p = Pool(30, 16, 6, 8)
        for _ in range(60):
            s = rng.permutation(6)[:rng.integers(1, 7)].tolist()
            before = (p.refs.copy(), p.tables.copy(), p.lens.copy())
            try:
                rng.choice([lambda: p.extend(s, rng.integers(0, 40, len(s)).tolist()), lambda: p.free(s), p.compact,
                            lambda: p.fork(rng.integers(0, 6, len(s)).tolist(), s)])()
            except Refused:
                assert all(np.array_equal(a, b) for a, b in zip(before, (p.refs, p.tables, p.lens)))
            p.sound()


def test_types_are_checked_before_the_call(tb):
    """A buffer with enough elements of a smaller type has too few bytes."""
    dev = tb.QuantComputeDevice.__new__(tb.QuantComputeDevice)
    dev._ctx, dev._L = None, NoDevice()
    dev.alloc = dev.upload = NoDevice
    buf = lambda n, dt=tb.I32: tb.Buffer(dev, 64, n, dt, owns=False)
    logits, out = buf(12, tb.F32), lambda **kw: tb.TokenLogprobs(**{**dict(logprobs=buf(2, tb.F32), entropy=buf(2, tb.F32), top_ids=buf(6), top_logprobs=buf(6, tb.F32)), **kw})
    for kw in (dict(tokens=buf(2, tb.U8)), dict(tokens=buf(2, tb.F64)), dict(out=out(logprobs=buf(2, tb.BF16))), dict(out=out(entropy=buf(2, tb.U8))),
               dict(out=out(top_ids=buf(6, tb.I8))), dict(out=out(top_logprobs=buf(6, tb.BF16)))):
        with pytest.raises(tb.TangqError, match="type"):
            dev.token_logprobs(**{**dict(logits=logits, rows=2, cols=6, tokens=buf(2), top=3, out=out()), **kw})
    pool = tb.PagePool.__new__(tb.PagePool)
    pool.dev, pool.n_pages, pool.page_rows, pool.handle = dev, 2, 16, 0
    ok = dict(q=buf(8 * 128, tb.BF16), k_pages=buf(2 * 16 * 256, tb.BF16), v_pages=buf(2 * 16 * 256, tb.BF16), pool=pool, batch=1, n_heads=8, n_kv_heads=2, head_dim=128,
              max_len=5, seqs=buf(1), group_starts=buf(1), shared=buf(1), n_groups=1, max_shared=1, out=buf(8 * 128, tb.BF16))
    for kw in ({"q": buf(8 * 128, tb.U8)}, {"k_pages": buf(2 * 16 * 256, tb.U8)}, {"v_pages": buf(2 * 16 * 256, tb.F32)}, {"seqs": buf(1, tb.U8)}, {"group_starts": buf(1, tb.I8)},
               {"shared": buf(1, tb.BF16)}):
        with pytest.raises(tb.TangqError, match="type"):
            dev.gqa_decode_paged(**{**ok, **kw})
    model = tb.LlamaModel.__new__(tb.LlamaModel)
    model.dev, model.handle, model.cfg = dev, 0, tb.LlamaConfig(vocab=6)
    ok = dict(token_ids=buf(1), pool=pool, batch=1, max_len=5, logits=logits, seqs=buf(1), group_starts=buf(1), shared=buf(1), n_groups=1)
    for kw in ({"token_ids": buf(1, tb.U8)}, {"logits": buf(12, tb.BF16)}, {"seqs": buf(1, tb.U8)}, {"group_starts": buf(1, tb.F64)}, {"shared": buf(1, tb.U8)}):
        with pytest.raises(tb.TangqError, match="type"):
            model.decode_paged(**{**ok, **kw})
    for used in (buf(1, tb.U8), buf(0)):
        with pytest.raises(tb.TangqError):
            pool.compact(used)
