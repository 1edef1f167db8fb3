"""What the calls over packed rows and pages of 4 bits refuse before a GPU is asked, and the rule of 4 bits in plain numbers."""
import ctypes as C

import numpy as np
import pytest

from packed_util import HD, pack, row_bytes


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
    L, z, bad = tb.load(), C.c_void_p(), tb._lib.TQ_EINVAL
    assert L.tq_kv_append_paged(z, z, 0, 0, z, z, 1, z, z, z, 1, 1, 8, 2, 128, z, z, z, 0) == bad
    assert L.tq_kv_read_paged(z, z, z, 0, z, z, z, 1, 1, 2, 128, z, z) == bad
    assert L.tq_gqa_prefill_paged(z, z, z, z, 0, z, z, z, 1, 1, 8, 2, 128, 1, z) == bad
    assert L.tq_gqa_decode_paged_q4(z, z, z, z, z, z, 1, 8, 2, 128, 1, z) == bad


def test_row_bytes(tb):
    for n in range(1, 40):
        assert tb.load().tq_q4_row_bytes(n) == tb.q4_row_bytes(n) == row_bytes(n) and row_bytes(n) % 16 == 0 and row_bytes(n) - 72 * n in (0, 8)


def test_sizes_and_types_are_checked_before_the_call(tb):
    dev = tb.QuantComputeDevice.__new__(tb.QuantComputeDevice)
    dev._ctx, dev._L = None, NoDevice()
    dev.alloc = dev.upload = NoDevice
    buf = lambda n, dt=tb.I32: tb.Buffer(dev, 64, n, dt, owns=False)  # noqa: E731
    pool = tb.PagePool.__new__(tb.PagePool)
    pool.dev, pool.n_pages, pool.page_rows, pool.handle = dev, 2, 16, 0
    pages, bytes_ = buf(32 * 256, tb.BF16), buf(32 * 144, tb.U8)
    common = dict(pool=pool, batch=2, rows=5, n_kv_heads=2, head_dim=128, seq_rows=buf(3), seqs=buf(2))
    for k in (pages, bytes_):
        both = dict(k_pages=k, v_pages=k)
        append = dict(x=buf(5 * 12 * 128, tb.F32), cos=buf(640, tb.F32), sin=buf(640, tb.F32), n_heads=8, q_out=buf(5 * 1024, tb.BF16), **common, **both)
        read = dict(k_out=buf(5 * 256, tb.BF16), v_out=buf(5 * 256, tb.BF16), **common, **both)
        prefill = dict(q=buf(5 * 1024, tb.BF16), n_heads=8, max_len=5, out=buf(5 * 1024, tb.BF16), **common, **both)
        other = bytes_ if k is pages else pages
        shared = ({"seqs": buf(1)}, {"seqs": buf(2, tb.U8)}, {"seq_rows": buf(2)}, {"seq_rows": buf(3, tb.F32)}, {"seq_rows": None}, {"v_pages": other}, {"k_pages": other},
                  {"k_pages": buf(k.n - 1, k.dtype)}, {"v_pages": buf(k.n + 16, k.dtype)}, {"k_pages": buf(k.n, tb.F32), "v_pages": buf(k.n, tb.F32)})
        for call, ok, own in ((dev.kv_append_paged, append, ({"x": buf(5 * 12 * 128 - 1, tb.F32)}, {"ldx": 2000}, {"cos": buf(600, tb.F32)}, {"cos": buf(640, tb.BF16)},
                                                             {"sin": buf(640)}, {"q_out": buf(5 * 1024 - 1, tb.BF16)}, {"q_out": buf(5 * 1024, tb.U8)})),
                              (dev.kv_read_paged, read, ({"k_out": buf(9, tb.BF16)}, {"v_out": buf(5 * 256, tb.U8)}, {"v_out": buf(5 * 256 - 1, tb.BF16)})),
                              (dev.gqa_prefill_paged, prefill, ({"q": buf(9, tb.BF16)}, {"q": buf(5 * 1024, tb.U8)}, {"out": buf(9, tb.BF16)}, {"out": buf(5 * 1024, tb.I8)}))):
            for kw in (*shared, *own):
                with pytest.raises(tb.TangqError):
                    call(**{**ok, **kw})
    ok = dict(q=buf(2 * 1024, tb.BF16), k_pages=bytes_, v_pages=bytes_, pool=pool, batch=2, n_heads=8, n_kv_heads=2, head_dim=128, max_len=5, seqs=buf(2),
              out=buf(2 * 1024, tb.BF16))
    for kw in ({"k_pages": pages, "v_pages": pages}, {"q": buf(9, tb.BF16)}, {"q": buf(2 * 1024, tb.U8)}, {"out": buf(2 * 1024, tb.F32)}, {"out": buf(1, tb.BF16)}, {"seqs": buf(1)}):
        with pytest.raises(tb.TangqError):
            dev.gqa_decode_paged_q4(**{**ok, **kw})


def test_what_reaches_the_library_of_buffers_that_may_be_missing(tb):
    """No sequences, empty ones and present ones: null or the buffer's address, which the declared types have to take."""
    seen = []

    class Library:
        def __getattr__(self, name):
            types = getattr(tb.load(), name).argtypes

            def call(*args):
                assert len(args) == len(types)
                for t, a in zip(types[1:], args[1:]):
                    t.from_param(a)
                seen.append((name, args))
                return 0
            return call

    dev = tb.QuantComputeDevice.__new__(tb.QuantComputeDevice)
    dev._ctx, dev._L = None, Library()
    at = iter(range(64, 1 << 20, 64))
    buf = lambda n, dt=tb.I32: tb.Buffer(dev, next(at), n, dt, owns=False)  # noqa: E731
    pool = tb.PagePool.__new__(tb.PagePool)
    pool.dev, pool.n_pages, pool.page_rows, pool.handle = dev, 2, 16, 0
    k, v, q, out, table = buf(32 * 144, tb.U8), buf(32 * 144, tb.U8), buf(2048, tb.BF16), buf(2048, tb.BF16), buf(640, tb.F32)
    for batch, seqs, starts in ((2, None, None), (2, buf(2), buf(3)), (2, None, buf(3)), (0, buf(0), buf(1)), (0, buf(0), None)):
        seen.clear()
        packed = dict(seqs=seqs, seq_rows=starts)
        dev.kv_append_paged(buf(batch * 12 * 128, tb.F32), table, table, pool, k, v, batch, batch, 8, 2, 128, q_out=q, **packed)
        dev.kv_read_paged(k, v, pool, batch, batch, 2, 128, k_out=q, v_out=out, **packed)
        dev.gqa_prefill_paged(q, k, v, pool, batch, batch, 8, 2, 128, 9, out=out, **packed)
        dev.gqa_decode_paged_q4(q, k, v, pool, batch, 8, 2, 128, 9, seqs=seqs, out=out)
        assert [n for n, _ in seen] == ["tq_kv_append_paged", "tq_kv_read_paged", "tq_gqa_prefill_paged", "tq_gqa_decode_paged_q4"]
        s, r = (None if b is None else b.ptr for b in (seqs, starts))
        assert [a[i:i + 2] for (_, a), i in zip(seen, (8, 5, 6))] == [(s, r)] * 3 and seen[3][1][5] == s


def test_four_bits_of_ordinary_numbers():
    """Values are bf16 numbers, within half a step (the scale, up to a sixteenth more than the largest / 7) of what they stand for."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 3, HD)) * np.exp(rng.uniform(-20, 20, (50, 3, 1)))).astype(np.float32)
    raw, v = pack(x)
    amax = np.abs(x).reshape(50, 3, 4, 32).max(-1)
    assert raw.shape == (50, row_bytes(3)) and (raw[:, 216:] == 0).all()
    assert np.array_equal(v, ((v.astype(np.float32).view(np.uint32) & 0xFFFF0000).view(np.float32)))
    assert (np.abs(v - x).reshape(50, 3, 4, 32).max(-1) <= amax / 7 * (1 + 1 / 16) / 2 * (1 + 2.0 ** -20)).all()


def test_the_scale_from_a_product():
    """What the kernel computes instead of a division (a product with a number just below 1 / 7, rounded up to 5 bits, and one step more where seven times
    that is still below the largest magnitude) is the rule: at the borders, beside them and elsewhere."""
    f = np.float32
    rng = np.random.default_rng(0)
    k = (np.arange(16, 33)[:, None] * 7.0 * 2.0 ** np.arange(-90, 110)[None]).ravel().astype(f)
    a = np.concatenate([np.exp(rng.uniform(-60, 80, 200000)).astype(f), *((k.view(np.int32) + np.int32(d)).view(f) for d in range(-20, 21))])
    a = a[(a >= 2.0 ** -100) & (a < 2.0 ** 120)]
    s = (((a * f(0.14285707)).view(np.uint32) + np.uint32(0x7FFFF)) & np.uint32(0xFFF80000)).view(f)
    s = np.where(f(7) * s < a, (s.view(np.uint32) + np.uint32(0x80000)).view(f), s)
    frac, e = np.frexp(a.astype(np.float64) / 7)
    assert np.array_equal(s.astype(np.float64), np.ldexp(np.ceil(frac * 32) / 32, e))
