"""Pages of a cache (tq_pages_*) against their definition in plain Python: state, rows copied, refusals, graphs."""
import numpy as np
import pytest

from pages_util import Pool, Refused

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    import tang_b200

    d = tang_b200.QuantComputeDevice(0)
    yield d
    d.close()


class Both:
    """A pool on the device and its definition, with caches whose rows carry their first place."""

    def __init__(self, dev, n_pages, P, n_seqs, ld, n_arrays=3, row=8):
        import tang_b200 as tb

        self.dev, self.want, self.P = dev, Pool(n_pages, P, n_seqs, ld), P
        rng = np.random.default_rng(n_pages)
        self.data = rng.integers(0, 1 << 16, (n_arrays, n_pages, P, row)).astype(np.uint16)
        self.bufs = [dev.upload(a, tb.BF16) for a in self.data]
        self.pool = tb.PagePool(dev, n_pages, P, n_seqs, ld, self.bufs)

    def copy(self, copies):
        for a, b, n in copies:
            self.data[:, b, :n] = self.data[:, a, :n]

    def check(self):
        self.dev.sync()
        refs, tables, lens = self.pool.state()
        assert np.array_equal(refs, self.want.refs) and np.array_equal(tables, self.want.tables) and np.array_equal(lens, self.want.lens)
        self.want.sound()
        for b, d in zip(self.bufs, self.data):
            assert np.array_equal(b.to_vec().reshape(d.shape), d)

    def extend(self, seqs, counts=None):
        self.pool.extend(seqs, counts=counts)
        self.copy(self.want.extend(list(seqs), counts))

    def fork(self, src, dst, keep=None):
        self.pool.fork(src, dst, keep=keep)
        self.want.fork(list(src), list(dst), keep)

    def free(self, seqs):
        self.pool.free(seqs)
        self.want.free(list(seqs))

    def compact(self):
        self.pool.compact()
        self.copy(self.want.compact()[0])


def test_samples_of_one_prompt(dev):
    b = Both(dev, 40, 16, 6, 8)
    b.extend([0], [37])
    b.check()
    b.fork([0, 0, 0], [1, 2, 3])
    b.check()
    b.extend([1, 3, 2])                # three copies: the prompt keeps its own last page
    b.check()
    b.free([0])
    b.fork([1], [0])
    b.extend([1, 0])                   # the only two holders: the second keeps the page
    b.check()
    b.extend([0, 1, 2, 3], [0, 11, 16, 64])
    b.check()
    b.free([2])
    b.compact()
    b.check()
    b.extend([4], [1])
    b.fork([4, 1], [5, 2], keep=[0, 20])
    b.check()


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("n_pages,P,n_seqs,ld,n_arrays,row", [(50, 16, 9, 12, 2, 8), (300, 32, 40, 20, 5, 24), (9000, 16, 70, 200, 1, 8), (33, 256, 5, 9, 2, 64)])
def test_any_order_of_calls(dev, n_pages, P, n_seqs, ld, n_arrays, row, seed):
    rng = np.random.default_rng(seed * 1000 + n_pages)
    b = Both(dev, n_pages, P, n_seqs, ld, n_arrays, row)
    for _ in range(25):
        what = rng.choice(["extend", "extend", "extend", "fork", "free", "compact"])
        seqs = rng.permutation(n_seqs)[:rng.integers(1, n_seqs + 1)].tolist()
        if what == "extend":
            counts = (rng.integers(0, 3, len(seqs)) * rng.integers(1, 2 * P, len(seqs))).tolist()
            trial = Pool(n_pages, P, n_seqs, ld)
            trial.refs, trial.tables, trial.lens = b.want.refs, b.want.tables, b.want.lens
            try:
                trial.extend(seqs, counts)
            except Refused:
                continue
            b.extend(seqs, counts)
        elif what == "fork":
            empty, held = [s for s in seqs if not b.want.lens[s]], [s for s in range(n_seqs) if b.want.lens[s]]
            if empty and held:
                src = rng.choice(held, len(empty)).tolist()
                b.fork(src, empty, None if rng.random() < 0.5 else rng.integers(0, P * 4, len(empty)).tolist())
        elif what == "free":
            b.free(seqs[:max(1, len(seqs) // 2)])
        else:
            b.compact()
    b.check()


def test_a_thousand_sequences(dev):
    b = Both(dev, 5000, 16, 1024, 6, 1, 8)
    every = np.random.default_rng(0).permutation(1024).tolist()
    b.extend([3], [40])
    b.fork([3] * 1023, [s for s in every if s != 3])
    b.extend(every)
    b.check()
    b.extend(every, [(7 * s) % 33 for s in every])
    b.free(every[:1000])
    b.compact()
    b.check()


def test_large_rows_and_offsets_behind_32_bits(dev):
    """Pages further than 2^32 bytes from the array's start."""
    import tang_b200 as tb

    n_pages, P, row = 3000, 64, 2048 * 8                     # 1 MiB a page in two arrays, 2 GiB behind page 2048
    bufs = [dev.alloc(n_pages * P * row, tb.U8) for _ in range(2)]
    for buf in bufs:
        dev.memset(buf, 1)
    refs = np.zeros(n_pages, np.int32)
    tables = np.full((2, 4), -1, np.int32)
    tables[0, :2], refs[[n_pages - 1, 5]] = [n_pages - 1, 5], 1
    refs[:5] = refs[6:n_pages - 9] = 1                       # (only the last few are free)
    state = [dev.upload(a, tb.I32) for a in (refs, tables, np.array([70, 0], np.int32))]
    pool = tb.PagePool(dev, n_pages, P, 2, 4, bufs, *state)
    pages = [tb.Buffer(dev, buf.ptr + (n_pages - 1) * P * row, P * row, tb.U8, owns=False) for buf in bufs]
    for i, page in enumerate(pages):
        dev.memset(page, 7 + i)
    pool.fork([0], [1], keep=[33])                           # page n_pages - 1, partly filled
    pool.extend([1])
    dev.sync()
    refs, tables, lens = pool.state()
    to = n_pages - 9
    assert tables[1].tolist() == [to, -1, -1, -1] and lens.tolist() == [70, 34] and refs[to] == 1 and refs[n_pages - 1] == 1
    for i, buf in enumerate(bufs):
        got = tb.Buffer(dev, buf.ptr + to * P * row, P * row, tb.U8, owns=False).to_vec().reshape(P, row)
        assert (got[:33] == 7 + i).all() and (got[33:] == 1).all()
    pool.destroy()


def test_refused_calls_change_nothing(dev):
    import tang_b200 as tb

    b = Both(dev, 12, 16, 4, 6)
    b.extend([0, 1], [40, 16])
    b.fork([0], [2])
    b.check()

    def refused(call, status):
        call()
        with pytest.raises(tb.TangqError) as e:
            dev.sync()
        assert e.value.status == status
        b.check()

    bad, full = tb._lib.TQ_EINVAL, tb._lib.TQ_ENOMEM
    refused(lambda: b.pool.extend([0, 4]), bad)
    refused(lambda: b.pool.extend([-1]), bad)
    refused(lambda: b.pool.extend([1, 0, 1]), bad)
    refused(lambda: b.pool.extend([0], counts=[-1]), bad)
    refused(lambda: b.pool.extend([1], counts=[81]), full)                   # the table has six entries
    refused(lambda: b.pool.extend([1], counts=[2 ** 31 - 1]), full)
    refused(lambda: b.pool.extend([3, 1, 0, 2], counts=[64, 48, 16, 16]), full)
    refused(lambda: b.pool.fork([0], [1]), bad)                              # not empty
    refused(lambda: b.pool.fork([0, 0], [3, 3]), bad)
    refused(lambda: b.pool.fork([3], [3]), bad)
    refused(lambda: b.pool.fork([0, 3], [3, 3]), bad)
    refused(lambda: b.pool.fork([7], [3]), bad)
    refused(lambda: b.pool.fork([0], [3], keep=[-5]), bad)
    refused(lambda: b.pool.free([0, 0]), bad)
    refused(lambda: b.pool.free([2, 9]), bad)
    b.free([2])
    b.extend([1], [1])
    b.check()
    for args in ((0, 16, 1, 1), (4, 24, 1, 1), (4, 8, 1, 1), (4, 2048, 1, 1), (4, 16, 0, 1), (4, 16, 1, 0)):
        with pytest.raises(tb.TangqError):
            tb.PagePool(dev, *args)
    bare = tb.PagePool(dev, 4, 16, 2, 2)
    for call in (lambda: bare.extend([0]), bare.compact, lambda: bare.set_arrays([]), lambda: bare.set_arrays([dev.alloc(4 * 16 * 4, tb.BF16)]),
                 lambda: b.pool.free(list(range(1025)))):
        with pytest.raises(tb.TangqError):
            call()
    bare.free([0, 1])
    dev.sync()


def test_calls_recorded_in_a_graph(dev):
    """Forty tokens for three samples: one recorded step, replayed."""
    import tang_b200 as tb

    b = Both(dev, 40, 16, 4, 8)
    b.extend([0], [21])
    b.fork([0, 0], [1, 2])
    seqs = dev.upload(np.array([2, 0, 1], np.int32), tb.I32)
    b.pool.extend(seqs)
    b.copy(b.want.extend([2, 0, 1]))
    dev.sync()
    dev.begin_capture()
    b.pool.extend(seqs)
    g = dev.end_capture()
    for _ in range(40):
        g.launch()
        b.copy(b.want.extend([2, 0, 1]))
    b.check()
    g.free()


@pytest.mark.parametrize("page", [-1, 12, 2 ** 31 - 1, -2 ** 31])
def test_a_table_with_a_page_that_does_not_exist_changes_nothing(dev, page):
    """Of a caller's tables: the second of three sequences names such a page behind good ones."""
    import tang_b200 as tb

    refs, tables, lens = np.zeros(12, np.int32), np.full((6, 4), -1, np.int32), np.array([40, 33, 5, 0, 0, 0], np.int32)
    tables[0, :3], tables[1, :3], tables[2, 0] = [7, 1, 3], [2, 0, page], 9
    refs[[7, 1, 3, 2, 0, 9]] = 1
    data = np.random.default_rng(0).integers(0, 1 << 16, (12, 16, 8)).astype(np.uint16)
    caches = dev.upload(data, tb.BF16)
    pool = tb.PagePool(dev, 12, 16, 6, 4, [caches], *(dev.upload(a, tb.I32) for a in (refs, tables, lens)))
    for call in (lambda: pool.fork([0, 1, 2], [3, 4, 5]), lambda: pool.fork([1], [4], keep=[33]), lambda: pool.free([0, 1, 2]), lambda: pool.extend([0, 1, 2])):
        call()
        with pytest.raises(tb.TangqError) as e:
            dev.sync()
        assert e.value.status == tb._lib.TQ_EINVAL
        assert all(np.array_equal(a, b) for a, b in zip(pool.state(), (refs, tables, lens))) and np.array_equal(caches.to_vec().reshape(data.shape), data)
    pool.fork([0, 1], [3, 4], keep=[40, 32])           # (the page is not among these)
    pool.free([0, 3, 4, 2])
    dev.sync()
    assert pool.state()[2].tolist() == [0, 33, 0, 0, 0, 0] and pool.state()[0].tolist() == [1, 0, 1] + [0] * 9
    pool.destroy()


def test_a_graph_over_a_pool_that_is_gone_is_refused(dev):
    """Destroyed, or with other arrays; graphs over other pools and over none go on."""
    import tang_b200 as tb

    seqs, x = dev.upload(np.array([0], np.int32), tb.I32), dev.alloc(16 * 128, tb.BF16)
    pools = [tb.PagePool(dev, 4, 16, 2, 4, [dev.alloc(4 * 16 * 8, tb.BF16)]) for _ in range(7)]
    kv, out = dev.alloc(4 * 16 * 128, tb.BF16), dev.alloc(128, tb.BF16)
    dev.memset(kv, 0)
    dev.memset(x, 0)
    q = tb.Buffer(dev, x.ptr, 128, tb.BF16, owns=False)
    attend = lambda p: dev.gqa_decode_paged(q, kv, kv, p, 1, 1, 1, 128, 16, out=out)
    uses = [lambda p: p.extend(seqs), lambda p: p.fork(seqs, seqs, 1), lambda p: p.free(seqs), lambda p: p.compact(), attend,
            lambda p: (p.free(seqs), attend(p), attend(pools[6]))]
    attend(pools[0])                                   # (workspaces)
    dev.sync()

    def record(call):
        dev.begin_capture()
        call()
        return dev.end_capture()

    graphs = [record(lambda: use(p)) for use, p in zip(uses, pools)]
    both, none = record(lambda: [p.free(seqs) for p in pools[:6]]), record(lambda: dev.memset(out, 0))
    last = record(lambda: pools[6].free(seqs))
    for i, p in enumerate(pools[:6]):
        if i % 2:
            p.set_arrays([dev.alloc(4 * 16 * 8, tb.BF16)])
        else:
            p.destroy()
        with pytest.raises(tb.TangqError, match="pool of pages"):
            graphs[i].launch()
        with pytest.raises(tb.TangqError, match="pool of pages"):
            both.launch()
        last.launch()
        none.launch()
        if i < 5:
            fresh = tb.PagePool(dev, 4, 16, 2, 4)      # (one that may stand where the old one stood)
            with pytest.raises(tb.TangqError, match="pool of pages"):
                graphs[i].launch()
            fresh.destroy()
        dev.sync()
    for g in (*graphs, both, none, last):
        g.free()
    for p in pools:
        p.destroy()


def test_a_pool_that_outlives_its_handle():
    """Calls are refused, and it can still be destroyed."""
    import tang_b200 as tb

    d = tb.QuantComputeDevice(0)
    pools = [tb.PagePool(d, 4, 16, 2, 4) for _ in range(3)]
    seqs = d.upload(np.array([0], np.int32), tb.I32)
    pools[1].destroy()
    handles, L = [tb._lib.C.c_void_p(p.handle) for p in pools], d._L
    d.close()
    z = tb._lib.C.c_void_p(seqs.ptr)
    for h in (handles[0], handles[2]):
        assert L.tq_pages_extend(h, z, None, 1) == L.tq_pages_fork(h, z, z, None, 1) == L.tq_pages_free(h, z, 1) == L.tq_pages_compact(h, None) == tb._lib.TQ_EINVAL
        assert L.tq_pages_arrays(h, None, 1, 16) == tb._lib.TQ_EINVAL
    for p in pools:
        p.destroy()
        p.destroy()


def test_more_pages_than_32_bits_count(dev):
    """What 1024 sequences ask for together: 2^31, 2^32 and 2^32 + 1 pages, of tables that are large enough."""
    import tang_b200 as tb

    ld, n = (1 << 22) + 1, 1024
    pool = tb.PagePool(dev, 64, 16, n, ld, [dev.alloc(64 * 16 * 8, tb.BF16)])
    seqs, small = dev.upload(np.arange(n, dtype=np.int32), tb.I32), [3, 5]
    pool.extend(small, counts=[20, 7])
    pool.fork([3], [9])                                # (a partly filled page that would be copied)
    dev.sync()
    refs, lens = pool.refs.to_vec(), pool.lens.to_vec()
    row = lambda s: tb.Buffer(dev, pool.tables.ptr + 4 * s * ld, 4, tb.I32, owns=False).to_vec().tolist()
    rows = [row(s) for s in (0, 3, 5, 9, n - 1)]
    for pages, more in ((1 << 21, 0), (1 << 22, 0), (1 << 22, 1)):
        counts = np.full(n, 16 * pages, np.int32)
        counts[[3, 5, 9]] -= 32                        # (with what they have, and one copy: five pages too few, which five others ask for)
        counts[10:15 + more] += 16
        pool.extend(seqs, n, counts=dev.upload(counts, tb.I32))
        with pytest.raises(tb.TangqError) as e:
            dev.sync()
        assert e.value.status == tb._lib.TQ_ENOMEM
        assert np.array_equal(pool.refs.to_vec(), refs) and np.array_equal(pool.lens.to_vec(), lens) and [row(s) for s in (0, 3, 5, 9, n - 1)] == rows
    pool.extend([9])
    dev.sync()
    assert pool.lens.to_vec()[9] == 21
    pool.destroy()


def test_a_recorded_call_takes_its_lists_from_the_device(dev):
    """A list of the host's is refused while a graph is recorded, and the recording goes on."""
    import tang_b200 as tb

    b = Both(dev, 20, 16, 3, 8)
    b.extend([0], [5])
    seqs = dev.upload(np.array([0], np.int32), tb.I32)
    dev.sync()
    dev.begin_capture()
    for call in (lambda: b.pool.extend([0]), lambda: b.pool.extend(seqs, counts=[1]), lambda: b.pool.fork(seqs, [1]), lambda: b.pool.free([0])):
        with pytest.raises(tb.TangqError, match="recorded"):
            call()
    b.pool.extend(seqs)
    g = dev.end_capture()
    for _ in range(3):
        g.launch()
        b.copy(b.want.extend([0]))
    b.check()
    g.free()
    b.extend([0])
    b.check()
