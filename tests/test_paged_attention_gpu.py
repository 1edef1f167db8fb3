"""Decode attention over pages (tq_gqa_decode_paged) against 64 bits: lengths from nothing to long ones, groups that share a prefix, every page
size and group of heads, rows behind a sequence's end that hold NaN, pages that do not exist, refusals."""
import numpy as np
import pytest

from util import bf16_round

pytestmark = pytest.mark.gpu
HD = 128
NAN = 0x7FC0


@pytest.fixture(scope="module")
def dev():
    import tang_b200

    d = tang_b200.QuantComputeDevice(0)
    yield d
    d.close()


class Setup:
    """Sequences in a pool: `groups` is a list of (shared positions, lengths of the members); every row that nobody holds is NaN."""

    def __init__(self, nh, nkv, P, groups, seed, extra=3, q_std=1.5, order=None):
        rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.P = nh, nkv, P
        lens = np.array([n for _, m in groups for n in m])
        self.B, self.lens = len(lens), lens
        held = -(-lens // P)
        self.ld = max(1, int(held.max())) + 1
        self.starts = np.cumsum([0] + [len(m) for _, m in groups]).astype(np.int32)
        self.shared = np.array([s for s, _ in groups], np.int32)
        n_pages = int(held.sum()) + extra
        free = rng.permutation(n_pages).tolist()
        self.tables = np.full((self.B, self.ld), -1, np.int32)
        for g, (s, m) in enumerate(groups):
            first = int(self.starts[g])
            whole = s // P
            for b in range(first, first + len(m)):
                for j in range(held[b]):
                    share = b > first and j < whole and j < held[first]
                    self.tables[b, j] = self.tables[first, j] if share else free.pop()
        self.n_pages = n_pages
        self.q_bits, self.q = bf16_round((rng.standard_normal((self.B, nh, HD)) * q_std).astype(np.float32))
        self.kv_bits = np.full((2, n_pages, P, nkv, HD), NAN, np.uint16)
        self.kv = np.zeros((2, n_pages, P, nkv, HD), np.float32)
        for b in range(self.B):
            for j in range(held[b]):
                rows = min(P, int(lens[b]) - j * P)
                bits, f = bf16_round(rng.standard_normal((2, rows, nkv, HD)).astype(np.float32))
                page = self.tables[b, j]
                self.kv_bits[:, page, :rows], self.kv[:, page, :rows] = bits.reshape(f.shape), f
        # the part of the shared positions that is no whole page is the same in every member's own page
        for g, (s, m) in enumerate(groups):
            first, whole, rest = int(self.starts[g]), s // P, s % P
            for b in range(first + 1, first + len(m)):
                n = min(rest, int(lens[b]) - whole * P, int(lens[first]) - whole * P)
                if n > 0:
                    for a in (self.kv_bits, self.kv):
                        a[:, self.tables[b, whole], :n] = a[:, self.tables[first, whole], :n]

    def put(self, dev, seqs=None):
        import tang_b200 as tb

        self.dev = dev
        refs = np.zeros(self.n_pages, np.int32)
        np.add.at(refs, self.tables[self.tables >= 0], 1)
        tables, lens = self.tables, self.lens.astype(np.int32)
        n = self.B
        self.seqs = None
        if seqs is not None:           # the batch is these sequences of a larger pool
            n = int(max(seqs)) + 1
            t, l = np.full((n, self.ld), -1, np.int32), np.zeros(n, np.int32)
            t[seqs], l[seqs] = tables, lens
            tables, lens = t, l
            self.seqs = dev.upload(np.array(seqs, np.int32), tb.I32)
        self.state = [dev.upload(a, tb.I32) for a in (refs, tables, lens)]
        self.pool = tb.PagePool(dev, self.n_pages, self.P, n, self.ld, None, *self.state)
        self.qb, self.kb, self.vb = (dev.upload(a.reshape(-1), tb.BF16) for a in (self.q_bits, self.kv_bits[0], self.kv_bits[1]))
        self.gb, self.sb = dev.upload(self.starts, tb.I32), dev.upload(self.shared, tb.I32)
        return self

    def run(self, f32, grouped=True, max_len=None, out=None):
        import tang_b200 as tb

        kw = {"group_starts": self.gb, "shared": self.sb, "n_groups": len(self.shared), "max_shared": int(self.shared.max())} if grouped else {}
        return self.dev.gqa_decode_paged(self.qb, self.kb, self.vb, self.pool, self.B, self.nh, self.nkv, HD, max_len or max(1, int(self.lens.max())), seqs=self.seqs,
                                         out=out, out_dtype=tb.F32 if f32 else tb.BF16, **kw)

    def reference(self):
        """(result, sum of the weights times the values' sizes), 64 bits."""
        out, size = np.zeros((self.B, self.nh, HD)), np.zeros((self.B, self.nh, HD))
        for b in range(self.B):
            n = int(self.lens[b])
            if not n:
                continue
            pages = self.tables[b, :-(-n // self.P)]
            k, v = (self.kv[i, pages].reshape(-1, self.nkv, HD)[:n].astype(np.float64).transpose(1, 0, 2) for i in (0, 1))
            q = self.q[b].astype(np.float64).reshape(self.nkv, -1, HD)
            s = q @ k.transpose(0, 2, 1) / np.sqrt(HD)
            e = np.exp(s - s.max(-1, keepdims=True))
            w = e / e.sum(-1, keepdims=True)
            out[b], size[b] = (w @ v).reshape(self.nh, HD), (w @ np.abs(v)).reshape(self.nh, HD)
        return out, size

    def check(self, got, f32, rows=slice(None)):
        """f32: the weights are two bf16 terms (2^-16 of themselves) and the scores, sums of 128 exact products in f32, are off by 2^-23 of their parts' sum
        per step of 16 (at most 2^-17 here), every sum of up to 2^12 steps likewise: 2^-14 of the sum of |weight value|.  bf16: one term of the weights
        (2^-9) and the result's rounding (2^-9) more."""
        want, size = self.reference()
        got = got.astype(np.float64) if f32 else (got.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        got = got.reshape(want.shape)
        tol = (2.0 ** -14 if f32 else 2.0 ** -14 + 2.0 ** -8) * size + 1e-30
        assert np.isfinite(got[rows]).all()
        err = np.abs(got - want)[rows] / tol[rows]
        assert err.max() <= 1, (err.max(), np.unravel_index(err.argmax(), err.shape))


CASES = {
    "one": (8, 2, 16, [(0, [1])]),
    "nothing": (8, 2, 16, [(0, [0])]),
    "lengths": (8, 2, 16, [(0, [0]), (0, [1]), (0, [15]), (0, [16]), (0, [17]), (0, [63]), (0, [64]), (0, [65]), (0, [127]), (0, [128]), (0, [129]), (0, [700])]),
    "samples": (8, 2, 16, [(64, [65, 70, 64, 100])]),
    "odd prefix": (32, 8, 32, [(135, [136, 300, 135, 140, 136, 190])]),
    "groups": (16, 4, 16, [(0, [5]), (130, [131, 260]), (1, [1, 2, 3]), (600, [601, 640, 700, 601, 601]), (0, [33])]),
    "one to one": (8, 8, 64, [(256, [257, 300, 511]), (129, [129, 129])]),
    "one kv head": (8, 1, 128, [(1024, [1025, 1100] + [1030] * 15)]),
    "three to one": (6, 2, 256, [(700, [701, 900, 777]), (0, [255])]),
    "five to one": (5, 1, 16, [(384, [400] * 30)]),
    "many": (32, 8, 64, [(512, [513 + 7 * i for i in range(64)])]),
    "long": (8, 2, 16, [(0, [9001]), (4096, [4097, 4500]), (0, [3])]),
    "short members": (16, 4, 16, [(512, [600, 100, 0, 513, 511])]),
    "empty first": (16, 4, 16, [(512, [0, 0, 0])]),
    "pages of 1024": (8, 2, 1024, [(1500, [1501, 1600, 2049]), (0, [1024])]),
    "two hundred": (4, 4, 32, [(256, [257 + i % 40 for i in range(200)])]),
}


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("name", list(CASES))
def test_against_64_bits(dev, name, f32):
    s = Setup(*CASES[name], seed=len(name)).put(dev)
    got = s.run(f32).to_vec()
    dev.sync()
    s.check(got, f32)
    alone = s.run(f32, grouped=False).to_vec()
    dev.sync()
    s.check(alone, f32)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("P", [16, 32, 64, 128, 256, 512, 1024])
def test_every_page_size(dev, P, f32):
    s = Setup(8, 2, P, [(3 * P // 2 + 130, [3 * P // 2 + 131, 2 * P + 200, 3 * P + 300])], seed=P).put(dev)
    got = s.run(f32).to_vec()
    dev.sync()
    s.check(got, f32)


@pytest.mark.parametrize("seed", range(12))
def test_drawn_batches(dev, seed):
    rng = np.random.default_rng(seed + 500)
    nkv, group, P = int(rng.choice([1, 2, 3, 8])), int(rng.integers(1, 9)), int(rng.choice([16, 32, 64, 128]))
    groups = []
    for _ in range(rng.integers(1, 7)):
        shared = int(rng.choice([0, 5, 128, 200, 1000]))
        groups.append((shared, [shared + int(rng.integers(0, 400)) + 1 for _ in range(rng.integers(1, 12))]))
    s = Setup(nkv * group, nkv, P, groups, seed)
    s.put(dev, rng.permutation(s.B + 9)[:s.B].tolist())
    for f32 in (False, True):
        got = s.run(f32).to_vec()
        dev.sync()
        s.check(got, f32)


def test_sharp_and_flat_scores(dev):
    for std in (0.0, 40.0):
        s = Setup(8, 2, 16, [(256, [300, 290, 400]), (0, [77])], seed=3, q_std=std).put(dev)
        got = s.run(True).to_vec()
        dev.sync()
        want, size = s.reference()
        # scores of size 40 * 128 / sqrt(128): 2^-23 of each of eight steps
        assert (np.abs(got.reshape(want.shape) - want) <= (2.0 ** -14 + std * 40 * 2.0 ** -20) * size + 1e-30).all()


@pytest.mark.parametrize("group", [4, 1])
def test_scores_that_leave_their_reference_far_behind(dev, group):
    """Scores that grow along the sequence by more than an f32 exponent: the last keys have all the weight."""
    s = Setup(8, 8 // group, 16, [(256, [700, 400] + [300] * 40), (0, [500])], seed=21)
    for b in range(s.B):
        n = int(s.lens[b])
        for j in range(n):
            page, r = s.tables[b, j // 16], j % 16
            bits, f = bf16_round(np.full((8 // group, HD), (j // 64) * 4.0 + (j % 64) / 64, np.float32))
            s.kv_bits[0, page, r], s.kv[0, page, r] = bits.reshape(f.shape), f
    s.q_bits, s.q = bf16_round(np.full(s.q.shape, 1.5, np.float32))
    s.q_bits, s.q = s.q_bits.reshape(s.B, 8, HD), s.q.reshape(s.B, 8, HD)
    s.put(dev)
    for f32 in (False, True):
        got = s.run(f32).to_vec()
        dev.sync()
        # scores up to 45 * 1.5 * 128 / sqrt(128): off by 2^-23 of that per step of 16, 2^-10 in all
        want, size = s.reference()
        g = got.astype(np.float64) if f32 else (got.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        assert (np.abs(g.reshape(want.shape) - want) <= (2.0 ** -10 + (0 if f32 else 2.0 ** -8)) * size + 1e-30).all()


def test_max_len_cuts_and_rows_behind_the_batch_stay(dev):
    import tang_b200 as tb

    s = Setup(8, 2, 16, [(128, [300, 200, 150])], seed=8).put(dev)
    out = dev.upload(np.full((s.B + 1) * 8 * HD, 5, np.float32))
    part = tb.Buffer(dev, out.ptr, s.B * 8 * HD, tb.F32, owns=False)
    s.run(True, max_len=180, out=part)
    dev.sync()
    s.lens = np.minimum(s.lens, 180)
    got = out.to_vec()
    s.check(got[:-8 * HD], True)
    assert (got[-8 * HD:] == 5).all()


def test_infinities_reach_only_those_who_see_them(dev):
    s = Setup(8, 2, 16, [(256, [300, 257, 400]), (0, [40])], seed=9)
    bits = [0x7F80, NAN]
    s.kv_bits[1, s.tables[0, 290 // 16], 290 % 16, :, 3] = bits[0]          # sequence 0 alone
    s.kv_bits[1, s.tables[2, 390 // 16], 390 % 16, :, 4] = bits[1]          # sequence 2 alone
    s.put(dev)
    for f32 in (False, True):
        got = s.run(f32).to_vec()
        dev.sync()
        g = got.reshape(4, 8, HD).astype(np.float64) if f32 else (got.astype(np.uint32) << 16).view(np.float32).astype(np.float64).reshape(4, 8, HD)
        assert (g[0, :, 3] == np.inf).all() and np.isnan(g[2, :, 4]).all()
        mask = np.isfinite(g)
        mask[0, :, 3] = mask[2, :, 4] = True
        assert mask.all()
        want, size = s.reference()
        ok = np.isfinite(g)
        assert (np.abs(g - want)[ok] <= (2.0 ** -14 + 2.0 ** -8) * size[ok]).all()


def test_pages_and_sequences_that_do_not_exist_are_reported(dev):
    import tang_b200 as tb

    for page in (-1, 10 ** 6, -2 ** 31):
        s = Setup(8, 2, 16, [(256, [300, 290]), (0, [77]), (0, [200])], seed=10)
        s.tables[0, 2] = s.tables[1, 2] = s.tables[3, 4] = page
        refs = s.tables.copy()
        s.tables = np.where((refs < 0) | (refs >= s.n_pages), -1, refs)      # (for the reference counts)
        s.put(dev)
        dev.upload_into(s.pool.tables, refs)
        got = s.run(True).to_vec()
        with pytest.raises(tb.TangqError) as e:
            dev.sync()
        assert e.value.status == tb._lib.TQ_EINVAL
        dev.sync()
        s.check(got, True, rows=slice(2, 3))                  # the sequence whose pages exist
    s = Setup(8, 2, 16, [(256, [300, 290]), (128, [177, 150, 140])], seed=16).put(dev)
    for starts in ([1, 2], [0, -1], [0, 6], [3, 2]):          # starts that do not ascend from 0: reported, and nothing is shared
        dev.upload_into(s.gb, np.array(starts + [0], np.int32))
        got = s.run(True).to_vec()
        with pytest.raises(tb.TangqError):
            dev.sync()
        s.check(got, True)
    dev.upload_into(s.gb, s.starts)
    got = s.run(True).to_vec()
    dev.sync()
    s.check(got, True)
    s = Setup(8, 2, 16, [(0, [77]), (0, [20])], seed=11).put(dev, [3, 1])
    dev.upload_into(s.seqs, np.array([3, 99], np.int32))
    got = s.run(True).to_vec()
    with pytest.raises(tb.TangqError):
        dev.sync()
    s.check(got, True, rows=slice(0, 1))
    assert (got.reshape(2, -1)[1] == 0).all()
    dev.sync()


def test_the_same_bits_again_from_a_graph_and_beside_another_handle(dev):
    import tang_b200 as tb

    s = Setup(32, 8, 32, [(640, [700 + 9 * i for i in range(20)]), (0, [1500])], seed=12).put(dev)
    out = s.run(True)
    first = out.to_vec()
    dev.sync()
    other = tb.QuantComputeDevice(0)
    z = Setup(8, 2, 16, [(256, [600] * 9)], seed=13).put(other)
    dev.begin_capture()
    s.run(True, out=out)
    g = dev.end_capture()
    for _ in range(3):
        dev.memset(out, 1)
        g.launch()
        second = z.run(True)
        dev.sync()
        other.sync()
        assert np.array_equal(out.to_vec(), first)
        z.check(second.to_vec(), True)
    # a longer cache under the same graph: the lengths are the device's
    g.free()
    del second
    for b in (z.pool, z.qb, z.kb, z.vb, z.gb, z.sb, *z.state):
        b.destroy() if hasattr(b, "destroy") else b.free()
    other.close()


def test_pages_behind_32_bits(dev):
    """Rows whose offset in elements is larger than 2^32."""
    import tang_b200 as tb

    nh, nkv, P, n_pages = 8, 8, 1024, 4200                    # 1024 elements a row, 2^20 a page
    k, v = (dev.alloc(n_pages * P * nkv * HD, tb.BF16) for _ in range(2))
    s = Setup(nh, nkv, P, [(1024, [1030, 1100])], seed=14)
    far = {int(p): n_pages - 1 - i for i, p in enumerate(sorted(set(s.tables[s.tables >= 0].tolist())))}
    for buf, src in ((k, s.kv_bits[0]), (v, s.kv_bits[1])):
        for p, to in far.items():
            dev.upload_into(tb.Buffer(dev, buf.ptr + to * P * nkv * HD * 2, P * nkv * HD, tb.BF16, owns=False), src[p])
    tables = np.array([[far.get(int(p), -1) for p in row] for row in s.tables], np.int32)
    refs = np.zeros(n_pages, np.int32)
    pool = tb.PagePool(dev, n_pages, P, 2, s.ld, None, dev.upload(refs, tb.I32), dev.upload(tables, tb.I32), dev.upload(s.lens.astype(np.int32), tb.I32))
    q = dev.upload(s.q_bits.reshape(-1), tb.BF16)
    for grouped in (False, True):
        kw = {"group_starts": dev.upload(s.starts, tb.I32), "shared": dev.upload(s.shared, tb.I32), "n_groups": 1, "max_shared": 1024} if grouped else {}
        got = dev.gqa_decode_paged(q, k, v, pool, 2, nh, nkv, HD, 1100, out_dtype=tb.F32, **kw).to_vec()
        dev.sync()
        s.check(got, True)


def test_refusals(dev):
    import tang_b200 as tb

    s = Setup(8, 2, 16, [(16, [20, 30])], seed=15).put(dev)
    call = dev.gqa_decode_paged
    base = dict(q=s.qb, k_pages=s.kb, v_pages=s.vb, pool=s.pool, batch=2, n_heads=8, n_kv_heads=2, head_dim=HD, max_len=30)
    wide = dev.alloc(2 * 18 * HD, tb.BF16)
    for kw in ({"batch": 3}, {"n_heads": 4}, {"max_len": 0}, {"n_kv_heads": 4}, {"group_starts": s.gb}, {"group_starts": s.gb, "shared": s.sb, "n_groups": 2},
               {"group_starts": s.gb, "shared": s.sb, "n_groups": 0}, {"head_dim": 64, "q": dev.alloc(2 * 8 * 64, tb.BF16), "k_pages": dev.alloc(s.n_pages * 16 * 128, tb.BF16),
                                                                      "v_pages": dev.alloc(s.n_pages * 16 * 128, tb.BF16)},
               {"n_heads": 18, "q": wide}, {"out": dev.alloc(2 * 8 * HD, tb.I32)}, {"out": dev.alloc(8, tb.F32)}, {"seqs": dev.alloc(1, tb.I32)}):
        with pytest.raises(tb.TangqError):
            call(**{**base, **kw})
    off = tb.Buffer(dev, s.qb.ptr + 2, s.qb.n, tb.BF16, owns=False)
    with pytest.raises(tb.TangqError):
        call(**{**base, "q": off})
    call(**base)
    dev.sync()


@pytest.mark.parametrize("shared", [False, True])
def test_long_sums_keep_the_precision_of_f32(dev, shared):
    """64 sequences of 16384 positions in the same pages, values of one sign: what the tensor core truncates must not add up over a long sequence.  An error
    of 2^-17 for weights of two bf16 terms (2^-18 each, of a weight and of the sum) and of 6e-9 for each of the 2048 positions that are added up at once."""
    import tang_b200 as tb

    rng, L, P, B, nh, nkv = np.random.default_rng(8), 16384, 64, 64, 8, 2
    n_pages = L // P
    k_bits, k = bf16_round(rng.standard_normal((L, nkv, HD)).astype(np.float32))
    v_bits, v = bf16_round((1 + 0.1 * rng.standard_normal((L, nkv, HD))).astype(np.float32))
    q_bits, q = bf16_round(rng.standard_normal((B, nh, HD)).astype(np.float32))
    pool = tb.PagePool(dev, n_pages, P, B, n_pages, None, dev.upload(np.full(n_pages, B, np.int32), tb.I32),
                       dev.upload(np.tile(np.arange(n_pages, dtype=np.int32), (B, 1)), tb.I32), dev.upload(np.full(B, L, np.int32), tb.I32))
    kw = dict(group_starts=dev.upload(np.zeros(1, np.int32), tb.I32), shared=dev.upload(np.full(1, L, np.int32), tb.I32), n_groups=1, max_shared=L) if shared else {}
    got = dev.gqa_decode_paged(dev.upload(q_bits.reshape(-1), tb.BF16), dev.upload(k_bits.reshape(-1), tb.BF16), dev.upload(v_bits.reshape(-1), tb.BF16), pool, B, nh, nkv,
                               HD, L, out_dtype=tb.F32, **kw).to_vec().reshape(B, nh, HD)
    for b, h in ((0, 0), (31, 5), (63, 7)):
        s = k[:, h // 4].reshape(L, HD).astype(np.float64) @ q[b, h].reshape(HD).astype(np.float64) / np.sqrt(HD)
        w = np.exp(s - s.max())
        want = w @ v[:, h // 4].reshape(L, HD).astype(np.float64) / w.sum()
        assert np.abs(got[b, h] / want - 1).max() <= 2.0 ** -17 + 2048 * 6e-9, (b, h)
    pool.destroy()


def test_the_largest_batch_many_kv_heads_and_a_loose_bound(dev):
    import tang_b200 as tb

    # 1024 sequences, a group each or all in one
    s = Setup(8, 1, 16, [(0, [i % 37]) for i in range(1024)], seed=31).put(dev)
    for f32 in (False, True):
        s.check(s.run(f32).to_vec(), f32)
    s = Setup(2, 2, 16, [(200, [200 + i % 9 for i in range(1024)])], seed=32).put(dev)
    s.check(s.run(True).to_vec(), True)
    with pytest.raises(tb.TangqError):
        dev.gqa_decode_paged(dev.alloc(1025 * 2 * HD, tb.BF16), s.kb, s.vb, s.pool, 1025, 2, 2, HD, 209, seqs=dev.alloc(1025, tb.I32))
    # more KV heads than SMs
    s = Setup(320, 160, 16, [(130, [131, 150, 140]), (0, [33])], seed=33).put(dev)
    for f32 in (False, True):
        s.check(s.run(f32).to_vec(), f32)
    # tables for a million positions, of which sequences have few
    s = Setup(8, 2, 16, [(256, [300, 400, 290]), (0, [5000])], seed=34)
    s.tables = np.concatenate([s.tables, np.full((s.B, 65536 - s.ld), -1, np.int32)], 1)
    s.ld = 65536
    s.put(dev)
    for f32 in (False, True):
        s.check(s.run(f32, max_len=1 << 20).to_vec(), f32)
    dev.sync()


@pytest.mark.parametrize("name", ["samples", "groups", "many", "one kv head", "five to one", "two hundred"])
def test_bf16_results_are_off_by_their_own_rounding(dev, name):
    """Shared tiles too, whatever number of rows meets them: 2^-14 of the sum of |weight value| for what f32 results may be off (``Setup.check``), and the
    rounding to bf16 of what that gives, 2^-8 of it."""
    s = Setup(*CASES[name], seed=40 + len(name)).put(dev)
    got = (s.run(False).to_vec().astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    dev.sync()
    want, size = s.reference()
    off = 2.0 ** -14 * size
    err = np.abs(got.reshape(want.shape) - want) / (off + 2.0 ** -8 * (np.abs(want) + off) + 1e-30)
    assert err.max() <= 1, (err.max(), np.unravel_index(err.argmax(), err.shape))


@pytest.mark.parametrize("shared", [False, True])
def test_a_loose_bound_costs_no_precision(dev, shared):
    """As ``test_long_sums_keep_the_precision_of_f32``, with the bounds of a caller who has recorded a graph for any length: eight KV heads, tables for a
    million positions.  A piece has no more than 2176 positions."""
    import tang_b200 as tb

    rng, L, P, B, nh, nkv, ld = np.random.default_rng(28), 16384, 128, 64, 32, 8, 8192
    n_pages, most = L // P, ld * P
    k_bits, k = bf16_round(rng.standard_normal((L, nkv, HD)).astype(np.float32))
    v_bits, v = bf16_round((1 + 0.1 * rng.standard_normal((L, nkv, HD))).astype(np.float32))
    q_bits, q = bf16_round(rng.standard_normal((B, nh, HD)).astype(np.float32))
    tables = np.full((B, ld), -1, np.int32)
    tables[:, :n_pages] = np.arange(n_pages)
    pool = tb.PagePool(dev, n_pages, P, B, ld, None, dev.upload(np.full(n_pages, B, np.int32), tb.I32), dev.upload(tables, tb.I32),
                       dev.upload(np.full(B, L, np.int32), tb.I32))
    kw = dict(group_starts=dev.upload(np.zeros(1, np.int32), tb.I32), shared=dev.upload(np.full(1, L, np.int32), tb.I32), n_groups=1, max_shared=most) if shared else {}
    got = dev.gqa_decode_paged(dev.upload(q_bits.reshape(-1), tb.BF16), dev.upload(k_bits.reshape(-1), tb.BF16), dev.upload(v_bits.reshape(-1), tb.BF16), pool, B, nh, nkv,
                               HD, most, out_dtype=tb.F32, **kw).to_vec().reshape(B, nh, HD)
    dev.sync()
    for b, h in ((0, 0), (31, 17), (63, 31)):
        s = k[:, h // 4].reshape(L, HD).astype(np.float64) @ q[b, h].reshape(HD).astype(np.float64) / np.sqrt(HD)
        w = np.exp(s - s.max())
        want = w @ v[:, h // 4].reshape(L, HD).astype(np.float64) / w.sum()
        assert np.abs(got[b, h] / want - 1).max() <= 2.0 ** -17 + 2176 * 6e-9, (b, h)
    pool.destroy()


@pytest.mark.parametrize("f32", [False, True])
def test_runs_of_several_pieces(dev, f32):
    """One CTA for each of 75 KV heads: runs that end at, before and behind the tiles of a piece, of three rows and of nine."""
    if f32:
        groups = [(0, [n]) for n in (1, 2048, 2049, 2177, 2305, 4225)] + [(2500, [2500, 2540, 2600]), (2176, [2180, 2177, 2300])]
    else:
        groups = [(0, [16513]), (0, [300]), (16900, [16901, 16900, 17000])]
    s = Setup(225, 75, 128, groups, seed=51).put(dev)
    want = s.reference()
    s.reference = lambda: want
    for grouped in (True, False):
        got = s.run(f32, grouped=grouped).to_vec()
        dev.sync()
        s.check(got, f32)


def later_keys_weigh_more(s, factor):
    """Makes the scores of a set-up grow along each sequence: `factor` (natural logarithm) for every 128 positions, q . k / sqrt(128) = 1.5 * sqrt(128) * k."""
    for b in range(s.B):
        for j in range(int(s.lens[b])):
            page, r = s.tables[b, j // s.P], j % s.P
            bits, f = bf16_round(np.full((s.nkv, HD), factor * (j // 128) / (1.5 * np.sqrt(HD)), np.float32))
            s.kv_bits[0, page, r], s.kv[0, page, r] = bits.reshape(f.shape), f
    s.q_bits, s.q = (a.reshape(s.q.shape) for a in bf16_round(np.full(s.q.shape, 1.5, np.float32)))


@pytest.mark.parametrize("f32", [False, True])
def test_large_values_under_weights_far_above_their_reference(dev, f32):
    """Weights of 2^64 against the first tile's, which are f32 numbers, and values of 1e18, whose weighted sum is none: the result is one."""
    s = Setup(225, 75, 16, [(256, [300, 270, 290]), (0, [200]), (256, [256] * 3), (0, [256])], seed=61)       # (a CTA for each KV head)
    later_keys_weigh_more(s, 44.4)                                     # 2^64 for each tile
    s.kv_bits[1], s.kv[1] = (a.reshape(s.kv[1].shape) for a in bf16_round((1 + 0.1 * s.kv[1]) * np.float32(1e18)))
    for b in range(s.B):
        if s.lens[b] % 16:
            s.kv_bits[1, s.tables[b, s.lens[b] // 16], s.lens[b] % 16:] = NAN
    s.put(dev)
    want, size = s.reference()
    for grouped in (True, False):
        got = s.run(f32, grouped=grouped).to_vec()
        dev.sync()
        g = (got.astype(np.float64) if f32 else (got.astype(np.uint32) << 16).view(np.float32).astype(np.float64)).reshape(want.shape)
        # scores up to 3 * 44.4, a sum of 128 products: off by 2^-24 of it a product
        off = (2.0 ** -14 + 128 * 133 * 2.0 ** -24) * size
        assert np.isfinite(g).all() and (np.abs(g - want) <= off + (0 if f32 else 2.0 ** -8) * (np.abs(want) + off)).all()


def test_shared_positions_are_the_first_sequences_whatever_the_scores(dev):
    """What the other members' tables say of the shared positions counts as little for a row that is attended key by key."""
    for factor in (0.0, 80.0):
        s = Setup(225, 75, 16, [(256, [300, 270, 290]), (0, [500])], seed=62)               # (a CTA for each KV head)
        later_keys_weigh_more(s, factor)
        true = s.tables.copy()
        s.put(dev)
        other = true.copy()
        other[1, :16], other[2, :16] = true[3, 1:17], true[3, 15::-1]  # pages of the sequence behind the group
        dev.upload_into(s.pool.tables, other)
        got = s.run(True).to_vec().reshape(s.B, 225, HD)
        dev.sync()
        want, size = s.reference()
        assert (np.abs(got - want) <= (2.0 ** -14 + 128 * 4 * factor * 2.0 ** -24) * size).all(), factor


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("P", [16, 1024])
def test_rows_that_are_attended_again(dev, P, f32):
    """Every number of keys that the last turn of four keys and four warps can have, beside a NaN in another element; scores that start at -infinity too."""
    s = Setup(8, 2, P, [(256, [256 + i for i in range(1, 18)])] + [(0, [i]) for i in range(1, 18)], seed=63)
    s.kv_bits[1, :, :, :, 5] = NAN
    for b in range(s.B):
        s.kv_bits[0, s.tables[b, 0], 0], s.kv[0, s.tables[b, 0], 0] = bf16_round(np.full((2, HD), -3e38, np.float32))
    s.q_bits, s.q = (a.reshape(s.q.shape) for a in bf16_round(np.abs(s.q) + 1))        # (the first key's score is -infinity)
    s.put(dev)
    got = s.run(f32).to_vec()
    dev.sync()
    with np.errstate(over="ignore"):
        want, size = s.reference()
    g = (got.astype(np.float64) if f32 else (got.astype(np.uint32) << 16).view(np.float32).astype(np.float64)).reshape(want.shape)
    ok = np.ones(want.shape, bool)
    ok[:, :, 5] = False
    ok[np.array(s.lens) == 1] = False                  # (nothing but the first key: 0 over 0 in 32 bits)
    assert np.isnan(g[s.lens > 1][:, :, 5]).all()
    off = (2.0 ** -14 + 128 * 2.0 ** -24 * 8 * 12) * size              # scores up to 8 * 12 here, sums of 128 products
    assert (np.abs(g - want)[ok] <= (off + (0 if f32 else 2.0 ** -8) * (np.abs(want) + off))[ok]).all()


@pytest.mark.parametrize("case", ["few rows", "sixteen rows", "many rows"])
def test_f32_results_keep_all_bits_of_the_weights(dev, case):
    """Scores of one product each, which f32 holds, of two keys that count and others far below them: what is left of the error is the weights'.  An exponent
    (base 2: a score of 2.9 at most, 5.7 from the largest) is off by 2^-24 of either, 2^-21.4 of the weight, its exponential by 2^-22: for numerator and
    denominator 2^-19.7; two sums and a division, 3 * 2^-23: 2^-19 of the sum of |weight value|.  Where rows are the lanes (more than 16 of a
    group), a weight is two terms: 2^-16 of it more."""
    s = Setup(16, 4, 16, {"few rows": [(0, [16])] * 60, "sixteen rows": [(128, [128] * 4)] * 20, "many rows": [(128, [128] * 12)] * 8}[case], seed=71)
    rng = np.random.default_rng(72)
    s.q_bits[:], s.q[:] = 0, 0
    bits, f = bf16_round(rng.uniform(8, 22, (s.B, 16)).astype(np.float32))
    s.q_bits[:, :, 0], s.q[:, :, 0] = bits.reshape(f.shape), f
    for page in np.unique(s.tables[s.tables >= 0]):
        x = np.full((s.P, s.nkv), -300, np.float32)
        first = case == "few rows" or page in s.tables[:, 0]
        for g in range(s.nkv if first else 0):
            x[rng.permutation(s.P)[:2], g] = rng.uniform(-1, 1, 2)
        bits, f = bf16_round(x)
        s.kv_bits[0, page], s.kv[0, page] = 0, 0
        s.kv_bits[0, page, :, :, 0], s.kv[0, page, :, :, 0] = bits.reshape(f.shape), f
    s.put(dev)
    got = s.run(True).to_vec()
    dev.sync()
    want, size = s.reference()
    err = np.abs(got.reshape(want.shape) - want) / size
    assert err.max() <= 2.0 ** -19 + (2.0 ** -16 if case == "many rows" else 0), (err.max(), np.sqrt((err ** 2).mean()))
