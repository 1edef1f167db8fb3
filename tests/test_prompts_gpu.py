"""Prompts of different lengths through the model over pages, against the oracle; appending, attention over prompts and decode attention over 4 bits
one after the other as a generation has them, recorded and replayed, on streams of two handles."""
import numpy as np
import pytest

from llama_util import HostLlama
from packed_util import HD, attend, check_attention, pack, rotate, row_bytes, tables
from util import bf16_round

pytestmark = pytest.mark.gpu
BAR = 2e-2      # of the logits' rms: what the bf16 pipeline may be off the oracle


@pytest.fixture(scope="module")
def dev():
    import tang_b200

    d = tang_b200.QuantComputeDevice(0)
    yield d
    d.close()


def host_model(seed, n_heads=4, n_kv=2):
    return HostLlama(np.random.default_rng(seed), n_layers=2, d=256, n_heads=n_heads, n_kv=n_kv, hd=128, ffn=512, vocab=1024)


class Followed:
    """A sequence as the oracle runs it."""

    def __init__(self, host, orc, max_seq):
        self.host, self.orc, self.n = host, orc, 0
        self.k = [np.zeros((max_seq, host.n_kv * host.hd), np.uint16) for _ in range(host.n_layers)]
        self.v = [np.zeros_like(k) for k in self.k]

    def run(self, tokens):
        for t in tokens:
            out = self.host.oracle_decode(self.orc, int(t), self.k, self.v, self.n)
            self.n += 1
        return out

    def fork(self):
        f = Followed(self.host, self.orc, len(self.k[0]))
        f.n, f.k, f.v = self.n, [k.copy() for k in self.k], [v.copy() for v in self.v]
        return f


def near(got, want):
    rms = np.sqrt(np.mean(want * want))
    return np.abs(got - want).max() <= BAR * rms


@pytest.mark.parametrize("heads", [(4, 2), (8, 1), (6, 2)])
def test_prompts_in_portions_behind_a_shared_beginning(dev, orc, heads):
    """Prompts of different lengths in one step; the rest of each, some with nothing, in another; two sequences forked from one of them go on with portions of
    their own; then all decode a token."""
    import tang_b200 as tb

    host, max_seq, B = host_model(5, *heads), 256, 5
    model = host.to_device(dev, max_seq, B)
    pool = model.page_pool(B, 16)
    rng = np.random.default_rng(1)
    lg = dev.alloc(B * host.vocab)
    ints = lambda v: dev.upload(np.asarray(v, np.int32), tb.I32)  # noqa: E731
    seqs = [Followed(host, orc, max_seq) for _ in range(B)]

    def step(portions, room=0):
        """portions: {sequence: tokens}; `room`: rows behind them."""
        which, toks = list(portions), [rng.integers(0, host.vocab, n) for n in portions.values()]
        pool.extend(which, counts=[len(t) for t in toks])
        rows = sum(len(t) for t in toks)
        model.prefill_paged(ints(np.concatenate([*toks, np.zeros(room, int)])), pool, len(which), rows + room, max_seq, lg, seqs=ints(which),
                            seq_rows=ints(np.concatenate([[0], np.cumsum([len(t) for t in toks])])))
        got = lg.to_vec().reshape(B, -1)
        dev.sync()
        for i, (s, t) in enumerate(zip(which, toks)):
            if len(t):
                assert near(got[i], seqs[s].run(t)), (which, s)

    step({0: 37, 2: 1, 1: 140})
    step({1: 9, 0: 0, 2: 60}, room=11)
    pool.fork([1, 1], [3, 4], keep=[149, 100])
    seqs[3], seqs[4] = seqs[1].fork(), Followed(host, orc, max_seq)
    seqs[4].n, seqs[4].k, seqs[4].v = 100, [k.copy() for k in seqs[1].k], [v.copy() for v in seqs[1].v]
    step({3: 21, 4: 5, 1: 2})
    pool.extend(list(range(B)))
    toks = rng.integers(0, host.vocab, B)
    model.decode_paged(ints(toks), pool, B, max_seq, lg)
    got = lg.to_vec().reshape(B, -1)
    dev.sync()
    for b in range(B):
        assert near(got[b], seqs[b].run([toks[b]])), b
    model.destroy()


def test_samples_of_prompts_of_different_lengths(dev, orc):
    """As for equal lengths: each sample's log probabilities are the oracle's for the tokens that were drawn."""
    import tang_b200 as tb

    host, N, m, max_seq = host_model(8), 4, 3, 256
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, host.vocab, n).astype(np.int32) for n in (77, 1, 150, 16)]
    model = host.to_device(dev, max_seq, len(prompts) * m)
    got = model.sample(prompts, N, m, tb.SamplerConfig(1.0, 0, 1.0, 1.0), seed=3)
    assert got.tokens.shape == got.logprobs.shape == (4, m, N)
    for b, p in enumerate(prompts):
        start = Followed(host, orc, max_seq)
        if len(p) > 1:
            start.run(p[:-1])
        for j in range(m):
            f, tok = start.fork(), p[-1]
            for i, t in enumerate(got.tokens[b, j]):
                logits = f.run([tok])
                x = logits - logits.max()
                want = x[t] - np.log(np.exp(x).sum())
                assert abs(got.logprobs[b, j, i] - want) <= 2 * BAR * np.sqrt(np.mean(logits * logits)) + 1e-5, (b, j, i)
                tok = t
    again = model.sample(prompts, N, m, tb.SamplerConfig(1.0, 0, 1.0, 1.0), seed=3)
    assert np.array_equal(again.tokens, got.tokens)
    for bad in ([1, 2, 3], [[1], []], [[[1, 2]], [[3, 4]]]):
        with pytest.raises(tb.TangqError):
            model.sample(bad, 1, 1)
    model.destroy()


def test_model_refusals(dev):
    import tang_b200 as tb

    host = host_model(9)
    model, other = host.to_device(dev, 64, 2), tb.QuantComputeDevice(0)
    pool = model.page_pool(2, 16)
    ints = lambda v: dev.upload(np.asarray(v, np.int32), tb.I32)  # noqa: E731
    lg, toks, rows = dev.alloc(2 * host.vocab), ints([1, 2, 3]), ints([0, 1, 3])
    pool.extend([0, 1], counts=[1, 2])
    ok = dict(token_ids=toks, pool=pool, batch=2, rows=3, max_len=64, logits=lg, seq_rows=rows)
    model.prefill_paged(**ok)
    dev.sync()
    for kw in ({"batch": 3}, {"batch": 0}, {"rows": 4}, {"rows": 0}, {"max_len": 65}, {"max_len": 0}, {"seq_rows": None}, {"seq_rows": ints([0, 1])}, {"seqs": ints([0])},
               {"logits": dev.alloc(host.vocab)}, {"token_ids": dev.alloc(3)}, {"pool": tb.PagePool(other, 4, 16, 2, 4)}, {"pool": tb.PagePool(dev, 99, 16, 2, 4)}):
        with pytest.raises(tb.TangqError):
            model.prefill_paged(**{**ok, **kw})
    dev.sync()
    # what would have to grow is not recorded
    many = ints(np.zeros(500, int))
    dev.begin_capture()
    with pytest.raises(tb.TangqError):
        model.prefill_paged(**{**ok, "token_ids": many, "rows": 500})
    dev.end_capture().free()
    dev.sync()
    model.destroy()
    other.close()


class Generation:
    """Sequences over pages of 4 bits from their prompts on: each step's rows are appended and attended; the same in numpy."""

    def __init__(self, dev, seed, nh=8, nkv=2, P=16, n_seqs=3, max_pages=20):
        import tang_b200 as tb

        self.dev, self.tb, self.nh, self.nkv, self.P, self.n = dev, tb, nh, nkv, P, n_seqs
        self.rng = np.random.default_rng(seed)
        pages = n_seqs * max_pages
        self.pool = tb.PagePool(dev, pages, P, n_seqs, max_pages)
        self.k, self.v = (dev.upload(np.full(pages * P * row_bytes(nkv), 0xFF, np.uint8), tb.U8) for _ in range(2))
        self.pool.set_arrays([self.k, self.v])
        self.cos, self.sin = tables(max_pages * P)
        self.cb, self.sb = dev.upload(self.cos), dev.upload(self.sin)
        self.held = [[np.zeros((0, nkv, HD)), np.zeros((0, nkv, HD))] for _ in range(n_seqs)]

    def rows(self, n):
        return self.rng.standard_normal((n, self.nh + 2 * self.nkv, HD)).astype(np.float32)

    def expect(self, x, counts):
        """Appends to what the sequences hold; (result, size) of the rows' attention."""
        want, first = [], 0
        for s, c in enumerate(counts):
            r, pos = x[first:first + c], np.arange(len(self.held[s][0]), len(self.held[s][0]) + c)
            first += c
            turned = rotate(r[:, :self.nh + self.nkv], self.cos[pos], self.sin[pos])
            for i, new in enumerate((turned[:, self.nh:], r[:, self.nh + self.nkv:])):
                self.held[s][i] = np.concatenate([self.held[s][i], pack(new)[1]])
            if c:
                want.append(attend(bf16_round(np.ascontiguousarray(turned[:, :self.nh]))[1].reshape(c, self.nh, HD), *self.held[s]))
        return [np.concatenate(a) for a in zip(*want)]

    def prompts(self, counts):
        x = self.rows(sum(counts))
        self.pool.extend(list(range(self.n)), counts=counts)
        starts = self.dev.upload(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), self.tb.I32)
        q = self.dev.kv_append_paged(self.dev.upload(x), self.cb, self.sb, self.pool, self.k, self.v, self.n, len(x), self.nh, self.nkv, HD, seq_rows=starts)
        out = self.dev.gqa_prefill_paged(q, self.k, self.v, self.pool, self.n, len(x), self.nh, self.nkv, HD, 320, seq_rows=starts)
        got = out.to_vec()
        self.dev.sync()
        check_attention(got, *self.expect(x, counts), terms=1)

    def buffers(self):
        self.xb, self.qb, self.out = self.dev.alloc(self.n * (self.nh + 2 * self.nkv) * HD), self.dev.alloc(self.n * self.nh * HD, self.tb.BF16), None
        self.out = self.dev.alloc(self.n * self.nh * HD, self.tb.BF16)
        self.every = self.dev.upload(np.arange(self.n, dtype=np.int32), self.tb.I32)

    def step(self):
        self.pool.extend(self.every, self.n)
        self.dev.kv_append_paged(self.xb, self.cb, self.sb, self.pool, self.k, self.v, self.n, self.n, self.nh, self.nkv, HD, q_out=self.qb)
        self.dev.gqa_decode_paged_q4(self.qb, self.k, self.v, self.pool, self.n, self.nh, self.nkv, HD, 320, out=self.out)

    def put(self):
        x = self.rows(self.n)
        self.dev.upload_into(self.xb, x)
        return x

    def check(self, x):
        got = self.out.to_vec()
        check_attention(got, *self.expect(x, [1] * self.n), terms=2)


def test_a_generation_over_four_bits(dev):
    """Prompts in two portions, a step as it is, then the step recorded and replayed over page borders."""
    g = Generation(dev, 1)
    g.prompts([40, 7, 130])
    g.prompts([3, 0, 61])
    g.buffers()
    x = g.put()
    g.step()
    g.check(x)
    dev.begin_capture()
    g.step()
    graph = dev.end_capture()
    for _ in range(20):
        x = g.put()
        graph.launch()
        dev.sync()
        g.check(x)
    g.prompts([0, 33, 1])              # beside a graph that lives
    x = g.put()
    graph.launch()
    g.check(x)
    dev.sync()
    graph.free()


def test_two_recorded_generations_share_the_workspace_and_two_handles_do_not():
    """Graphs of one handle, replayed in turn without waiting, and those of another handle on its own stream beside them."""
    import tang_b200 as tb

    devs = [tb.QuantComputeDevice(0) for _ in range(2)]
    gens = [Generation(d, 10 + i) for i, d in enumerate([devs[0], devs[0], devs[1]])]
    graphs = []
    for i, g in enumerate(gens):
        g.prompts([20 + i, 150 - i, 1])
        g.buffers()
        x = g.put()
        g.step()
        g.check(x)
        g.dev.sync()
        g.dev.begin_capture()
        g.step()
        graphs.append(g.dev.end_capture())
    for _ in range(12):
        xs = [g.put() for g in gens]
        for graph in graphs:
            graph.launch()
        for g, x in zip(gens, xs):
            g.check(x)
    for d in devs:
        d.sync()
    for graph in graphs:
        graph.free()
    for g in gens:
        g.pool.destroy()


@pytest.mark.parametrize("form", ["bf16", "q4"])
def test_pages_whose_bytes_are_behind_32_bits(dev, form):
    """A cache of more than 5 GB for keys and as much for values, the sequences in its last pages."""
    import tang_b200 as tb

    nh, nkv, P, B = 32, 8, 1024, 2
    row = nkv * HD * 2 if form == "bf16" else row_bytes(nkv)
    pages = -(-(5 << 30) // (row * P))
    per = 1 if form == "q4" else 2
    k, v = (dev.alloc(pages * P * row // per, tb.U8 if form == "q4" else tb.BF16) for _ in range(2))
    tables_h, lens = np.full((B, 3), -1, np.int32), np.array([1500, 90], np.int32)
    tables_h[0, :2], tables_h[1, 0] = [pages - 1, pages - 3], pages - 2
    refs = np.zeros(pages, np.int32)
    refs[[pages - 1, pages - 2, pages - 3]] = 1
    state = [dev.upload(a, tb.I32) for a in (refs, tables_h, lens)]
    pool = tb.PagePool(dev, pages, P, B, 3, None, *state)
    rng, cs = np.random.default_rng(3), tables(1500)
    x = rng.standard_normal((1590, nh + 2 * nkv, HD)).astype(np.float32)
    starts = dev.upload(np.array([0, 1500, 1590], np.int32), tb.I32)
    q = dev.kv_append_paged(dev.upload(x), dev.upload(cs[0]), dev.upload(cs[1]), pool, k, v, B, 1590, nh, nkv, HD, seq_rows=starts)
    ko, vo = dev.kv_read_paged(k, v, pool, B, 1590, nkv, HD, seq_rows=starts)
    out = dev.gqa_prefill_paged(q, k, v, pool, B, 1590, nh, nkv, HD, 1500, seq_rows=starts)
    pos = np.concatenate([np.arange(1500), np.arange(90)])
    turned = rotate(x[:, :nh + nkv], cs[0][pos], cs[1][pos])
    stored = lambda a: pack(a)[1] if form == "q4" else bf16_round(np.ascontiguousarray(a))[1].reshape(a.shape)  # noqa: E731
    kv = [stored(turned[:, nh:]), stored(x[:, nh + nkv:])]
    for got, want in ((ko, kv[0]), (vo, kv[1])):
        assert np.array_equal((got.to_vec().astype(np.uint32) << 16).view(np.float32).reshape(want.shape), want)
    qf = bf16_round(np.ascontiguousarray(turned[:, :nh]))[1].reshape(1590, nh, HD)
    got = out.to_vec().reshape(1590, nh, HD)
    for r, n in ((1499, 1500), (1023, 1024), (0, 1)):
        check_attention(got[r:r + 1], *attend(qf[r:r + 1], kv[0][:n], kv[1][:n]), terms=1)
    check_attention(got[1500:], *attend(qf[1500:], kv[0][1500:], kv[1][1500:]), terms=1)
    if form == "q4":
        last = dev.upload(np.ascontiguousarray(q.to_vec().reshape(1590, -1)[[1499, 1589]]), tb.BF16)
        one = dev.gqa_decode_paged_q4(last, k, v, pool, B, nh, nkv, HD, 1500).to_vec().reshape(B, nh, HD)
        check_attention(one[:1], *attend(qf[1499:1500], kv[0][:1500], kv[1][:1500]), terms=2)
        check_attention(one[1:], *attend(qf[1589:], kv[0][1500:], kv[1][1500:]), terms=2)
    dev.sync()
    pool.destroy()


def test_prefill_is_recorded_with_room_for_more_rows(dev):
    """One graph for steps of up to 60 rows: what the starts say is read when it is replayed; parts of the keys share a workspace that has its size."""
    import tang_b200 as tb

    g = Generation(dev, 20)
    room = 60
    x_b, starts, counts_b = dev.alloc(room * 12 * HD), dev.upload(np.zeros(4, np.int32), tb.I32), dev.upload(np.zeros(3, np.int32), tb.I32)
    every, q, out = dev.upload(np.arange(3, dtype=np.int32), tb.I32), dev.alloc(room * 8 * HD, tb.BF16), dev.alloc(room * 8 * HD, tb.BF16)

    def step():
        g.pool.extend(every, 3, counts=counts_b)
        dev.kv_append_paged(x_b, g.cb, g.sb, g.pool, g.k, g.v, 3, room, 8, 2, HD, seq_rows=starts, q_out=q)
        dev.gqa_prefill_paged(q, g.k, g.v, g.pool, 3, room, 8, 2, HD, 320, seq_rows=starts, out=out)

    def put(counts):
        x = g.rows(sum(counts))
        dev.upload_into(x_b, np.concatenate([x, np.full((room - len(x), 12, HD), np.nan, np.float32)]))
        dev.upload_into(starts, np.concatenate([[0], np.cumsum(counts)]))
        dev.upload_into(counts_b, counts)
        return x

    def check(x, counts):
        dev.sync()
        check_attention(out.to_vec().reshape(room, -1)[:len(x)], *g.expect(x, counts), terms=1)

    counts = [5, 30, 25]
    x = put(counts)
    step()
    check(x, counts)
    dev.begin_capture()
    step()
    graph = dev.end_capture()
    for counts in ([1, 1, 1], [58, 0, 2], [0, 0, 1], [20, 20, 20], [0, 60, 0], [3, 9, 40], [33, 1, 20]):
        x = put(counts)
        graph.launch()
        check(x, counts)
    graph.free()


def test_refusals(dev):
    import tang_b200 as tb

    other = tb.QuantComputeDevice(0)
    pool, theirs = tb.PagePool(dev, 4, 16, 2, 4), tb.PagePool(other, 4, 16, 2, 4)
    keep = [dev.alloc(1 << 16, t) for t in (tb.F32, tb.BF16)]
    f, b = (k.ptr for k in keep)
    h, L, ctx = pool.handle, dev._L, dev._ctx
    append = [ctx, f, 0, 0, f, f, 64, h, None, None, 2, 2, 4, 2, 128, b, b, b, 0]
    read = [ctx, b, b, 0, h, None, None, 2, 2, 2, 128, b, b]
    prefill = [ctx, b, b, b, 0, h, None, None, 2, 2, 4, 2, 128, 64, b + 4096]
    decode = [ctx, b, b, b, h, None, 2, 4, 2, 128, 64, b]
    for fn, ok, batch, bad in (
            (L.tq_kv_append_paged, append, 10, {1: [None, f + 4], 2: [2, 9], 3: [100, 8 * 128 + 2], 4: [None, f + 8], 5: [None], 6: [0], 7: [None, theirs.handle], 10: [3, 1025],
                                            11: [1, 3], 12: [0, 70000], 13: [0], 14: [64], 15: [None, b + 2], 16: [None], 17: [None, b + 8], 18: [2, -1]}),
            (L.tq_kv_read_paged, read, 7, {1: [None], 2: [None, b + 8], 3: [2], 4: [None, theirs.handle], 7: [3], 8: [1], 9: [0], 10: [64], 11: [None], 12: [None, b + 4]}),
            (L.tq_gqa_prefill_paged, prefill, 8, {1: [None, b + 8], 2: [None], 3: [None], 4: [2], 5: [None, theirs.handle], 8: [3, 5000], 9: [1], 10: [0, 3, 18], 11: [0], 12: [64],
                                               13: [0, 1 << 31], 14: [None, b + 2, b]}),
            (L.tq_gqa_decode_paged_q4, decode, 6, {1: [None, b + 8], 2: [None], 3: [None, b + 4], 4: [None, theirs.handle], 6: [3], 7: [3, 18, 0], 8: [0], 9: [64],
                                                10: [0, 1 << 31], 11: [None, b + 2]})):
        for at, values in bad.items():
            for v in values:
                args = list(ok)
                args[at] = v
                assert fn(*args) == tb._lib.TQ_EINVAL, (fn, at, v)
        none = list(ok)
        none[batch] = 0
        assert fn(*none) == tb._lib.TQ_OK
    dev.sync()
    pool.destroy()
    theirs.destroy()
    other.close()
