"""Several continuations of a prompt over forked pages, and the log probabilities that rank them: the steps of a model over pages against its
steps over slots and against the oracle, the log probabilities of generated and of given tokens, and the command line."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

from llama_util import HostLlama
from tofazen_util import CONFIGS, save, views, weights

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAR = 2e-2      # of the logits' rms: what the bf16 pipeline may be off the oracle


@pytest.fixture(scope="module")
def dev():
    import tang_b200

    d = tang_b200.QuantComputeDevice(0)
    yield d
    d.close()


def log_softmax(x):
    x = np.asarray(x, np.float64)
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


def logprob_error(x):
    """Of a log probability from the f32 logits x: the exponentials' arguments are rounded in units of 2^-24 of |x| + |max|, the exponentials, their
    sum, its logarithm and the last difference to a few 2^-23 of what they are."""
    return 2.0 ** -20 * (2 + np.abs(x).max() + np.log(x.shape[-1]))


def host_model(seed, n_heads=4, n_kv=2):
    return HostLlama(np.random.default_rng(seed), n_layers=2, d=256, n_heads=n_heads, n_kv=n_kv, hd=128, ffn=512, vocab=1024)


@pytest.mark.parametrize("P,m,greedy", [(1, 3, False), (3, 1, True), (3, 4, True), (17, 2, False), (200, 3, True), (200, 3, False), (145, 1, False)])
def test_samples_follow_the_oracle(dev, orc, P, m, greedy):
    """Every sample's log probabilities are the oracle's for the tokens that were drawn, and a greedy sample takes the oracle's likeliest token up to
    the logits' bar.  (A log probability is one logit less a mean of them, both within the bar.)"""
    import tang_b200 as tb

    host = host_model(P + m)
    B, N, max_seq = 2, 5, 256
    prompts = np.random.default_rng(P).integers(0, host.vocab, (B, P)).astype(np.int32)
    model = host.to_device(dev, max_seq, B * m)
    got = model.sample(prompts, N, m, None if greedy else tb.SamplerConfig(1.0, 0, 1.0, 1.0), seed=3)
    assert got.tokens.shape == got.logprobs.shape == (B, m, N) and got.order.shape == (B, m)
    if not greedy and m > 1:
        assert all(len({tuple(s) for s in got.tokens[b]}) == m for b in range(B))       # (chances of two equal ones: 1024^-5 or so)
    sums = got.logprobs.astype(np.float64).sum(2)
    for b in range(B):
        assert sorted(got.order[b]) == list(range(m)) and np.all(np.diff(sums[b][got.order[b]]) <= 0)
        kc = [np.zeros((max_seq, host.n_kv * host.hd), np.uint16) for _ in range(host.n_layers)]
        vc = [np.zeros_like(k) for k in kc]
        for p in range(P - 1):
            host.oracle_decode(orc, int(prompts[b, p]), kc, vc, p)
        for j in range(m):
            tok = int(prompts[b, -1])
            for i, t in enumerate(got.tokens[b, j]):
                logits = host.oracle_decode(orc, tok, kc, vc, P - 1 + i)
                rms = np.sqrt(np.mean(logits * logits))
                assert abs(got.logprobs[b, j, i] - log_softmax(logits)[t]) <= 2 * BAR * rms + 1e-5, (b, j, i)
                if greedy:
                    assert logits[t] >= logits.max() - BAR * rms, (b, j, i)
                tok = int(t)
    again = model.sample(prompts, N, m, None if greedy else tb.SamplerConfig(1.0, 0, 1.0, 1.0), seed=3)
    assert np.array_equal(again.tokens, got.tokens)
    model.destroy()


@pytest.mark.parametrize("heads", [(4, 2), (8, 1)])
def test_steps_over_pages_are_steps_over_slots(dev, heads):
    """Ragged sequences in another order than the pool's, in pages that end between, on and behind the new positions, with and without a group; extend,
    step and log probabilities once eagerly and then as one replayed graph."""
    import tang_b200 as tb

    host = host_model(5, *heads)
    lens, steps, max_seq, V = [15, 16, 1, 31, 130], 4, 160, host.vocab
    B = len(lens)
    rng = np.random.default_rng(6)
    past = rng.integers(0, V, (B, max_seq)).astype(np.int32)
    past[3, :31] = past[1, :31] = past[0, :31]          # 0, 1 and 3 begin alike
    a, b = host.to_device(dev, max_seq, 8), host.to_device(dev, max_seq, 8)
    lg, seqs = dev.alloc(8 * V), [4, 0, 1, 3, 2]       # batch order: 0, 1 and 3 next to one another
    want = np.zeros((B, steps, V))
    for i, n in enumerate(lens):                       # over slots, a sequence at a time
        for p in range(n + steps):
            a.decode(dev.upload(past[i:i + 1, p], tb.I32), dev.upload(np.array([p], np.int32), tb.I32), 1, max_seq, lg)
            if p >= n:
                want[i, p - n] = dev.download(lg)[:V]
        dev.sync()
    # over pages: the longest common run is put in once and forked
    for grouped in (False, True):
        pool = b.page_pool(6, 16)
        for p in range(15):
            pool.extend([0])
            b.decode_paged(dev.upload(past[0:1, p], tb.I32), pool, 1, max_seq, lg, seqs=dev.upload(np.array([0], np.int32), tb.I32))
        pool.fork([0, 0], [1, 3])
        for i in (1, 2, 3, 4):
            for p in range(15 if i in (1, 3) else 0, lens[i]):
                pool.extend([i])
                b.decode_paged(dev.upload(past[i:i + 1, p], tb.I32), pool, 1, max_seq, lg, seqs=dev.upload(np.array([i], np.int32), tb.I32))
        assert pool.state()[2].tolist() == lens + [0]
        every, tok = dev.upload(np.array(seqs, np.int32), tb.I32), dev.alloc(B, tb.I32)
        g = dict(group_starts=dev.upload(np.array([0, 1, 4], np.int32), tb.I32), shared=dev.upload(np.array([0, 15, 0], np.int32), tb.I32), n_groups=3, max_shared=15) if grouped else {}
        rates = dev.alloc(B)

        def one():
            pool.extend(every, B)
            b.decode_paged(tok, pool, B, max_seq, lg, seqs=every, **g)
            dev.token_logprobs(b_logits, B, V, tok, entropy=False, out=tb.TokenLogprobs(logprobs=rates))

        b_logits = tb.Buffer(dev, lg.ptr, B * V, tb.F32, owns=False)
        graph = None
        for k in range(steps):
            now = np.array([past[s, lens[s] + k] for s in seqs], np.int32)
            dev.upload_into(tok, now)
            if k == 0:
                one()
                dev.sync()
                dev.begin_capture()
                one()
                graph = dev.end_capture()
            else:
                graph.launch()
            x = dev.download(b_logits).reshape(B, V)
            for i, s in enumerate(seqs):
                rms = np.sqrt(np.mean(want[s, k] ** 2))
                assert np.abs(x[i] - want[s, k]).max() <= 2 * BAR * rms, (grouped, k, s)      # (each within the bar of the oracle)
            assert np.abs(rates.to_vec() - log_softmax(x)[np.arange(B), now]).max() <= logprob_error(x)
        graph.free()
        pool.destroy()
    a.destroy()
    b.destroy()


def test_the_whole_cache_and_long_shared_prefixes(dev, orc):
    """Forks from a fork over a prefix of several tiles: what they read is what one sequence alone reads."""
    import tang_b200 as tb

    host = host_model(9, 8, 2)
    max_seq, V = 512, host.vocab
    model = host.to_device(dev, max_seq, 8)
    tokens = np.random.default_rng(2).integers(0, V, 300).astype(np.int32)
    lg = dev.alloc(8 * V)
    model.prefill(dev.upload(tokens[None], tb.I32), dev.upload(np.zeros(1, np.int32), tb.I32), 1, 300, lg)
    model.decode(dev.upload(tokens[:1], tb.I32), dev.upload(np.array([300], np.int32), tb.I32), 1, max_seq, lg)
    want = dev.download(lg)[:V].astype(np.float64)
    pool = model.page_pool(8, 64)
    refs, tables, lens = pool.state()
    tables[0, :5], refs[:5], lens[0] = np.arange(5), 1, 300
    for buf, v in ((pool.refs, refs), (pool.tables, tables), (pool.lens, lens)):
        dev.upload_into(buf, v)
    pool.fork([0, 0], [1, 2])
    pool.fork([1, 2, 2], [3, 4, 5], keep=[300, 300, 290])
    pool.extend([5], counts=[10])                       # (rows that no step wrote: its step's result is not looked at)
    every = dev.upload(np.arange(6, dtype=np.int32), tb.I32)
    pool.extend(every)
    model.decode_paged(dev.upload(np.full(6, tokens[0], np.int32), tb.I32), pool, 6, max_seq, lg, group_starts=dev.upload(np.array([0], np.int32), tb.I32),
                       shared=dev.upload(np.array([290], np.int32), tb.I32), n_groups=1, max_shared=300)
    x = dev.download(lg).reshape(8, V)
    rms = np.sqrt(np.mean(want ** 2))
    assert np.abs(x[:5] - want).max() <= 2 * BAR * rms
    assert pool.state()[2].tolist() == [301] * 6 + [0, 0]
    pool.destroy()
    model.destroy()


def test_generated_tokens_with_their_log_probabilities(dev, orc):
    import tang_b200 as tb

    host = host_model(12)
    prompts, N = np.array([[5, 17], [44, 3], [5, 17]], np.int32), 6
    cfg = tb.SamplerConfig(0.9, 30, 0.92, 1.3)
    model = host.to_device(dev, 16, 3)
    plain = model.generate(prompts, N, cfg, seed=7)
    tokens, rates = model.generate(prompts, N, cfg, seed=7, logprobs=True)
    assert np.array_equal(tokens, plain) and rates.dtype == np.float32 and rates.shape == tokens.shape
    logits = dev.alloc(3 * host.vocab)
    seqs = np.concatenate([prompts, tokens], 1)
    model.prefill(dev.upload(np.ascontiguousarray(prompts[:, :1]), tb.I32), dev.upload(np.zeros(3, np.int32), tb.I32), 3, 1, logits)
    for p in range(1, N + 1):
        model.decode(dev.upload(np.ascontiguousarray(seqs[:, p]), tb.I32), dev.upload(np.full(3, p, np.int32), tb.I32), 3, N + 2, logits)
        x = dev.download(logits).reshape(3, host.vocab)
        assert np.abs(rates[:, p - 1] - log_softmax(x)[np.arange(3), seqs[:, p + 1]]).max() <= logprob_error(x)
    one = model.generate(prompts[:, :1], 1, logprobs=True)
    assert one[0].shape == one[1].shape == (3, 1)
    model.destroy()


@pytest.mark.parametrize("rows", [7, 64])
def test_given_tokens_rated_by_an_engine(dev, rows):
    """The rates are those of the logits that ``step`` gives for the same portions."""
    import tang_b200 as tb

    cfg = CONFIGS["mixed"]
    w = weights(cfg, 11)
    model = tb.TofazenModel.from_tensors(dev, cfg, views(w), tb.F32, max_slots=3, max_seq=128)
    rng = np.random.default_rng(1)
    texts = [rng.integers(0, cfg["vocab"], n).tolist() for n in (90, 1, 33)]
    e, f = tb.Engine(model, max_rows=rows), tb.Engine(model)
    f.score_rows = rows
    want = e.step([(i, t, range(len(t))) for i, t in enumerate(texts)])
    got = f.score(list(enumerate(texts)), top=5)
    at = 0
    for t, g in zip(texts, got):
        x = want[at:at + len(t)][:-1]
        at += len(t)
        assert g["logprobs"].shape == (len(t) - 1,)
        if not len(x):
            continue
        lp = log_softmax(x)
        assert np.abs(g["logprobs"] - lp[np.arange(len(x)), t[1:]]).max() <= logprob_error(x)
        order = np.argsort(-x, axis=1, kind="stable")[:, :5]
        assert np.array_equal(g["top_ids"], order)
        assert np.abs(g["top_logprobs"] - np.take_along_axis(lp, order, 1)).max() <= logprob_error(x)
    model.destroy()


def test_command_line(dev, tmp_path):
    import tang_b200 as tb

    cfg = CONFIGS["odd"]
    w = weights(cfg, 11)
    save(tmp_path, cfg, w)
    run = lambda *a: subprocess.run([sys.executable, "-m", "tang_b200", *a, "--model", str(tmp_path), "--dtype", "float32"], capture_output=True, text=True, cwd=ROOT)
    r = run("generate", "--prompt", "1,2,3,4", "--max-new", "6", "--logprobs")
    assert r.returncode == 0, r.stderr
    tokens, rates = r.stdout.split()
    text = "1,2,3,4," + tokens
    r = run("score", "--tokens", text, "--tokens", "7")
    assert r.returncode == 0, r.stderr
    lines = r.stdout.split("\n")
    # the same positions' logits, of one step and of steps of one token: the 32-bit model's own bar, and six decimals
    assert len(lines[0].split(",")) == 9 and lines[1] == ""
    assert np.allclose([float(x) for x in lines[0].split(",")][3:], [float(x) for x in rates.split(",")], rtol=0, atol=1e-3)


def test_refusals(dev):
    import tang_b200 as tb

    host = host_model(3)
    model = host.to_device(dev, 48, 2)
    lg, tok = dev.alloc(2 * host.vocab), dev.upload(np.array([1, 2], np.int32), tb.I32)
    pool = model.page_pool(2)
    assert (pool.page_rows, pool.n_pages, pool.max_pages) == (16, 6, 3)
    with pytest.raises(tb.TangqError, match="multiple"):
        model.page_pool(2, 32)
    ints = dev.upload(np.array([0, 1], np.int32), tb.I32)
    for kw in (dict(batch=0), dict(batch=3), dict(max_len=0), dict(max_len=49), dict(group_starts=ints), dict(group_starts=ints, shared=ints, n_groups=3),
               dict(group_starts=ints, shared=ints, n_groups=0)):
        with pytest.raises(tb.TangqError):
            model.decode_paged(**{**dict(token_ids=tok, pool=pool, batch=2, max_len=48, logits=lg), **kw})
    big = tb.PagePool(dev, 7, 16, 2, 3)                # more rows than the caches have
    with pytest.raises(tb.TangqError, match="rows"):
        model.decode_paged(tok, big, 2, 48, lg)
    for prompts, n, m in (([[1, 2]], 4, 3), ([[1, 2]], 4, 0), ([[1, 2], [3, 4]], 4, 2), ([[1] * 40], 9, 2), ([[1, 2]], 0, 1)):
        with pytest.raises(tb.TangqError):
            model.sample(prompts, n, m)
    # sequences without a position, and sequences that do not exist, are reported; the model goes on
    model.decode_paged(tok, pool, 2, 48, lg)
    with pytest.raises(tb.TangqError, match="position"):
        dev.sync()
    pool.extend([0])
    model.decode_paged(tok, pool, 2, 48, lg, seqs=dev.upload(np.array([0, 5], np.int32), tb.I32))
    with pytest.raises(tb.TangqError):
        dev.sync()
    assert model.sample([[1, 2]], 4, 2).tokens.shape == (1, 2, 4)
    odd = host.to_device(dev, 50, 2)
    with pytest.raises(tb.TangqError, match="multiple"):
        odd.sample([[1, 2]], 4, 2)
    for x in (big, pool, model, odd):
        x.destroy()


def caches(model):
    return [b.to_vec() for layer in range(model.cfg.n_layers) for b in model.kv_buffers(layer)[:2]]


def test_a_step_behind_a_refused_call_writes_nothing(dev):
    """A recorded step (extend, decode) whose pool runs out: caches and pool stay as they are to the byte, and the same step goes on once there is room."""
    import tang_b200 as tb

    host = host_model(23)
    V, max_seq, n = host.vocab, 64, 4
    a, b = host.to_device(dev, max_seq, n), host.to_device(dev, max_seq, n)
    prompt = np.random.default_rng(4).integers(0, V, 20).astype(np.int32)
    ints = lambda v: dev.upload(np.asarray(v, np.int32), tb.I32)
    lg = dev.alloc(n * V)
    pool = b.page_pool(6, 16)                          # 16 pages
    one = ints([0])
    for t in prompt:
        pool.extend(one)
        b.decode_paged(ints([t]), pool, 1, max_seq, lg, seqs=one)
    pool.fork([0, 0, 0], [1, 2, 3])
    pool.extend([4, 5], counts=[64, 64])               # 2 + 8 pages held, 6 free: three copies, and then one too few for four new pages
    seqs, tok = ints(np.arange(n)), ints(np.arange(n) + 7)

    def step():
        pool.extend(seqs, n)
        b.decode_paged(tok, pool, n, max_seq, lg)

    step()
    dev.sync()
    dev.begin_capture()
    step()
    graph = dev.end_capture()
    for _ in range(21, 32):
        graph.launch()
    dev.sync()
    assert pool.state()[2].tolist() == [32] * 4 + [64] * 2
    before, state = caches(b), pool.state()
    dev.upload_into(tok, np.arange(n) + 90)            # (the tokens of the step before would give the rows that are there)
    for _ in range(2):
        graph.launch()
        with pytest.raises(tb.TangqError) as e:
            dev.sync()
        assert e.value.status == tb._lib.TQ_ENOMEM
        assert all(np.array_equal(x, y) for x, y in zip(before, caches(b))) and all(np.array_equal(x, y) for x, y in zip(state, pool.state()))
    b.decode_paged(tok, pool, 2, max_seq, lg, seqs=ints([2, 0]))       # and without asking once more
    with pytest.raises(tb.TangqError) as e:
        dev.sync()
    assert e.value.status == tb._lib.TQ_EINVAL and all(np.array_equal(x, y) for x, y in zip(before, caches(b)))
    pool.extend([2, 0], counts=[0, 0])                 # (no new position: still not)
    b.decode_paged(tok, pool, 2, max_seq, lg, seqs=ints([2, 0]))
    with pytest.raises(tb.TangqError):
        dev.sync()
    assert all(np.array_equal(x, y) for x, y in zip(before, caches(b)))
    pool.free([5])
    dev.upload_into(tok, np.arange(n) + 7)
    graph.launch()
    dev.sync()
    got = dev.download(lg).reshape(n, V)
    assert pool.state()[2].tolist() == [33] * 4 + [64, 0]
    for j in range(n):                                 # as over slots
        for p, t in enumerate([*prompt, *[j + 7] * 13]):
            a.decode(ints([t]), ints([p]), 1, max_seq, lg)
        want = dev.download(lg)[:V]
        assert np.abs(got[j] - want).max() <= 2 * BAR * np.sqrt(np.mean(want.astype(np.float64) ** 2)), j
    graph.free()
    pool.destroy()
    a.destroy()
    b.destroy()


def test_a_forked_sequence_is_not_stepped_before_it_is_extended(dev):
    import tang_b200 as tb

    host = host_model(24)
    model = host.to_device(dev, 64, 4)
    ints = lambda v: dev.upload(np.asarray(v, np.int32), tb.I32)
    lg = dev.alloc(4 * host.vocab)
    for n in (5, 16):
        pool = model.page_pool(4, 16)
        for t in range(n):
            pool.extend([0])
            model.decode_paged(ints([t]), pool, 1, 64, lg)
        pool.fork([0], [2])
        dev.sync()
        before = caches(model)
        for seqs in ([2], [0], [2, 0]):
            model.decode_paged(ints([3, 4]), pool, len(seqs), 64, lg, seqs=ints(seqs))
            with pytest.raises(tb.TangqError) as e:
                dev.sync()
            assert e.value.status == tb._lib.TQ_EINVAL
            assert all(np.array_equal(x, y) for x, y in zip(before, caches(model)))
        pool.extend([2, 0])
        model.decode_paged(ints([3, 4]), pool, 2, 64, lg, seqs=ints([2, 0]))
        dev.sync()
        assert not all(np.array_equal(x, y) for x, y in zip(before, caches(model)))
        pool.destroy()
    model.destroy()


def test_a_pool_of_another_handle_is_refused(dev):
    """Its calls run on another stream, with nothing to order them."""
    import tang_b200 as tb

    host = host_model(25)
    model, other = host.to_device(dev, 64, 2), tb.QuantComputeDevice(0)
    pool = tb.PagePool(other, 8, 16, 2, 4)
    tok, lg = dev.upload(np.zeros(2, np.int32), tb.I32), dev.alloc(2 * host.vocab)
    with pytest.raises(tb.TangqError, match="context"):
        model.decode_paged(tok, pool, 2, 64, lg)
    kv = dev.alloc(8 * 16 * 256, tb.BF16)
    with pytest.raises(tb.TangqError, match="context"):
        dev.gqa_decode_paged(dev.alloc(2 * 512, tb.BF16), kv, kv, pool, 2, 4, 2, 128, 64)
    pool.destroy()
    other.close()
    model.destroy()


def test_the_calls_of_the_integration_guide(dev):
    """Prefill, the pool's state, fork, one step as it is, the rest from a graph: through the C interface, and the same tokens as ``sample``."""
    import ctypes as C

    import tang_b200 as tb

    host = host_model(27)
    V, max_seq, n, n_new, length = host.vocab, 256, 3, 9, 150
    model = host.to_device(dev, max_seq, n)
    prompt = np.random.default_rng(27).integers(0, V, length).astype(np.int32)
    cfg = tb.SamplerConfig(0.9, 0, 1.0, 1.0)
    want = model.sample(prompt[None], n_new, n, cfg, seed=5)

    L, ctx, m, vp = dev._L, dev._ctx, C.c_void_p(model.handle), C.c_void_p
    ok = lambda st: dev._check(st)
    keep = []

    def ints(v):
        keep.append(dev.upload(np.asarray(v, np.int32), tb.I32))
        return vp(keep[-1].ptr)

    def room(k, dtype=tb.F32):
        keep.append(dev.alloc(k, dtype))
        return vp(keep[-1].ptr)

    page_rows = 64
    n_pages, table_ld = n * max_seq // page_rows, max_seq // page_rows
    pool, arrays = vp(), [b for layer in range(host.n_layers) for b in model.kv_buffers(layer)[:2]]
    for b in arrays:
        dev.memset(b, 0xFF)                            # (NaN wherever these calls do not write)
    ok(L.tq_pages_create(ctx, n_pages, page_rows, n, table_ld, None, None, None, C.byref(pool)))
    ok(L.tq_pages_arrays(pool, (vp * len(arrays))(*[b.ptr for b in arrays]), len(arrays), host.n_kv * host.hd * 2))
    held = length - 1
    used = -(-held // page_rows)
    refs, tables, lens = np.zeros(n_pages, np.int32), np.full((n, table_ld), -1, np.int32), np.zeros(n, np.int32)
    refs[:used], tables[0, :used], lens[0] = 1, np.arange(used), held
    logits, rates, chosen = room(n * V), room(n), room(n, tb.I32)
    ok(L.tq_llama_prefill(m, ints(prompt[:held]), ints([0]), 1, held, logits))
    state = [vp() for _ in range(3)]
    ok(L.tq_pages_data(pool, *(C.byref(p) for p in state)))
    for p, a in zip(state, (refs, tables, lens)):
        ok(L.tq_upload(ctx, p, vp(a.ctypes.data), a.nbytes))
    ok(L.tq_pages_fork(pool, ints([0] * (n - 1)), ints(range(1, n)), None, n - 1))
    tokens, positions, out_tokens, step_no = ints([prompt[-1]] * n), ints([held] * n), ints(np.zeros((n, n_new))), ints([0])
    seqs, starts, shared = ints(range(n)), ints([0]), ints([held])
    keep.append(dev.upload((5 + np.arange(n, dtype=np.uint64)).view(np.float64), tb.F64))
    rng = vp(keep[-1].ptr)

    def step():
        ok(L.tq_pages_extend(pool, seqs, None, n))
        ok(L.tq_llama_decode_paged(m, tokens, pool, seqs, n, starts, shared, 1, held, length + n_new, logits))
        ok(L.tq_sample(ctx, logits, 1, n, V, C.byref(cfg), rng, None, None, 0, chosen))
        ok(L.tq_token_logprobs(ctx, logits, tb.F32, 0, 1, n, V, chosen, 1, 0, rates, None, None, None))
        ok(L.tq_generate_advance(ctx, chosen, n, tokens, positions, out_tokens, n_new, step_no, None))

    step()
    ok(L.tq_graph_begin(ctx))
    step()
    g = vp()
    ok(L.tq_graph_end(ctx, C.byref(g)))
    for _ in range(1, n_new):
        ok(L.tq_graph_launch(ctx, g))
    dev.sync()
    read = lambda p: next(b for b in keep if b.ptr == p.value).to_vec()
    assert np.array_equal(read(out_tokens).reshape(n, n_new), want.tokens[0]) and np.array_equal(read(rates), want.logprobs[0, :, -1])
    ok(L.tq_graph_free(ctx, g))
    L.tq_pages_destroy(pool)
    model.destroy()


def test_a_models_pools_go_with_it(dev):
    """They would copy rows of caches that are gone; so would a recorded step."""
    import tang_b200 as tb

    host = host_model(29)
    model, other = host.to_device(dev, 64, 2), host.to_device(dev, 64, 2)
    pool, more = model.page_pool(2), other.page_pool(2)
    seqs, tok, lg = dev.upload(np.arange(2, dtype=np.int32), tb.I32), dev.upload(np.zeros(2, np.int32), tb.I32), dev.alloc(2 * host.vocab)

    def step(m, p):
        p.extend(seqs)
        m.decode_paged(tok, p, 2, 64, lg)

    graphs = []
    for m, p in ((model, pool), (other, more)):
        step(m, p)
        dev.sync()
        dev.begin_capture()
        step(m, p)
        graphs.append(dev.end_capture())
    model.destroy()
    with pytest.raises(tb.TangqError, match="pool of pages"):
        graphs[0].launch()
    for call in (lambda: pool.extend(seqs), lambda: pool.free(seqs), pool.compact):
        with pytest.raises(tb.TangqError):
            call()
    graphs[1].launch()
    dev.sync()
    assert more.state()[2].tolist() == [2, 2]
    for x in graphs:
        x.free()
    other.destroy()
    pool.destroy()


def test_a_sequence_that_stands_in_a_step_twice(dev):
    """Two tokens for one place: reported, and nothing is written for it; the others' step is what it is without it."""
    import tang_b200 as tb

    host = host_model(31)
    model = host.to_device(dev, 64, 4)
    pool, ints, lg = model.page_pool(4, 16), lambda v: dev.upload(np.asarray(v, np.int32), tb.I32), dev.alloc(4 * host.vocab)
    for t in range(7):
        pool.extend([0, 1, 2])
        model.decode_paged(ints([t, t + 1, t + 2]), pool, 3, 64, lg)
    pool.extend([0, 1, 2])
    dev.sync()
    before = caches(model)
    model.decode_paged(ints([5, 6, 7, 8]), pool, 4, 64, lg, seqs=ints([0, 1, 0, 2]))
    with pytest.raises(tb.TangqError) as e:
        dev.sync()
    assert e.value.status == tb._lib.TQ_EINVAL
    after, refs_tables = caches(model), pool.state()[1]
    pages = [int(refs_tables[s, 0]) for s in range(3)]
    width = host.n_kv * host.hd
    for a, b in zip(before, after):
        a, b = (x.reshape(-1, 16, width) for x in (a, b))
        assert np.array_equal(a[pages[0]], b[pages[0]]) and not np.array_equal(a[pages[1], 7], b[pages[1], 7]) and not np.array_equal(a[pages[2], 7], b[pages[2], 7])
        rest = np.ones(a.shape[:2], bool)
        rest[pages[1], 7] = rest[pages[2], 7] = False
        assert np.array_equal(a[rest], b[rest])
    model.decode_paged(ints([5, 6, 8]), pool, 3, 64, lg)
    dev.sync()
    pool.destroy()
    model.destroy()
