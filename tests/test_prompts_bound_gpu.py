"""Prompts through the model over pages whose lengths pass the bound that the caller gives."""
import numpy as np
import pytest

from test_prompts_gpu import BAR, Followed, host_model, near  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    import tang_b200

    d = tang_b200.QuantComputeDevice(0)
    yield d
    d.close()


@pytest.mark.parametrize("over", [0, 1, 20])
def test_a_prompt_longer_than_the_bound_is_reported(dev, orc, over):
    """Positions from the bound on are written in no layer; those before it, and the other sequence, are what they are under a bound that holds."""
    import tang_b200 as tb

    host, max_seq, bound = host_model(21), 256, 60
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, host.vocab, n) for n in (bound + over, 33)]
    ints = lambda v: dev.upload(np.asarray(v, np.int32), tb.I32)  # noqa: E731
    caches = []
    for max_len in (max_seq, bound):
        model = host.to_device(dev, max_seq, 2)
        pool = model.page_pool(2, 16)
        bufs = [b for layer in range(host.n_layers) for b in model.kv_buffers(layer)[:2]]
        for b in bufs:
            dev.upload_into(b, np.full(b.n, 0x1234, np.uint16))
        lg = dev.alloc(2 * host.vocab)
        pool.extend([0, 1], counts=[len(p) for p in prompts])
        model.prefill_paged(ints(np.concatenate(prompts)), pool, 2, sum(map(len, prompts)), max_len, lg, seq_rows=ints([0, len(prompts[0]), bound + over + 33]))
        logits = lg.to_vec().reshape(2, -1)
        if over and max_len == bound:
            with pytest.raises(tb.TangqError):
                dev.sync()
        else:
            dev.sync()
            assert near(logits[0], Followed(host, orc, max_seq).run(prompts[0]))
        assert near(logits[1], Followed(host, orc, max_seq).run(prompts[1]))
        table = pool.tables.to_vec().reshape(2, -1)
        caches.append([(b.to_vec().reshape(2 * max_seq, -1), table) for b in bufs])
        model.destroy()
    for (want, table), (got, table2) in zip(*caches):
        assert np.array_equal(table, table2)
        want = want.copy()
        past = np.arange(bound, bound + over)
        want[table[0, past // 16] * 16 + past % 16] = 0x1234
        assert np.array_equal(got, want)
