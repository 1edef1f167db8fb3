"""Host-side driver of the Llama-shaped decode step (``tq_llama_*`` in include/tangq.h), mirroring
the reference's decode loop, crates/tang-train/examples/smollm.rs:255-296 (``LlamaModel::forward``
for one new token per sequence) and its use of ``tang_infer::KVCache``."""
from __future__ import annotations

import ctypes as C
import weakref
from dataclasses import dataclass

import numpy as np

from . import _lib
from .device import Buffer, QBuffer, QuantComputeDevice, _check_types
from .generation import check_lengths, decode_loop
from .pages import PagePool


class LlamaConfig(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in ("n_layers", "d_model", "n_heads", "n_kv_heads", "head_dim", "ffn", "vocab",
                                          "max_seq", "max_batch")] + [("eps", C.c_float), ("rope_base", C.c_double)]


class Comm:
    """NCCL communicator bound to a device context (``tq_comm_*``)."""

    def __init__(self, dev: QuantComputeDevice, unique_id: bytes, rank: int, world: int):
        self.dev = dev
        h = C.c_void_p()
        buf = C.create_string_buffer(unique_id, 128)
        dev._check(dev._L.tq_comm_create(dev._ctx, buf, rank, world, C.byref(h)))
        self.handle, self.rank, self.world = h.value, rank, world

    @staticmethod
    def unique_id() -> bytes:
        buf = C.create_string_buffer(128)
        st = _lib.load().tq_comm_unique_id(buf)
        if st != _lib.TQ_OK:
            raise _lib.TangqError(st, "tq_comm_unique_id failed (NCCL not loadable?)")
        return buf.raw

    def enable_peer(self, max_elems: int) -> None:
        """Peer-memory path for all-reduces of up to `max_elems` floats (``tq_comm_enable_peer``); collective."""
        self.dev._check(self.dev._L.tq_comm_enable_peer(self.dev._ctx, C.c_void_p(self.handle), max_elems))

    @classmethod
    def peer_local(cls, dev: QuantComputeDevice, rank: int, world: int, bufs, max_elems: int) -> "Comm":
        """A communicator over buffers already visible to this GPU (``tq_comm_peer_local``): `bufs[r]` is rank r's."""
        self = cls.__new__(cls)
        self.dev = dev
        arr = (C.c_void_p * world)(*[b.ptr for b in bufs])
        h = C.c_void_p()
        dev._check(dev._L.tq_comm_peer_local(dev._ctx, rank, world, arr, max_elems, C.byref(h)))
        self.handle, self.rank, self.world = h.value, rank, world
        return self

    def set_wait_limit(self, polls: int) -> None:
        st = self.dev._L.tq_comm_set_wait_limit(C.c_void_p(self.handle), polls)
        if st != _lib.TQ_OK:
            raise _lib.TangqError(st, "tq_comm_set_wait_limit: no peer path on this communicator")

    def all_reduce(self, buf: Buffer) -> None:
        self.dev._check(self.dev._L.tq_all_reduce_f32(self.dev._ctx, C.c_void_p(self.handle), C.c_void_p(buf.ptr), buf.n))

    def destroy(self) -> None:
        if self.handle:
            self.dev._L.tq_comm_destroy(self.dev._ctx, C.c_void_p(self.handle))
            self.handle = 0


@dataclass
class LlamaLayerWeights:
    """One block's device weights in the fused form the kernels take (shard shapes under TP)."""
    wqkv: QBuffer
    wo: QBuffer
    wgate_up: QBuffer
    wdown: QBuffer
    attn_norm: Buffer   # bf16 [d_model]
    ffn_norm: Buffer    # bf16 [d_model]


@dataclass
class Samples:
    """What ``LlamaModel.sample`` draws: int32 and f32 [prompts, samples, n_new], and for every prompt its samples' numbers from the
    likeliest (largest sum of log probabilities) to the least."""
    tokens: np.ndarray
    logprobs: np.ndarray
    order: np.ndarray


class LlamaModel:
    def __init__(self, dev: QuantComputeDevice, cfg: LlamaConfig, comm: Comm | None = None):
        self.dev, self.cfg, self.comm = dev, cfg, comm
        self.tp = comm.world if comm else 1
        h = C.c_void_p()
        dev._check(dev._L.tq_llama_create(dev._ctx, C.byref(cfg), C.c_void_p(comm.handle if comm else 0), C.byref(h)))
        self.handle = h.value
        self._keep = []
        self._pools = weakref.WeakSet()      # over this model's caches

    def set_layer(self, layer: int, w: LlamaLayerWeights) -> None:
        self._keep.append(w)
        self.dev._check(self.dev._L.tq_llama_set_layer(
            C.c_void_p(self.handle), layer, C.c_void_p(w.wqkv.handle), C.c_void_p(w.wo.handle),
            C.c_void_p(w.wgate_up.handle), C.c_void_p(w.wdown.handle), C.c_void_p(w.attn_norm.ptr),
            C.c_void_p(w.ffn_norm.ptr)))

    def set_head(self, embed: Buffer, final_norm: Buffer, lm_head: QBuffer) -> None:
        self._keep.append((embed, final_norm, lm_head))
        self.dev._check(self.dev._L.tq_llama_set_head(C.c_void_p(self.handle), C.c_void_p(embed.ptr),
                                                      C.c_void_p(final_norm.ptr), C.c_void_p(lm_head.handle)))

    def kv_cache(self, layer: int):
        """(k_ptr, v_ptr, seq_stride_elems) of this rank's bf16 cache for `layer`."""
        k, v, s = C.c_void_p(), C.c_void_p(), C.c_size_t()
        self.dev._check(self.dev._L.tq_llama_kv_cache(C.c_void_p(self.handle), layer, C.byref(k), C.byref(v), C.byref(s)))
        return k.value, v.value, s.value

    def kv_buffers(self, layer: int):
        k, v, s = self.kv_cache(layer)
        n = self.cfg.max_batch * s
        return (Buffer(self.dev, k, n, _lib.BF16, owns=False), Buffer(self.dev, v, n, _lib.BF16, owns=False), s)

    def trim_to(self, seq_lens: Buffer, batch: int, keep: int) -> None:
        """``KVCache::trim_to(keep)`` (crates/tang-infer/src/kv_cache.rs:138-149) for `batch` sequences: each keeps its
        last `keep` positions (moved to the front of its cache rows); `seq_lens` (int32, device) is updated in place."""
        self.dev._check(self.dev._L.tq_llama_kv_trim(C.c_void_p(self.handle), C.c_void_p(seq_lens.ptr), batch, keep))

    def decode(self, token_ids: Buffer, positions: Buffer, batch: int, max_len: int, logits: Buffer,
               rope_positions: Buffer | None = None) -> None:
        """``model.forward(&[tok], cache, pos)`` for `batch` sequences (smollm.rs:535); asynchronous.  `positions` are the
        cache rows the new tokens are appended at; `rope_positions` the positions their rotation uses when that differs
        (a trimmed cache)."""
        self.dev._check(self.dev._L.tq_llama_decode_at(C.c_void_p(self.handle), C.c_void_p(token_ids.ptr), C.c_void_p(positions.ptr),
                                                       C.c_void_p(rope_positions.ptr if rope_positions is not None else 0),
                                                       batch, max_len, C.c_void_p(logits.ptr)))

    def prefill(self, token_ids: Buffer, cache_start: Buffer, batch: int, q_len: int, logits: Buffer) -> None:
        """``model.forward(&tokens, cache, pos)`` for a chunk of `q_len` tokens per sequence (prompt processing): appends the
        chunk to the cache and leaves the logits of each sequence's last chunk position; asynchronous."""
        self.dev._check(self.dev._L.tq_llama_prefill(C.c_void_p(self.handle), C.c_void_p(token_ids.ptr), C.c_void_p(cache_start.ptr),
                                                     batch, q_len, C.c_void_p(logits.ptr)))

    def page_pool(self, n_seqs: int, page_rows: int | None = None, **state) -> PagePool:
        """A ``PagePool`` over the caches of all layers, seen as max_batch * max_seq / page_rows pages: the rows that ``prefill`` and ``decode``
        give sequence b are the pages from b * max_seq / page_rows on.  `page_rows`: the largest of 64, 32 and 16 that divides max_seq unless
        given.  `state`: refs, tables, lens of ``PagePool``.  The pool starts empty: rows that ``prefill`` wrote become a sequence's when its state
        says so (see ``sample``).  It is destroyed with the model."""
        c = self.cfg
        if page_rows is None:
            page_rows = next((p for p in (64, 32, 16) if c.max_seq % p == 0), 0)
        if page_rows < 1 or c.max_seq % page_rows:
            raise _lib.TangqError(_lib.TQ_EINVAL, f"page_pool: max_seq {c.max_seq} is not a multiple of the pages' rows (16 or more)")
        arrays = [b for layer in range(c.n_layers) for b in self.kv_buffers(layer)[:2]]
        pool = PagePool(self.dev, c.max_batch * c.max_seq // page_rows, page_rows, n_seqs, c.max_seq // page_rows, arrays, **state)
        self._pools.add(pool)
        return pool

    def decode_paged(self, token_ids: Buffer, pool: PagePool, batch: int, max_len: int, logits: Buffer, seqs: Buffer | None = None,
                     group_starts: Buffer | None = None, shared: Buffer | None = None, n_groups: int = 0, max_shared: int = 0) -> None:
        """``decode`` over a ``page_pool``: the last position of each sequence, for which ``PagePool.extend`` has made room, is its new token's
        (``tq_llama_decode_paged``); sequences and groups as in ``gqa_decode_paged``."""
        if token_ids.n < batch or logits.n < batch * self.cfg.vocab or (seqs is not None and seqs.n < batch):
            raise _lib.TangqError(_lib.TQ_EINVAL, "decode_paged: buffer sizes do not match the batch")
        if group_starts is not None and (group_starts.n < n_groups or shared is None or shared.n < n_groups):
            raise _lib.TangqError(_lib.TQ_EINVAL, "decode_paged: fewer starts or shared lengths than groups")
        _check_types("decode_paged", _lib.I32, token_ids=token_ids, seqs=seqs, group_starts=group_starts, shared=shared)
        _check_types("decode_paged", _lib.F32, logits=logits)
        ptr = lambda b: C.c_void_p(b.ptr if b is not None else 0)
        self.dev._check(self.dev._L.tq_llama_decode_paged(C.c_void_p(self.handle), ptr(token_ids), C.c_void_p(pool.handle), ptr(seqs), batch,
                                                          ptr(group_starts), ptr(shared), n_groups, max_shared, max_len, ptr(logits)))

    def sample(self, prompts, n_new: int, samples: int, sampling=None, seed: int = 42, comm_world: int = 1) -> Samples:
        """`samples` continuations of each prompt (equal lengths), each with its log probability.  A prompt is run through the model and kept in
        the cache once: its samples are forked from it, share its pages and attend them as one group.  Sample j draws as ``generate`` with
        seed + j does.  Uses the whole cache; prompts * samples are at most max_batch."""
        prompts = np.asarray(prompts, np.int32)
        check_lengths(prompts, n_new, self.cfg.max_seq)
        dev, c = self.dev, self.cfg
        B, P = prompts.shape
        if samples < 1 or B * samples > c.max_batch:
            raise _lib.TangqError(_lib.TQ_EINVAL, f"sample: {B} prompts with {samples} samples each need a model of that many sequences")
        N, first = B * samples, np.arange(B, dtype=np.int32) * samples
        pool = self.page_pool(N)
        try:
            if P > 1:
                scratch = dev.alloc(B * c.vocab, _lib.F32)
                self.prefill(dev.upload(np.ascontiguousarray(prompts[:, :P - 1]), _lib.I32), dev.upload(np.zeros(B, np.int32), _lib.I32), B, P - 1,
                             scratch)
                # the first sample of prompt i takes over the pages of the rows that prefill gave prompt i
                refs, tables, lens = np.zeros(pool.n_pages, np.int32), np.full((N, pool.max_pages), -1, np.int32), np.zeros(N, np.int32)
                used = -(-(P - 1) // pool.page_rows)
                for i, s in enumerate(first):
                    tables[s, :used] = i * pool.max_pages + np.arange(used)
                    refs[tables[s, :used]] = 1
                    lens[s] = P - 1
                for buf, v in ((pool.refs, refs), (pool.tables, tables), (pool.lens, lens)):
                    dev.upload_into(buf, v)
                if samples > 1:
                    pool.fork(np.repeat(first, samples - 1), [s + j for s in first for j in range(1, samples)])
            every, starts = dev.upload(np.arange(N, dtype=np.int32), _lib.I32), dev.upload(first, _lib.I32)
            shared = dev.upload(np.full(B, P - 1, np.int32), _lib.I32)

            def step(tok, pos, logits):
                pool.extend(every, N)
                self.decode_paged(tok, pool, N, P + n_new, logits, group_starts=starts, shared=shared, n_groups=B, max_shared=P - 1)

            tokens, logprobs = decode_loop(dev, step, np.repeat(prompts, samples, 0), n_new, c.vocab, sampling,
                                           np.tile(seed + np.arange(samples, dtype=np.uint64), B), comm_world, logprobs=True)
        finally:
            dev.sync()
            pool.destroy()
        tokens, logprobs = tokens.reshape(B, samples, n_new), logprobs.reshape(B, samples, n_new)
        return Samples(tokens, logprobs, np.argsort(-logprobs.sum(2, dtype=np.float64), axis=1, kind="stable"))

    def generate(self, prompts, n_new: int, sampling=None, seed: int = 42, comm_world: int = 1, logprobs: bool = False):
        """``generate`` (crates/tang-infer/src/sampling.rs:229-256) for a batch of equal-length prompts.  The prompt
        goes through one prefill chunk (all tokens but the last); then decode -> ``Sampler::sample`` -> advance is captured
        once as a CUDA graph and replayed `n_new` times, the logits never leaving the device.  `sampling` is a
        ``SamplerConfig`` (None or temperature 0: greedy, the first maximum); every sequence owns an LCG seeded
        with `seed` (as ``Sampler::with_seed`` per call of ``generate``); the repetition penalty sees the prompt and
        everything generated so far.  Returns int32 [batch, n_new]; the caller cuts at its stop token (what is
        drawn before a stop token does not depend on what follows); with `logprobs` also the tokens' log probabilities,
        f32 [batch, n_new]."""
        prompts = np.asarray(prompts, np.int32)
        check_lengths(prompts, n_new, self.cfg.max_seq)
        dev = self.dev
        B, P = prompts.shape
        if P > 1:                                   # all prompt tokens but the last: one prefill chunk fills the cache
            scratch = dev.alloc(B * self.cfg.vocab, _lib.F32)
            self.prefill(dev.upload(np.ascontiguousarray(prompts[:, :P - 1]), _lib.I32), dev.upload(np.zeros(B, np.int32), _lib.I32),
                         B, P - 1, scratch)
        return decode_loop(dev, lambda tok, pos, logits: self.decode(tok, pos, B, P + n_new, logits), prompts, n_new,
                           self.cfg.vocab, sampling, seed, comm_world, logprobs)

    def generate_greedy(self, prompts, n_new: int, comm_world: int = 1) -> np.ndarray:
        """``generate`` with ``SamplingConfig::greedy()``."""
        return self.generate(prompts, n_new, None, comm_world=comm_world)

    def destroy(self) -> None:
        if self.handle:
            for pool in list(self._pools):
                pool.destroy()
            self.dev._L.tq_llama_destroy(C.c_void_p(self.handle))
            self.handle = 0
