"""What the operators for several continuations of one prompt are measured on.

  logprobs   log probabilities of given tokens, entropy and the most likely tokens, from rows of logits
  attention  decode attention over a cache of pages, one new token per sequence; the positions that a group of sequences
             shares (their prompt) stand in the same pages
  fork       sequences are released, forked from others and extended by a token or more; a partly filled page that another
             sequence holds too is copied first
  compact    the pages in use move to the front of the pool

Head counts are those of the Llama shapes of perf/cases.py, vocabularies those of its models; caches, queries and logits
are normal values, lengths and page numbers follow from the seed.  ``run`` without ``own`` is the operator in elementary torch
operations, ``exact`` computes the same in 64 bits.
"""
import math

import torch

own = False

HEADS = {"8b": (32, 8), "1b": (16, 4), "one_to_one": (8, 8), "one_kv": (8, 1)}   # query heads, KV heads
DIM = 128
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of a single user's generation: latency
        {"name": "logprobs_1", "path": "logprobs", "rows": 1, "cols": 32000, "slices": 1, "dtype": "f32", "top": 5, "entropy": True, "masked": 0.0},
        # a server's decode step, the largest number of alternatives that a client asks for
        {"name": "logprobs_64_top20", "path": "logprobs", "rows": 64, "cols": 128256, "slices": 1, "dtype": "f32", "top": 20, "entropy": True, "masked": 0.0},
        # scoring the tokens of a prompt, one after the other: no alternatives
        {"name": "logprobs_score_2048", "path": "logprobs", "rows": 2048, "cols": 128256, "slices": 1, "dtype": "bf16", "top": 0, "entropy": False, "masked": 0.0},
        # a vocabulary gathered from four ranks, an odd number of columns, most tokens ruled out by a grammar
        {"name": "logprobs_ranks_masked", "path": "logprobs", "rows": 17, "cols": 8013, "slices": 4, "dtype": "f32", "top": 8, "entropy": True, "masked": 0.98},
        # a single sequence with a short context: latency
        {"name": "attention_1", "path": "attention", "heads": "8b", "batch": 1, "members": 1, "shared": 0, "own_most": 700, "page": 16, "out": "bf16"},
        # eight samples of one prompt, just begun
        {"name": "attention_8_samples", "path": "attention", "heads": "8b", "batch": 8, "members": 8, "shared": 2040, "own_most": 128, "page": 32, "out": "bf16"},
        # a batch behind one long system prompt
        {"name": "attention_64_one_prefix", "path": "attention", "heads": "8b", "batch": 64, "members": 64, "shared": 8192, "own_most": 512, "page": 64, "out": "bf16"},
        # several users with four samples each, odd lengths; f32 results, as a caller takes who adds up several parts
        {"name": "attention_16_groups", "path": "attention", "heads": "1b", "batch": 64, "members": 4, "shared": 1001, "own_most": 999, "page": 16, "out": "f32"},
        # nothing shared: as many bytes as the largest batch of the Llama-shaped model reads
        {"name": "attention_64_alone", "path": "attention", "heads": "8b", "batch": 64, "members": 1, "shared": 0, "own_most": 2048, "page": 128, "out": "bf16"},
        # four samples of a short prompt in a small model's cache, one token each: latency of the bookkeeping
        {"name": "fork_4", "path": "fork", "arrays": 8, "kv_heads": 4, "page": 16, "pages": 512, "sources": 1, "members": 4, "length": 135, "more": 1},
        # eight prompts, eight samples each, half a page to copy for each of them
        {"name": "fork_64", "path": "fork", "arrays": 32, "kv_heads": 8, "page": 64, "pages": 400, "sources": 8, "members": 8, "length": 992, "more": 1},
        # a pool that requests of all lengths have left half full
        {"name": "compact_half", "path": "compact", "arrays": 16, "kv_heads": 8, "page": 32, "pages": 1024, "used": 512, "sequences": 40},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: a kind as often as it is listed, sizes over its whole range."""
    path = rng.choice(["logprobs"] * 4 + ["attention"] * 5 + ["fork"] * 2 + ["compact"])
    if path == "logprobs":
        slices = rng.choice([1, 1, 1, 2, 4])
        cols = _log(rng, 1000, 128256) // slices
        rows = _log(rng, 1, 2048)
        return {"path": path, "rows": rows, "cols": cols, "slices": slices, "dtype": rng.choice(["f32", "bf16"]) if rows * cols * slices <= 2048 * 64128 else "bf16",
                "top": rng.choice([0, 0, 1, 5, 8, 20]), "entropy": rng.random() < 0.6, "masked": rng.choice([0.0, 0.0, 0.5, 0.98])}
    if path == "attention":
        members = rng.choice([1, 2, 4, 8, 16, 64])
        batch = members * max(1, _log(rng, 1, 64) // members)
        shared = _log(rng, 16, 8192) if members > 1 else 0
        return {"path": path, "heads": rng.choice(list(HEADS)), "batch": batch, "members": members, "shared": shared,
                "own_most": _log(rng, 1, 512 if members > 1 else 2048), "page": rng.choice([16, 32, 64, 128]),
                "out": rng.choice(["bf16", "bf16", "bf16", "f32"])}
    if path == "fork":
        sources, members, page = _log(rng, 1, 8), _log(rng, 1, 8), rng.choice([16, 32, 64])
        length, more = _log(rng, 1, 992), rng.choice([1, 1, 1, _log(rng, 2, 100)])
        pages = sources * (-(-length // page)) + sources * members * (5 + -(-more // page))
        return {"path": path, "arrays": 2 * _log(rng, 1, 16), "kv_heads": rng.choice([1, 4, 8]), "page": page, "pages": pages + _log(rng, 1, 200),
                "sources": sources, "members": members, "length": length, "more": more}
    pages = _log(rng, 32, 1024)
    used = max(1, int(pages * rng.uniform(0.1, 0.95)))
    return {"path": path, "arrays": 2 * _log(rng, 1, 8), "kv_heads": rng.choice([1, 4, 8]), "page": rng.choice([16, 32]), "pages": pages, "used": used,
            "sequences": max(1, used // rng.choice([2, 5, 13]))}


# ---------------------------------------------------------------------------------------------- inputs
def _gen(seed, tag=0):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + tag)


def _host(seed, tag=0):
    return torch.Generator().manual_seed(int(seed) * 1000003 + tag)


def _ints(values):
    return torch.as_tensor(values, dtype=torch.int32).cuda()


def prepare(case, seed):
    return {"logprobs": prepare_logprobs, "attention": prepare_attention, "fork": prepare_fork, "compact": prepare_compact}[case["path"]](case, seed)


def prepare_logprobs(case, seed):
    S, R, C, g = case["slices"], case["rows"], case["cols"], _gen(seed)
    dt = TYPES[case["dtype"]]
    x = torch.empty((S, R, C), dtype=dt, device="cuda")
    for s in range(S):
        x[s].normal_(0.0, 2.5, generator=g)
    best = torch.randint(0, S * C, (R,), device="cuda", generator=g)   # what the model is sure of, more or less
    rows = torch.arange(R, device="cuda")
    x[best // C, rows, best % C] = torch.empty(R, device="cuda").uniform_(6.0, 18.0, generator=g).to(dt)
    if case["masked"]:
        gone = torch.rand((S, 1, C), device="cuda", generator=g) < case["masked"]
        x.masked_fill_(gone, -math.inf)
        x[best // C, rows, best % C] = 9.0
    other = torch.randint(0, S * C, (R,), device="cuda", generator=g)
    tokens = torch.where(torch.rand(R, device="cuda", generator=g) < 0.7, best, other).int()
    new = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    out = {"logprobs": new(R), "entropy": new(R) if case["entropy"] else None, "top_ids": new(R, case["top"], dtype=torch.int32) if case["top"] else None,
           "top_logprobs": new(R, case["top"]) if case["top"] else None}
    return {"case": case, "x": x, "tokens": tokens, "out": out}


def _attention_lengths(case, seed):
    """Positions of every sequence: the shared ones and, from 1 to `own_most`, its own (each group has a member with the most)."""
    h, B, m = _host(seed, 1), case["batch"], case["members"]
    more = torch.randint(1, case["own_most"] + 1, (B,), generator=h)
    more[::m] = case["own_most"]
    return case["shared"] + more


def _attention_tables(case, seed):
    """Lengths [batch], tables [batch][pages] and the number of pages; the whole pages of the shared positions are the first member's."""
    P, B, m, lens = case["page"], case["batch"], case["members"], _attention_lengths(case, seed)
    whole = case["shared"] // P
    held = (lens + P - 1) // P
    ld = int(held.max())
    n_pages = (B // m) * whole + int((held - whole).sum()) + 5
    order = torch.randperm(n_pages, generator=_host(seed, 2)).int()
    tables = torch.full((B, ld), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        if b % m == 0:
            first, at = order[at:at + whole], at + whole
        tables[b, :whole] = first
        n = int(held[b]) - whole
        tables[b, whole:whole + n] = order[at:at + n]
        at += n
    return lens.int(), tables, n_pages, whole * P


def prepare_attention(case, seed):
    H, G = HEADS[case["heads"]]
    B, m, P = case["batch"], case["members"], case["page"]
    lens, tables, n_pages, shared = _attention_tables(case, seed)
    g = _gen(seed, 3)
    k = torch.empty((n_pages, P, G, DIM), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    v = torch.empty((n_pages, P, G, DIM), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    q = torch.empty((B, H, DIM), dtype=torch.bfloat16, device="cuda").normal_(0.0, 1.5, generator=g)
    refs = torch.zeros(n_pages, dtype=torch.int32)
    refs.index_add_(0, tables[tables >= 0], torch.ones(int((tables >= 0).sum()), dtype=torch.int32))
    return {"case": case, "q": q, "k": k, "v": v, "lens": lens.cuda(), "tables": tables.cuda(), "refs": refs.cuda(), "longest": int(lens.max()),
            "starts": _ints(list(range(0, B + 1, m))), "shared": _ints([shared] * (B // m)), "shared_most": shared,
            "out": torch.zeros((B, H, DIM), dtype=TYPES[case["out"]], device="cuda")}


def _pool(case, seed, tables, lens):
    """A pool of `arrays` caches (keys and values of the layers) under the given tables."""
    shape = (case["arrays"], case["pages"], case["page"], case["kv_heads"] * DIM)
    data = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=_gen(seed, 4))
    refs = torch.zeros(case["pages"], dtype=torch.int32)
    refs.index_add_(0, tables[tables >= 0], torch.ones(int((tables >= 0).sum()), dtype=torch.int32))
    return {"case": case, "data": data, "tables": tables.cuda(), "lens": lens.int().cuda(), "refs": refs.cuda()}


def prepare_fork(case, seed):
    """Sources with `length` positions each, and the samples of an earlier turn in the places of the new ones."""
    P, n, m, length = case["page"], case["sources"], case["members"], case["length"]
    held, most = -(-length // P), -(-(length + case["more"]) // P)
    h = _host(seed, 5)
    order = torch.randperm(case["pages"], generator=h).int()
    tables = torch.full((n + n * m, max(most, 3) + 1), -1, dtype=torch.int32)
    lens = torch.zeros(n + n * m, dtype=torch.int64)
    for s in range(n):
        tables[s, :held], lens[s] = order[s * held:(s + 1) * held], length
    at = n * held
    for d in range(n, n + n * m):
        old = int(torch.randint(0, 4, (), generator=h))
        tables[d, :old], lens[d] = order[at:at + old], old * P
        at += old
    st = _pool(case, seed, tables, lens)
    src = [s for s in range(n) for _ in range(m)]
    return {**st, "src": _ints(src), "dst": _ints(list(range(n, n + n * m))), "more": _ints([case["more"]] * (n * m)), "most": case["more"]}


def prepare_compact(case, seed):
    P, used, n = case["page"], case["used"], case["sequences"]
    h = _host(seed, 6)
    order = torch.randperm(case["pages"], generator=h)[:used].int()
    cuts = torch.arange(n + 1) * used // n
    held = cuts[1:] - cuts[:-1]
    tables = torch.full((n, int(held.max()) + 3), -1, dtype=torch.int32)
    lens = torch.zeros(n, dtype=torch.int64)
    for s in range(n):
        k = int(held[s])
        tables[s, :k] = order[int(cuts[s]):int(cuts[s + 1])]
        lens[s] = k * P - (int(torch.randint(0, P, (), generator=h)) if k else 0)
    st = _pool(case, seed, tables, lens)
    return {**st, "before": {n: st[n].clone() for n in ("tables", "lens", "refs")}}


def work(case):
    if case["path"] == "logprobs":
        n = case["rows"] * case["slices"] * case["cols"]
        outs = case["rows"] * (8 + (4 if case["entropy"] else 0) + 8 * case["top"])
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + outs, "flops": 4 * n}
    if case["path"] == "attention":
        H, G = HEADS[case["heads"]]
        B, m = case["batch"], case["members"]
        groups, mean = B // m, (1 + case["own_most"]) / 2
        mine = groups * case["own_most"] + (B - groups) * mean          # own positions, a group's longest member and the mean of the others
        return {"bytes": 4 * G * DIM * (groups * case["shared"] + mine) + (4 if case["out"] == "bf16" else 6) * B * H * DIM, "flops": 4 * H * DIM * (B * case["shared"] + mine)}
    row = 2 * case["kv_heads"] * DIM * case["arrays"]
    if case["path"] == "fork":
        n = case["sources"] * case["members"]
        return {"bytes": 2 * n * (case["length"] % case["page"]) * row + 4 * n * 16, "flops": 0}
    moves = case["used"] * (1 - case["used"] / case["pages"])
    return {"bytes": 2 * moves * case["page"] * row + 8 * case["pages"], "flops": 0}


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"logprobs": run_logprobs, "attention": run_attention, "fork": run_fork, "compact": run_compact}[state["case"]["path"]](state)


_handle = {}


def _device():
    """The program's one library handle, on a stream that torch can use too."""
    if not _handle:
        import tang_b200 as tb

        _handle["stream"] = torch.cuda.Stream()
        _handle["dev"] = tb.QuantComputeDevice(0, _handle["stream"].cuda_stream)
    return _handle["dev"]


def _buf(t):
    """A torch tensor's memory as the library sees it."""
    import tang_b200 as tb

    if t is None:
        return None
    return tb.Buffer(_device(), t.data_ptr(), t.numel(), {torch.bfloat16: tb.BF16, torch.float32: tb.F32, torch.int32: tb.I32}[t.dtype], owns=False)


def run_logprobs(state):
    case, out = state["case"], state["out"]
    S, R, C, top = case["slices"], case["rows"], case["cols"], case["top"]
    if own:
        if "own" not in state:
            import tang_b200 as tb

            state["own"] = (_buf(state["x"]), _buf(state["tokens"]), tb.TokenLogprobs(**{n: _buf(t) for n, t in out.items()}))
        x, tokens, into = state["own"]
        _device().token_logprobs(x, R, C, tokens, top=top, slices=S, entropy=case["entropy"], out=into)
        return out
    x = state["x"].float().permute(1, 0, 2).reshape(R, S * C)
    m = x.max(1, keepdim=True).values
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True)
    log_s = torch.log(s)
    got = {"logprobs": (x.gather(1, state["tokens"].long()[:, None]) - m - log_s)[:, 0], "entropy": None, "top_ids": None, "top_logprobs": None}
    if case["entropy"]:
        got["entropy"] = (log_s - (torch.where(e > 0, x - m, 0.0) * e).sum(1, keepdim=True) / s)[:, 0]
    if top:
        # one whole number a token, larger for a larger logit and, among equals, for a lower index
        bits = x.view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 31) + torch.arange(S * C - 1, -1, -1, device="cuda")
        ids = key.topk(top, 1).indices
        got["top_ids"], got["top_logprobs"] = ids.int(), x.gather(1, ids) - m - log_s
    return got


def _page_buffers(state):
    return {n: _buf(state[n]) for n in ("refs", "tables", "lens")}


def run_attention(state):
    case = state["case"]
    H, G = HEADS[case["heads"]]
    B, P = case["batch"], case["page"]
    if own:
        if "own" not in state:
            import tang_b200 as tb

            n_pages, (seqs, ld) = state["k"].shape[0], state["tables"].shape
            pool = tb.PagePool(_device(), n_pages, P, seqs, ld, **_page_buffers(state))
            state["own"] = (pool, *(_buf(state[n]) for n in ("q", "k", "v", "starts", "shared", "out")))
        pool, q, k, v, starts, shared, out = state["own"]
        groups = {"group_starts": starts, "shared": shared, "n_groups": B // case["members"], "max_shared": state["shared_most"]} if state["shared_most"] else {}
        _device().gqa_decode_paged(q, k, v, pool, B, H, G, DIM, state["longest"], out=out, **groups)
        return state["out"]
    pos = torch.arange(state["longest"], device="cuda")
    seen = pos[None] < state["lens"][:, None]
    rows = state["tables"][:, pos // P].long() * P + pos % P
    rows = torch.where(seen, rows, 0)
    k = state["k"].view(-1, G, DIM)[rows].float()
    score = torch.einsum("bghd,bjgd->bghj", state["q"].float().view(B, G, H // G, DIM), k) * DIM ** -0.5
    del k
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(score - score.max(-1, keepdim=True).values)
    del score
    v = state["v"].view(-1, G, DIM)[rows].float()
    o = torch.einsum("bghj,bjgd->bghd", e, v) / e.sum(-1, keepdim=True)
    return o.reshape(B, H, DIM).to(TYPES[case["out"]])


def _held(state, seqs):
    P, ld = state["case"]["page"], state["tables"].shape[1]
    return torch.arange(ld, device="cuda") < ((state["lens"][seqs].long() + P - 1) // P)[:, None]


def run_fork(state):
    case = state["case"]
    P, n, src, dst = case["page"], state["dst"].numel(), state["src"], state["dst"]
    if own:
        if "own" not in state:
            import tang_b200 as tb

            seqs, ld = state["tables"].shape
            pool = tb.PagePool(_device(), case["pages"], P, seqs, ld, arrays=[_buf(a) for a in state["data"]], **_page_buffers(state))
            state["own"] = (pool, _buf(src), _buf(dst), _buf(state["more"]))
        pool, s, d, more = state["own"]
        pool.free(d, n)
        pool.fork(s, d, n)
        pool.extend(d, n, more)
        return {k: state[k] for k in ("data", "tables", "lens", "refs")}
    tables, lens, refs = state["tables"], state["lens"], state["refs"]
    # the places of the new samples give back what they held
    held = _held(state, dst)
    old = tables[dst]
    refs.index_add_(0, old[held], torch.full_like(old[held], -1))
    tables[dst] = torch.where(held, -1, old)
    # a sample holds its source's pages
    held, pages = _held(state, src), tables[src]
    refs.index_add_(0, pages[held], torch.ones_like(pages[held]))
    tables[dst] = torch.where(held, pages, tables[dst])
    lens[dst] = lens[src]
    # room for the next tokens: lowest free pages first, in the order of the samples; a shared, partly filled page is copied
    L, c = lens[dst].long(), state["more"].long()
    last = tables[dst, ((L - 1) // P).clamp(min=0)].long()
    part = (L % P != 0) & (c > 0)
    before = ((last[:, None] == last[None]) & part[None]).tril(-1).sum(1)
    cow = part & (refs[last.clamp(min=0)] - before > 1)
    need = cow + (L + c + P - 1) // P - (L + P - 1) // P
    free = torch.argsort((refs != 0).int(), stable=True)
    first = need.cumsum(0) - need
    j = torch.arange((state["most"] + P - 1) // P + 1, device="cuda")
    mine = j[None] < need[:, None]
    page = free[(first[:, None] + j).clamp(max=free.numel() - 1)].int()
    at = ((L + P - 1) // P - cow.long())[:, None] + j
    who = dst[:, None].expand_as(at)
    refs.index_add_(0, last[cow], torch.full_like(last[cow], -1, dtype=torch.int32))
    refs[page[mine].long()] = 1
    tables[who[mine].long(), at[mine]] = page[mine]
    lens[dst] = (L + c).int()
    r = torch.arange(P, device="cuda")
    copied = r < (L % P)[cow][:, None]
    flat = state["data"].view(case["arrays"], -1, case["kv_heads"] * DIM)
    flat[:, (page[:, 0].long()[cow][:, None] * P + r)[copied]] = flat[:, (last[cow][:, None] * P + r)[copied]]
    return {k: state[k] for k in ("data", "tables", "lens", "refs")}


def run_compact(state):
    case, before = state["case"], state["before"]
    if own:
        if "own" not in state:
            import tang_b200 as tb

            seqs, ld = state["tables"].shape
            state["own"] = tb.PagePool(_device(), case["pages"], case["page"], seqs, ld, arrays=[_buf(a) for a in state["data"]], **_page_buffers(state))
        with torch.cuda.stream(_handle["stream"]):     # the pool as it was found; the pages that moved still hold their rows
            for n, t in before.items():
                state[n].copy_(t)
        state["own"].compact()
        return {k: state[k] for k in ("data", "tables", "lens", "refs")}
    for n, t in before.items():
        state[n].copy_(t)
    used = state["refs"] > 0
    ids, n = torch.arange(case["pages"], device="cuda"), used.sum()
    dst, src = torch.nonzero(~used & (ids < n))[:, 0], torch.nonzero(used & (ids >= n))[:, 0]
    state["data"][:, dst] = state["data"][:, src]
    ids[src] = dst
    state["tables"].copy_(torch.where(state["tables"] >= 0, ids[state["tables"].clamp(min=0).long()].int(), state["tables"]))
    state["refs"][dst] = state["refs"][src]
    state["refs"][src] = 0
    return {k: state[k] for k in ("data", "tables", "lens", "refs")}


# ---------------------------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    if case["path"] == "logprobs":
        st = prepare_logprobs(case, seed)
        R = case["rows"]
        got = {"logprobs": [], "entropy": [], "top_ids": None, "top_logprobs": []}
        step = max(1, (1 << 27) // (case["slices"] * case["cols"]))
        for r in range(0, R, step):
            x = torch.cat([s[r:r + step].double() for s in st["x"]], 1)
            lse = torch.logsumexp(x, 1)
            p = torch.exp(x - lse[:, None])
            got["logprobs"].append(x[torch.arange(x.shape[0]), st["tokens"][r:r + step].long()] - lse)
            got["entropy"].append(-torch.special.xlogy(p, p).sum(1))
            if case["top"]:
                got["top_logprobs"].append(x.topk(case["top"], 1).values - lse[:, None])
        return {"logprobs": torch.cat(got["logprobs"]), "entropy": torch.cat(got["entropy"]) if case["entropy"] else None, "top_ids": None,
                "top_logprobs": torch.cat(got["top_logprobs"]) if case["top"] else None}
    if case["path"] == "attention":
        st = prepare_attention(case, seed)
        H, G = HEADS[case["heads"]]
        out = torch.zeros((case["batch"], H, DIM), dtype=torch.float64, device="cuda")
        lens = st["lens"].tolist()
        for b, n in enumerate(lens):
            pages = st["tables"][b, :-(-n // case["page"])].long()
            k = st["k"][pages].reshape(-1, G, DIM)[:n].double().repeat_interleave(H // G, 1)
            v = st["v"][pages].reshape(-1, G, DIM)[:n].double().repeat_interleave(H // G, 1)
            s = (k * st["q"][b].double()[None]).sum(2) / math.sqrt(DIM)
            out[b] = (torch.softmax(s, 0)[:, :, None] * v).sum(0)
        return out
    st = prepare(case, seed)
    return (exact_fork if case["path"] == "fork" else exact_compact)(case, st)


def _moved(case, st, tables, lens, refs, moves):
    """The pool's state with the rows of `moves`, (from page, to page, rows), copied one after the other."""
    data = st["data"]
    for a, b, n in moves:
        data[:, b, :n] = data[:, a, :n]
    return {"data": data.double(), "tables": torch.tensor(tables), "lens": torch.tensor(lens), "refs": torch.tensor(refs)}


def exact_fork(case, st):
    """The three calls as their definition has them: sequence by sequence, page by page."""
    P = case["page"]
    tables, lens, refs = (st[n].tolist() for n in ("tables", "lens", "refs"))
    moves = []
    for d in st["dst"].tolist():
        for i in range(-(-lens[d] // P)):
            refs[tables[d][i]] -= 1
            tables[d][i] = -1
        lens[d] = 0
    for s, d in zip(st["src"].tolist(), st["dst"].tolist()):
        for i in range(-(-lens[s] // P)):
            tables[d][i] = tables[s][i]
            refs[tables[s][i]] += 1
        lens[d] = lens[s]
    free = [p for p in range(case["pages"]) if refs[p] == 0]
    for d, c in zip(st["dst"].tolist(), st["more"].tolist()):
        i = lens[d] // P
        if lens[d] % P and c and refs[tables[d][i]] > 1:
            page = free.pop(0)
            moves.append((tables[d][i], page, lens[d] % P))
            refs[tables[d][i]] -= 1
            tables[d][i], refs[page] = page, 1
        for i in range(-(-lens[d] // P), -(-(lens[d] + c) // P)):
            tables[d][i] = free.pop(0)
            refs[tables[d][i]] = 1
        lens[d] += c
    return _moved(case, st, tables, lens, refs, moves)


def exact_compact(case, st):
    tables, lens, refs = (st[n].tolist() for n in ("tables", "lens", "refs"))
    used = sum(r > 0 for r in refs)
    to = dict(zip([p for p in range(used, case["pages"]) if refs[p]], [p for p in range(used) if not refs[p]]))
    for a, b in to.items():
        refs[b], refs[a] = refs[a], 0
    tables = [[to.get(p, p) for p in t] for t in tables]
    return _moved(case, st, tables, lens, refs, [(a, b, case["page"]) for a, b in to.items()])
