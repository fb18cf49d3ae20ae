"""The operators that a serving program runs beside the decode GEMMs, as cases to be timed.

  attention  stride_amd.harness.window_attention: grouped-query attention of new rows
             over a paged bf16 KV cache. Row (slot, position p) sees position t <= p if
             p - t < window (or the window is 0: all of them) or t < sinks. fp32 queries
             in, bf16 x tiles out.
  pages      stride_amd.kv_pool.KvPool: pages of the cache shared between sequences with
             counted references. A free page is taken lowest number first.
               fork     a sequence goes on in several branches: whole pages are shared, the
                        part page is copied
               compact  a sequence keeps a list of its positions, which move together; the
                        pages behind them are released
  logits     stride_amd.logits.process: penalties for tokens that a sequence has, biases,
             a grammar's mask, then the greedy choice, which the counts take up.

Shapes are those of the repository's benchmark and tests (hidden 2048 as 32 query and 8 KV
heads of 64, 16 layers, vocabulary 128256, 16-token KV pages, 16 x 16 tiles) and head_dim
128, other group sizes, pages and vocabularies.
"""
import math

import torch

own = False  # True: run() calls this repository's operators instead of the plain forms

DEV = "cuda:0"
PROMPT_FLAG = -(1 << 31)  # counts: the token is in the prompt (the sign bit)


# ---------------------------------------------------------------------------
# The cases.

def listed():
    def attn(name, seqs, rows, ctx, window, sinks, head_dim=64, n_kv=8, n_q=4, page=16, ragged=True):
        return dict(name=name, op="attention", seqs=seqs, rows=rows, ctx=ctx, window=window, sinks=sinks,
                    head_dim=head_dim, n_kv=n_kv, n_q=n_q, page=page, ragged=ragged)

    def pages(name, op, seqs, ctx, layers=16, n_kv=8, head_dim=64, page=16, **more):
        return dict(name=name, op=op, seqs=seqs, ctx=ctx, layers=layers, n_kv=n_kv, head_dim=head_dim, page=page, **more)

    def logits(name, rows, vocab, written, mask=True, history=512):
        return dict(name=name, op="logits", rows=rows, vocab=vocab, written=written, mask=mask, history=history)

    return [
        # One user's next token, a thousand positions in: launches and latency.
        attn("attention_decode_1", 1, 1, 1000, 0, 0, ragged=False),
        # A serving batch of streams that run without end: a window and the first four tokens.
        attn("attention_decode_window_128", 128, 1, 4096, 1024, 4),
        # A few sequences over long documents: the length is what there is to split.
        attn("attention_decode_long_4", 4, 1, 32768, 0, 0, head_dim=128, n_q=8, page=64, ragged=False),
        # A chunk of one long prompt, each row behind a window.
        attn("attention_prefill_window_2048", 1, 2048, 5000, 512, 4, ragged=False),
        # Odd chunks of three prompts that see all before them.
        attn("attention_prefill_999", 3, 333, 3001, 0, 0, head_dim=128),
        # Best-of-four sampling: 16 prompts of about 300 tokens, each branched in four again.
        pages("pages_fork_16x4", "fork", 16, 300, branches=4),
        # Speculative decoding: of 16 tree tokens behind about 1000, the accepted ones move up.
        pages("pages_accept_64", "compact", 64, 1000, tail=16, keep=4),
        # Eviction: of 4096 positions the first four and 2044 chosen ones stay.
        pages("pages_evict_8", "compact", 8, 4, tail=4092, keep=2044),
        # One user, one constrained step.
        logits("logits_1", 1, 128256, False),
        # The serving batch, with the processed logits written for a sampler.
        logits("logits_128_written", 128, 128256, True),
        # An odd batch over an odd vocabulary, greedy.
        logits("logits_33_odd", 33, 50001, False, history=2000),
    ]


def _span(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """One more case of these ranges."""
    op = rng.choice(["attention", "attention", "attention", "fork", "compact", "logits", "logits"])
    if op == "attention":
        head_dim, n_kv, n_q = rng.choice([32, 64, 64, 128]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 7, 8, 16])
        if n_kv * n_q > 32:
            n_q = 32 // n_kv
        if rng.random() < 0.6:  # decode
            seqs, rows = _span(rng, 1, 160), 1
            ctx = _span(rng, 1, max(64, min(40000, 2 ** 29 // (seqs * n_kv * head_dim * 4))))
        else:
            seqs = _span(rng, 1, 6)
            rows = _span(rng, 2, 1000 // seqs)
            ctx = rows + _span(rng, 1, 2000)
        window = rng.choice([0, _span(rng, 1, 4096)])
        return dict(op=op, seqs=seqs, rows=rows, ctx=ctx, window=window, sinks=rng.choice([0, 4, _span(rng, 1, 300)]) if window else 0,
                    head_dim=head_dim, n_kv=n_kv, n_q=n_q, page=rng.choice([16, 16, 32, 64, 128]), ragged=rng.random() < 0.7)
    if op == "logits":
        rows = _span(rng, 1, 128)
        return dict(op=op, rows=rows, vocab=_span(rng, 500, 128256), written=rng.random() < 0.5, mask=rng.random() < 0.7,
                    history=_span(rng, 1, 3000))
    shape = dict(layers=rng.choice([4, 8, 16]), n_kv=rng.choice([2, 4, 8]), head_dim=rng.choice([32, 64, 128]), page=rng.choice([16, 32, 64]))
    if op == "fork":
        return dict(op=op, seqs=_span(rng, 1, 24), ctx=_span(rng, 1, 900), branches=rng.randint(1, 5), **shape)
    tail = _span(rng, 2, 650)
    return dict(op=op, seqs=_span(rng, 1, 12), ctx=_span(rng, 1, 500), tail=tail, keep=rng.randint(1, tail), **shape)


# ---------------------------------------------------------------------------
# Inputs.

def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + salt)


def _rand(gen, *shape):
    return torch.rand(*shape, generator=gen, device=DEV)


def _lengths(case, gen, n, least):
    """Context lengths: all `ctx`, or spread from an eighth of it upwards."""
    if not case.get("ragged", True):
        return torch.full((n,), case["ctx"], dtype=torch.int64, device=DEV)
    u = _rand(gen, n)
    return (case["ctx"] * (0.125 + 0.875 * u)).long().clamp(min=least)


def prepare(case, seed):
    return {"attention": _prepare_attention, "fork": _prepare_pages, "compact": _prepare_pages,
            "logits": _prepare_logits}[case["op"]](case, seed)


def _prepare_attention(c, seed):
    gen = _gen(seed, 1)
    n_kv, n_q, d, page, seqs, r = c["n_kv"], c["n_q"], c["head_dim"], c["page"], c["seqs"], c["rows"]
    layers, rows = 2, c["seqs"] * c["rows"]
    max_blocks = -(-c["ctx"] // page)
    nb = seqs * max_blocks
    table = torch.randperm(nb, generator=gen, device=DEV).reshape(seqs, max_blocks).to(torch.int32)
    arena = torch.empty((nb, layers, 2, n_kv, page, d), dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    q = torch.empty((rows, n_kv * n_q * d), device=DEV).normal_(generator=gen) * 1.25
    last = _lengths(c, gen, seqs, r) - 1
    pos = (last[:, None] + torch.arange(r, device=DEV)[None] - (r - 1)).reshape(-1).to(torch.int32)
    slot = torch.arange(seqs, device=DEV).repeat_interleave(r).to(torch.int32)
    s = dict(case=c, arena=arena, table=table, q=q, pos=pos, slot=slot, scale=d ** -0.5)
    if own:
        from stride_amd import harness

        s["kv"] = harness.PagedKv.over(arena.view(torch.int16).reshape(-1), table, n_kv, d, layers, page)
        s["out"] = torch.zeros(((rows + 15) // 16, n_kv * n_q * d // 16, 16, 16), dtype=torch.int16, device=DEV)
        s["scratch"] = harness.window_attention_scratch(rows, n_kv, n_q, d, c["window"], c["sinks"], -(-c["ctx"] // 64), DEV)
    return s


def _prepare_pages(c, seed):
    gen = _gen(seed, 2)
    n, page, fork = c["seqs"], c["page"], c["op"] == "fork"
    i32 = dict(dtype=torch.int32, device=DEV)
    most = c["ctx"] if fork else c["ctx"] + c["tail"]
    max_blocks = -(-most // page)
    slots = n * (1 + c["branches"]) if fork else n
    pages = n * max_blocks + (n * c["branches"] if fork else 0) + 8  # eight are left over
    arena = torch.randint(-32768, 32768, (pages, c["layers"], 2, c["n_kv"], page, c["head_dim"]), generator=gen,
                          dtype=torch.int16, device=DEV)
    order = torch.randperm(pages, generator=gen, device=DEV)
    table = torch.full((slots, max_blocks), -1, **i32)
    if fork:
        length = _lengths(c, gen, n, 1)
        held = -(-length // page)
    else:
        length = torch.full((n,), c["ctx"], dtype=torch.int64, device=DEV)
        held = torch.full((n,), max_blocks, dtype=torch.int64, device=DEV)
    trunk = order[: n * max_blocks].reshape(n, max_blocks)
    table[:n] = torch.where(torch.arange(max_blocks, device=DEV)[None] < held[:, None], trunk, -1).to(torch.int32)
    refs = torch.zeros(pages, **i32)
    refs.index_add_(0, table[:n].reshape(-1).clamp(min=0).long(), (table[:n] >= 0).reshape(-1).to(torch.int32))
    s = dict(case=c, arena=arena, table=table, refs=refs)
    if fork:
        s["src"] = torch.arange(n, device=DEV).repeat_interleave(c["branches"]).to(torch.int32)
        s["dst"] = torch.arange(n, slots, **i32)
        s["length"] = length.repeat_interleave(c["branches"]).to(torch.int32)
        s["lo"], s["hi"] = torch.zeros_like(s["dst"]), torch.full_like(s["dst"], max_blocks)
    else:
        s["slots"] = torch.randperm(n, generator=gen, device=DEV).to(torch.int32)
        s["first"] = length.to(torch.int32)
        # the kept positions: a random choice of the tail, ascending
        chosen = torch.argsort(_rand(gen, n, c["tail"]), dim=1)[:, : c["keep"]].sort(dim=1).values
        s["keep"] = (chosen + c["ctx"]).to(torch.int32)
        s["count"] = (1 + (_rand(gen, n) * 0.25 + 0.75) * (c["keep"] - 1)).long().to(torch.int32)
        s["lo"] = ((s["first"] + s["count"] + page - 1) // page).to(torch.int32)
        s["hi"] = torch.full_like(s["lo"], max_blocks)
    if own:
        from stride_amd import kv_pool

        s["pool"] = kv_pool.KvPool(arena, table, refs, c["n_kv"], c["head_dim"], c["layers"], page)
    return s


def _pack_bits(flags):
    """[n][vocab] truth values -> [n][ceil(vocab / 32)] int32 words, bit t % 32 of word t // 32."""
    n, v = flags.shape
    words = -(-v // 32)
    f = torch.zeros((n, words * 32), dtype=torch.int64, device=flags.device)
    f[:, :v] = flags
    w = (f.reshape(n, words, 32) << torch.arange(32, device=flags.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _prepare_logits(c, seed):
    gen = _gen(seed, 3)
    rows, vocab = c["rows"], c["vocab"]
    T, rt = -(-rows // 16), -(-vocab // 16)
    logits = torch.zeros((rt, T, 16, 16), device=DEV)
    logits.normal_(generator=gen).mul_(3.0)
    slot = torch.randperm(rows, generator=gen, device=DEV).to(torch.int32)
    # what each sequence holds: a prompt, and a quarter as many tokens that were generated, some of them often
    prompt = (vocab * _rand(gen, rows, c["history"]) ** 3).long().clamp(max=vocab - 1)
    made = (vocab * _rand(gen, rows, max(1, c["history"] // 4)) ** 4).long().clamp(max=vocab - 1)
    counts = torch.zeros((rows, vocab), dtype=torch.int32, device=DEV)
    counts.scatter_add_(1, made, torch.ones_like(made, dtype=torch.int32))
    flag = torch.zeros((rows, vocab), dtype=torch.bool, device=DEV).scatter_(1, prompt, True)
    counts = torch.where(flag, counts | PROMPT_FLAG, counts)
    seen = _pack_bits(counts != 0)
    penalties = torch.stack([1.0 + 0.3 * _rand(gen, rows), _rand(gen, rows), 0.5 * _rand(gen, rows)], 1)
    # up to 64 biases a row, tokens ascending
    per = torch.randint(0, min(64, vocab) + 1, (rows,), generator=gen, device=DEV)
    choice = torch.argsort(_rand(gen, rows, min(vocab, 4096)), dim=1)[:, : min(64, vocab)] * (vocab // min(vocab, 4096))
    have = torch.arange(choice.shape[1], device=DEV)[None] < per[:, None]
    choice = torch.where(have, choice, vocab).sort(dim=1).values
    bias_rows = torch.arange(rows, device=DEV)[:, None].expand_as(choice)[have.sort(dim=1, descending=True).values]
    tokens = choice[choice < vocab]
    values = 4.0 * _rand(gen, tokens.numel()) - 2.0
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), per.cumsum(0)]).to(torch.int32)
    s = dict(case=c, logits=logits, slot=slot, counts=counts, seen=seen, penalties=penalties, offsets=offsets,
             tokens=tokens.to(torch.int32), values=values, bias_rows=bias_rows, mask=None, mask_row=None)
    if c["mask"]:  # four states of a grammar, from a few tokens to nearly all; some rows have none
        dense = torch.tensor([0.001, 0.1, 0.5, 0.99], device=DEV)
        allowed = _rand(gen, 4, vocab) < dense[:, None]
        allowed[:, vocab // 3] = True
        s["mask"] = _pack_bits(allowed)
        s["mask_row"] = torch.randint(-1, 4, (rows,), generator=gen, device=DEV).to(torch.int32)
    if own:
        from stride_amd import logits as lg

        s["state"] = lg.TokenCounts(counts, seen)
        s["out"] = torch.zeros_like(logits) if c["written"] else None
        s["best"] = torch.empty((rows, 2), dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------
# One pass.

def run(s):
    return {"attention": _attention, "fork": _fork, "compact": _compact, "logits": _logits}[s["case"]["op"]](s)


def _tiles(a):
    """[rows][cols] -> [ceil(rows / 16)][cols / 16][16][16], lanes past the last row zero."""
    rows, cols = a.shape
    t = -(-rows // 16)
    out = torch.zeros((t * 16, cols), dtype=a.dtype, device=a.device)
    out[:rows] = a
    return out.reshape(t, 16, cols // 16, 16).permute(0, 2, 1, 3).contiguous()


def _attention(s):
    c = s["case"]
    n_kv, n_q, d, seqs, r = c["n_kv"], c["n_q"], c["head_dim"], c["seqs"], c["rows"]
    if own:
        from stride_amd import harness

        out = harness.window_attention(s["q"], s["kv"], s["slot"], s["pos"], n_kv, n_q, d, s["scale"], c["window"],
                                       c["sinks"], layer=1, max_pages=-(-c["ctx"] // 64), out_tiles=s["out"],
                                       scratch=s["scratch"], runs=r)
        return out.view(torch.bfloat16)
    blocks = s["table"].long()

    def dense(which):  # [seqs][n_kv][ctx][d]
        a = s["arena"][:, 1, which][blocks]
        return a.permute(0, 2, 1, 3, 4).reshape(seqs, n_kv, -1, d)[:, :, : c["ctx"]].float()

    k, v = dense(0), dense(1)
    q = s["q"].reshape(seqs, r, n_kv, n_q, d).permute(0, 2, 1, 3, 4).reshape(seqs, n_kv, r * n_q, d)
    score = torch.matmul(q * s["scale"], k.transpose(2, 3).contiguous())
    t, p = torch.arange(c["ctx"], device=DEV), s["pos"].long().reshape(seqs, r, 1)
    see = t <= p
    if c["window"] > 0:
        see = see & ((p - t < c["window"]) | (t < c["sinks"]))
    see = see[:, None, :, None, :].expand(seqs, 1, r, n_q, c["ctx"]).reshape(seqs, 1, r * n_q, c["ctx"])
    score = torch.where(see, score, -math.inf)
    w = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(w, v) / w.sum(-1, keepdim=True)
    o = o.reshape(seqs, n_kv, r, n_q, d).permute(0, 2, 1, 3, 4).reshape(seqs * r, n_kv * n_q * d)
    return _tiles(o.to(torch.bfloat16))


def _take(refs, want):
    """Free pages, lowest number first, for the entries of `want` that are true, in order."""
    free = torch.sort((refs != 0).to(torch.int8), stable=True).indices
    rank = torch.cumsum(want.reshape(-1).long(), 0) - 1
    return free[rank.clamp(min=0)].reshape(want.shape)


def _release(s, slots, sel):
    """Gives back the pages that the entries `sel` of the slots' table rows hold."""
    rows = s["table"][slots]
    sel = sel & (rows >= 0)
    s["refs"].index_add_(0, rows.reshape(-1).clamp(min=0).long(), -sel.reshape(-1).to(torch.int32))
    s["table"][slots] = torch.where(sel, -1, rows)


def _hold(s, slots, pages, sel):
    s["refs"].index_add_(0, torch.where(sel, pages, 0).reshape(-1).long(), sel.reshape(-1).to(torch.int32))
    s["table"][slots] = torch.where(sel, pages.to(torch.int32), s["table"][slots])


def _cache(s):
    return {"arena": s["arena"], "table": s["table"], "refs": s["refs"]}


def _fork(s):
    """The branches of the last round are given up, and every trunk is branched again."""
    if own:
        s["pool"].release(s["dst"], s["lo"], s["hi"])
        s["pool"].fork(s["src"], s["dst"], s["length"])
        return _cache(s)
    page, src, dst, length = s["case"]["page"], s["src"].long(), s["dst"].long(), s["length"].long()
    p = torch.arange(s["table"].shape[1], device=DEV)[None]
    _release(s, dst, p >= 0)
    rows = s["table"][src]
    full, part = (length // page)[:, None], length % page
    split = (p == full) & (part[:, None] > 0) & (rows >= 0)
    new = _take(s["refs"], split)
    _hold(s, dst, rows, (p < full) & (rows >= 0))
    _hold(s, dst, new, split)
    at = full.clamp(max=p.shape[1] - 1)
    a, b = rows.gather(1, at)[:, 0].long(), new.gather(1, at)[:, 0]
    b = torch.where(split.gather(1, at)[:, 0], b, a)  # a whole page has nothing to copy: onto itself
    s["arena"][b] = torch.where((torch.arange(page, device=DEV) < part[:, None])[:, None, None, None, :, None],
                                s["arena"][a], s["arena"][b])
    return _cache(s)


def _compact(s):
    """The kept positions move together, the pages behind go, and pages for the next ones come.
    (No page is shared here.)"""
    if own:
        s["pool"].compact(s["slots"], s["first"], s["count"], s["keep"])
        s["pool"].reserve(s["slots"], s["lo"], s["hi"])
        return _cache(s)
    page, slots, first, count = s["case"]["page"], s["slots"].long(), s["first"].long(), s["count"].long()
    rows = s["table"][slots].long()
    i = torch.minimum(torch.arange(s["keep"].shape[1], device=DEV)[None], count[:, None] - 1)  # past the last: it again
    old, new = s["keep"].long().gather(1, i), first[:, None] + i
    moved = s["arena"][rows.gather(1, old // page), :, :, :, old % page]
    s["arena"][rows.gather(1, new // page), :, :, :, new % page] = moved
    p = torch.arange(rows.shape[1], device=DEV)[None]
    _release(s, slots, p >= (first + count + page - 1)[:, None] // page)
    want = (p >= s["lo"][:, None]) & (p < s["hi"][:, None]) & (s["table"][slots] < 0)
    _hold(s, slots, _take(s["refs"], want), want)
    return _cache(s)


def _logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    if own:
        from stride_amd import logits as lg

        bias = (s["offsets"], s["tokens"], s["values"])
        best = lg.process(s["logits"], rows, vocab, counts=s["state"], row_slot=s["slot"], penalties=s["penalties"], bias=bias,
                          mask=s["mask"], mask_row=s["mask_row"], out=s["out"], best=s["best"])
        s["state"].record(s["slot"], best[:, 1])
        return {"logits": s["out"], "value": best.view(torch.float32)[:, 0], "index": best[:, 1], "counts": s["counts"],
                "seen": s["seen"]}
    slot = s["slot"].long()
    l = s["logits"].permute(1, 3, 0, 2).reshape(-1, s["logits"].shape[0] * 16)[:rows, :vocab]
    word = s["counts"][slot]
    n = (word & 0x7FFFFFFF).float()
    rep, pres, freq = (s["penalties"][:, k : k + 1] for k in range(3))
    l = torch.where(word != 0, torch.where(l > 0, l / rep, l * rep), l)
    l = l - freq * n
    l = torch.where(n > 0, l - pres, l)
    l = l.index_put((s["bias_rows"], s["tokens"].long()), s["values"], accumulate=True)
    if s["mask"] is not None:
        t = torch.arange(vocab, device=DEV)
        allowed = ((s["mask"][:, t // 32] >> (t % 32)[None]) & 1) != 0
        row = s["mask_row"].long()
        l = torch.where(allowed[row.clamp(min=0)] | (row < 0)[:, None], l, -math.inf)
    value = l.amax(1)
    t = torch.arange(vocab, device=DEV)[None]
    index = torch.where((l == value[:, None]) & (value > -math.inf)[:, None], t, vocab).amin(1)
    index = torch.where(index == vocab, -1, index)
    at, one = index.clamp(min=0), (index >= 0)
    s["counts"][slot, at] += one.to(torch.int32)
    s["seen"][slot, at // 32] |= torch.where(one, torch.ones_like(at) << (at % 32), 0).to(torch.int32)
    out = None
    if c["written"]:
        out = torch.zeros_like(s["logits"])
        wide = torch.zeros((out.shape[1] * 16, out.shape[0] * 16), device=DEV)
        wide[:rows, :vocab] = l
        out = wide.reshape(out.shape[1], 16, out.shape[0], 16).permute(2, 0, 3, 1).contiguous()
    return {"logits": out, "value": value, "index": index.to(torch.int32), "counts": s["counts"], "seen": s["seen"]}


# ---------------------------------------------------------------------------
# What a pass cannot do without.

def _visible(c, p):
    """Positions that a row at p sees."""
    if c["window"] <= 0 or p < c["window"]:
        return p + 1
    return c["window"] + min(c["sinks"], p + 1 - c["window"])


def work(case):
    c = case
    if c["op"] == "attention":
        heads, d = c["n_kv"] * c["n_q"], c["head_dim"]
        # ragged contexts: from an eighth of ctx to all of it, the middle stands for the mean
        last = [c["ctx"] - 1] if not c["ragged"] else [int(c["ctx"] * (0.125 + 0.875 * (i + 0.5) / 8)) - 1 for i in range(8)]
        seen = read = 0.0
        for p in last:
            p = max(p, c["rows"] - 1)
            seen += sum(_visible(c, x) for x in range(p - c["rows"] + 1, p + 1)) / len(last)
            read += min(p + 1, _visible(c, p) + c["rows"] - 1) / len(last)
        rows = c["seqs"] * c["rows"]
        return {"bytes": 6.0 * rows * heads * d + 4.0 * c["seqs"] * read * c["n_kv"] * d, "flops": 4.0 * c["seqs"] * seen * heads * d}
    if c["op"] == "logits":
        values = c["rows"] * c["vocab"]
        return {"bytes": values * (4.0 + 4.0 * c["written"] + 0.125) + (4 * c["vocab"] / 8 if c["mask"] else 0), "flops": 2.0 * values}
    token = 4.0 * c["layers"] * c["n_kv"] * c["head_dim"]
    if c["op"] == "fork":
        n, mean = c["seqs"] * c["branches"], max(1.0, 0.5625 * c["ctx"])
        # part pages are half full at the mean; table entries and references of the shared ones
        return {"bytes": n * (2 * token * min(mean, c["page"] / 2) + 24.0 * mean / c["page"]), "flops": 0.0}
    moved = c["seqs"] * (1 + 0.875 * (c["keep"] - 1))
    return {"bytes": 2 * moved * token + 4 * moved, "flops": 0.0}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, row by row.

def exact(case, seed):
    if case["op"] == "attention":
        return _exact_attention(prepare(case, seed))
    if case["op"] == "logits":
        return _exact_logits(prepare(case, seed))
    return None  # pages are copied: their outputs are whole numbers


def _exact_attention(s):
    c = s["case"]
    d, n_q, page = c["head_dim"], c["n_q"], c["page"]
    pos, slot, table = s["pos"].tolist(), s["slot"].tolist(), s["table"].tolist()
    rows = len(pos)
    full = torch.zeros((-(-rows // 16) * 16, c["n_kv"], n_q, d), dtype=torch.float64, device=DEV)
    q = s["q"].double().reshape(rows, c["n_kv"], n_q, d)
    for sl in range(c["seqs"]):
        mine = [j for j in range(rows) if slot[j] == sl]
        longest = max(pos[j] for j in mine) + 1
        part = s["arena"][table[sl][: -(-longest // page)], 1].double()  # [page][2][n_kv][token][d]
        for g in range(c["n_kv"]):
            k, v = (part[:, w, g].reshape(-1, d) for w in (0, 1))
            for a in range(0, len(mine), 128):
                js = mine[a : a + 128]
                x = torch.einsum("jhd,td->jht", q[js, g], k) * s["scale"]
                away = torch.tensor([pos[j] for j in js], device=DEV)[:, None] - torch.arange(k.shape[0], device=DEV)
                hidden = away < 0
                if c["window"] > 0:
                    far = away >= c["window"]
                    far[:, : c["sinks"]] = False
                    hidden = hidden | far
                x = x.masked_fill(hidden[:, None, :], float("-inf"))
                w = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
                full[js, g] = torch.einsum("jht,td->jhd", w, v)
    full = full.reshape(full.shape[0] // 16, 16, -1, 16)
    return full.transpose(1, 2).contiguous()


def _exact_logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    out = torch.zeros_like(s["logits"], dtype=torch.float64)
    slot, off = s["slot"].tolist(), s["offsets"].tolist()
    values = torch.empty(rows, dtype=torch.float64, device=DEV)
    masks = [] if s["mask"] is None else s["mask_row"].tolist()
    for j in range(rows):
        l = s["logits"][:, j // 16, :, j % 16].reshape(-1)[:vocab].double()
        word = s["counts"][slot[j]].long()
        made = word % (1 << 31)
        rep, pres, freq = s["penalties"][j].double().tolist()
        known = word.ne(0)
        l = torch.where(known & (l > 0), l / rep, torch.where(known, l * rep, l)) - freq * made - pres * made.clamp(max=1)
        at = s["tokens"][off[j] : off[j + 1]].long()
        l[at] += s["values"][off[j] : off[j + 1]].double()
        if masks and masks[j] >= 0:
            words = s["mask"][masks[j]].long() % (1 << 32)
            bits = (words[:, None] // (2 ** torch.arange(32, device=DEV))) % 2
            l[bits.reshape(-1)[:vocab] == 0] = float("-inf")
        values[j] = l.max()
        if c["written"]:
            pad = torch.zeros(out.shape[0] * 16, dtype=torch.float64, device=DEV)
            pad[:vocab] = l
            out[:, j // 16, :, j % 16] = pad.reshape(-1, 16)
    return {"logits": out if c["written"] else None, "value": values, "index": None, "counts": None, "seen": None}
