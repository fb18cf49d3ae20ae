"""A decode engine over the serving operators: bounded contexts, shared pages, logit rules.

ServingEngine is engine.Engine with three parts replaced. Attention is window_attention: every
position up to a row's own, or the last `window` and the first `sinks` ones. KV pages come from
a kv_pool.KvPool: a sequence holds those that its rows still see, a page behind its window goes
back before the step's own are taken, and a sequence whose prompt begins as another's goes on
from the other's pages. Tokens are chosen by logits.process where a sequence has Rules, from
lm_full's logits, and by lm_greedy elsewhere.

    eng = ServingEngine(weights, slots, max_ctx, max_rows, pages=512, window=1024, sinks=4)
    eng.begin(0, prompt, Rules(repetition=1.1))
    eng.begin(1, other, source=0, shared=eng.shareable(0, 96))   # from slot 0's first 96 tokens
    eng.step(rows, greedy)                                       # as Engine.step
    eng.finish(0)

As there, a row's result depends on its own sequence and rules only: sharing, the pool's size,
the order of rows and their batch change no bit. The reference has no counterpart.
"""
from __future__ import annotations

import dataclasses
import math
import typing

import torch

from . import engine, harness, logits, tc
from .kv_pool import KvPool


@dataclasses.dataclass(frozen=True)
class Rules:
    """How a sequence's next token is chosen (the formula: stride_amd.logits). bias: {token:
    value}; allowed: the tokens that may be chosen (None: all)."""

    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: typing.Mapping | None = None
    allowed: typing.Collection | None = None

    def __post_init__(self):
        numbers = (self.repetition, self.presence, self.frequency, *(self.bias or {}).values())
        if not all(math.isfinite(x) for x in numbers) or self.repetition <= 0:
            raise ValueError("penalties and biases are finite, and a repetition penalty is above 0")
        if self.allowed is not None and not len(self.allowed):
            raise ValueError("no token is allowed")

    @property
    def counted(self) -> bool:
        return (self.repetition, self.presence, self.frequency) != (1.0, 0.0, 0.0)


class RowRules(typing.NamedTuple):
    """Rules of the rows that get a token, on the device: logits.process's arguments."""

    counts: logits.TokenCounts | None
    row_slot: torch.Tensor
    penalties: torch.Tensor | None
    bias: tuple | None
    mask: torch.Tensor | None
    mask_row: torch.Tensor | None


class Pages:
    """The pages of a pool as the host counts them: which table entries each slot holds and how
    many slots hold a page together, so that a full pool is known before a launch. `sinks` and
    `window` in tokens as in window_attention (window 0: nothing is given up)."""

    def __init__(self, slots: int, pages: int, page_tokens: int, window: int = 0, sinks: int = 0):
        self.total, self.page, self.window = pages, page_tokens, window
        self.first = self.of(sinks)  # entries that are never given up
        self.used = 0
        self.held = [{} for _ in range(slots)]  # entry -> [its holders' number], one list a page
        self.gone = [self.first] * slots        # entries [first, gone) were given up
        self.end = [0] * slots                  # entries from here on were never held
        self.done = [0] * slots                 # tokens that steps have processed, or a branch began with

    def of(self, tokens: int) -> int:
        return (tokens + self.page - 1) // self.page

    def seen_from(self, pos: int) -> int:
        """The first entry behind the sinks that a row at `pos` sees."""
        return max(self.first, (pos - self.window + 1) // self.page) if self.window > 0 else self.first

    def most(self, tokens: int, max_rows: int) -> int:
        """The most pages that a sequence of `tokens` tokens holds, in steps of max_rows rows."""
        if self.window <= 0:
            return self.of(tokens)
        return min(self.of(tokens), self.first + (self.window + max_rows - 2) // self.page + 2)

    def drop(self, slot: int, entries) -> None:
        for b in entries:
            page = self.held[slot].pop(b, None)
            if page is not None:
                page[0] -= 1
                self.used -= page[0] == 0

    def shared(self, slot: int, entry: int) -> bool:
        return self.held[slot].get(entry, (1,))[0] > 1

    def step(self, rows):
        """(released, reserved) lists of (slot, first, end) for a step's rows [(slot, pos,
        token)], the released ones first. Raises, with nothing changed, where a row would see
        what was given up or write what another sequence holds too, or the pool is too small."""
        spans = {}
        for s, p, *_ in rows:
            lo, hi = spans.get(s, (p, p))
            spans[s] = min(lo, p), max(hi, p)
        released, reserved, freed, wanted = [], [], {}, 0
        for s, (lo, hi) in spans.items():
            seen, end = self.seen_from(lo), hi // self.page + 1
            if seen < self.gone[s]:
                raise ValueError(f"slot {s}: position {lo} sees pages that its window has passed")
            if any(self.shared(s, b) for b in range(lo // self.page, min(end, self.end[s]))):
                for p in (r[1] for r in rows if r[0] == s):
                    if self.shared(s, p // self.page):
                        raise ValueError(f"slot {s}: position {p} is in a page that another sequence holds too")
            if min(seen, self.end[s]) > self.gone[s]:
                released.append((s, self.gone[s], min(seen, self.end[s])))
                for b in range(*released[-1][1:]):
                    page = self.held[s][b]
                    freed[id(page)] = freed.get(id(page), page[0]) - 1
            if end > self.end[s]:
                reserved.append((s, self.end[s], end))
                wanted += end - self.end[s]
        if self.used + wanted - sum(left == 0 for left in freed.values()) > self.total:
            raise RuntimeError(f"the KV pool of {self.total} pages is too small for this step")
        for s, first, end in released:
            self.drop(s, range(first, end))
            self.gone[s] = end
        for s, first, end in reserved:
            for b in range(first, end):
                self.held[s][b] = [1]
            self.end[s] = end
        for s, (lo, hi) in spans.items():
            self.done[s] = max(self.done[s], hi + 1)
        self.used += wanted
        return released, reserved

    def shareable(self, src: int, length: int) -> int:
        """`length`, or 0 where src has not processed as much, a row at `length` would see what it
        has given up, or it is no slot."""
        if not 0 <= src < len(self.held):
            return 0
        return length if 0 < length <= self.done[src] and self.seen_from(length) >= self.gone[src] else 0

    def fork(self, src: int, dst: int, length: int) -> None:
        whole = length // self.page
        if not 0 <= dst < len(self.held) or self.held[dst]:
            raise ValueError(f"slot {dst} is in use, or none")
        if src == dst or self.shareable(src, length) != length:
            raise ValueError(f"slot {src} does not hold what a branch at {length} sees")
        part = length % self.page > 0 and whole in self.held[src]
        if self.used + part > self.total:
            raise RuntimeError("the pool has no page for a branch")
        for b, page in self.held[src].items():
            if b < whole:
                page[0] += 1
                self.held[dst][b] = page
        if part:
            self.held[dst][whole] = [1]
            self.used += 1
        self.gone[dst], self.end[dst], self.done[dst] = self.gone[src], self.of(length), length

    def finish(self, slot: int) -> int:
        """Gives a slot up; its entries end here."""
        if not 0 <= slot < len(self.held):
            raise ValueError(f"there is no slot {slot}")
        end = self.end[slot]
        self.drop(slot, list(self.held[slot]))
        self.gone[slot], self.end[slot], self.done[slot] = self.first, 0, 0
        return end


class ServingEngine(engine.Engine):
    """One model, a pool of `pages` KV pages (default: enough for every slot's max_ctx), window
    and sinks of every row's attention, and each slot's Rules."""

    def __init__(self, weights, slots: int, max_ctx: int, max_rows: int, page_tokens: int = 16, pages: int | None = None,
                 window: int = 0, sinks: int = 0):
        if window < 0 or sinks < 0 or (sinks and not window):
            raise ValueError("window and sinks are counts of tokens, and sinks need a window")
        self.window, self.sinks, self._pages = window, sinks, pages
        super().__init__(weights, slots, max_ctx, max_rows, page_tokens)
        self.most_pages = (self.kv.capacity + 63) // 64
        self.book = Pages(slots, self.pool.pages, page_tokens, window, sinks)
        self.rules = [None] * slots
        self.counts = self.masks = None
        self.lm_work = logits.scratch(max_rows, self.dev)

    def _check_heads(self, cfg) -> None:
        if cfg.head_dim not in (32, 64, 128) or cfg.heads % cfg.kv_heads or not 1 <= cfg.repeat() <= 16:
            raise ValueError("window_attention serves head_dim 32/64/128 with 1 to 16 query heads per KV head")

    def _cache(self, slots, max_ctx, page_tokens, shuffle_seed):
        cfg = self.cfg
        pages = self._pages if self._pages is not None else slots * ((max_ctx + page_tokens - 1) // page_tokens)
        self.pool = KvPool.create(slots, max_ctx, pages, cfg.kv_heads, cfg.head_dim, cfg.layers, page_tokens, self.dev)
        return self.pool.kv

    def _attention_scratch(self):
        return None  # a step's own: its size follows from the step's rows

    def device_rows(self, rows):
        """Device tensors (slot, pos, tok, None) for rows [(slot, pos, token)]."""
        t = torch.tensor([[r[i] for r in rows] for i in range(3)], dtype=torch.int32, device=self.dev)
        return t[0], t[1], t[2], None

    def _ready(self) -> None:
        """What a call allocates is torch's current stream's, and may go back to it while a launch
        on another one still reads it."""
        if tc._stream is not None:
            raise ValueError("a ServingEngine allocates for its steps, on torch's current stream: none may be set by set_kernel_stream")

    def _attention(self, n, slot, pos, items, runs):
        self._ready()
        cfg = self.cfg
        scale = float(math.pow(cfg.head_dim, -0.5))
        scratch = harness.window_attention_scratch(n, cfg.kv_heads, cfg.repeat(), cfg.head_dim, self.window, self.sinks,
                                                   self.most_pages, self.dev, runs)
        return lambda layer: harness.window_attention(
            self.q[:n], self.kv, slot, pos, cfg.kv_heads, cfg.repeat(), cfg.head_dim, scale, self.window, self.sinks, layer,
            self.most_pages, out_tiles=self.attn, scratch=scratch, runs=runs)

    def _choose(self, x, count, best, rules) -> None:
        if rules is None:
            return super()._choose(x, count, best, rules)
        tiles = harness.lm_full(self.w.lm, x, count)
        logits.process(tiles, count, self.cfg.vocab, rules.counts, rules.row_slot, rules.penalties, rules.bias, rules.mask,
                       rules.mask_row, best=best, work=self.lm_work)
        if rules.counts is not None:
            rules.counts.record(rules.row_slot, best[:, 1])

    def begin(self, slot: int, prompt, rules: Rules | None = None, source: int = -1, shared: int = 0) -> None:
        """A sequence begins in a free slot, from the first `shared` tokens of slot `source`
        (at most what shareable() says), so that its first row is at position `shared`."""
        self._ready()
        if not 0 <= slot < self.kv.slots or self.book.end[slot]:
            raise ValueError(f"slot {slot} is in use, or none")
        named = [] if rules is None else [*(rules.bias or ()), *(rules.allowed or ())]
        if not all(0 <= t < self.cfg.vocab for t in named):
            raise ValueError("the rules name a token outside the vocabulary")
        if shared and not 0 < shared <= len(prompt):
            raise ValueError(f"{shared} shared tokens of a prompt of {len(prompt)}")
        if shared:
            self.book.fork(source, slot, shared)
            self.pool.fork(*self._ints([[source], [slot], [shared]]))
        self.rules[slot] = rules
        if rules is None:
            return
        if rules.counted:
            if self.counts is None:
                self.counts = logits.TokenCounts.create(self.kv.slots, self.cfg.vocab, self.dev)
            at = torch.tensor([slot], dtype=torch.int32, device=self.dev)
            self.counts.reset(at)
            tokens = torch.tensor(list(prompt), dtype=torch.int32, device=self.dev)
            self.counts.record(at.expand(tokens.numel()).contiguous(), tokens, prompt=True)
        if rules.allowed is not None:
            if self.masks is None:
                self.masks = torch.zeros((self.kv.slots, logits.words(self.cfg.vocab)), dtype=torch.int32, device=self.dev)
            self.masks[slot] = logits.mask_of([rules.allowed], self.cfg.vocab, self.dev)[0]

    def finish(self, slot: int) -> None:
        """The slot's pages go back, and it is free."""
        self._ready()
        end = self.book.finish(slot)
        if end:
            self.pool.release(*self._ints([[slot], [0], [end]]))
        self.rules[slot] = None

    def shareable(self, source: int, length: int) -> int:
        """How many of the first `length` tokens of `source` another sequence can begin with: all of
        them, or none where it has not processed as many, or the window has passed what the
        other would see."""
        return self.book.shareable(source, length)

    def fits(self, tokens: int, others=()) -> bool:
        """Whether a sequence of `tokens` tokens can run to its end beside `others`, their
        tokens, whatever pages they share."""
        return sum(self.book.most(t, self.max_rows) for t in (tokens, *others)) <= self.book.total

    def _ints(self, lists):
        t = torch.tensor(lists, dtype=torch.int32, device=self.dev)
        return tuple(t[i] for i in range(len(lists)))

    def hold(self, rows) -> None:
        """Gives up the pages that the windows of a step's rows [(slot, pos, token)] have passed
        and takes those that the step writes. step() does so itself."""
        self._ready()
        slots, end = self.kv.slots, self.kv.capacity
        if not all(0 <= r[0] < slots and 0 <= r[1] < end for r in rows):
            raise ValueError("a row's slot or position is outside the cache")
        released, reserved = self.book.step(rows)
        if released:
            self.pool.release(*self._ints(list(zip(*released))))
        if reserved:
            self.pool.reserve(*self._ints(list(zip(*reserved))))

    def row_rules(self, slots) -> RowRules | None:
        """The rules of rows of these slots, on the device (None: none of them has any)."""
        rules = [self.rules[s] for s in slots]
        if not any(rules):
            return None
        plain = Rules()
        rules = [r or plain for r in rules]
        dev, counted = self.dev, any(r.counted for r in rules)
        row_slot = torch.tensor(slots, dtype=torch.int32, device=dev)
        penalties = mask_row = bias = None
        if counted:
            penalties = torch.tensor([(r.repetition, r.presence, r.frequency) for r in rules], dtype=torch.float32, device=dev)
        if any(r.bias for r in rules):
            bias = logits.bias_lists([r.bias for r in rules], dev)
        masked = any(r.allowed is not None for r in rules)
        if masked:
            mask_row = torch.tensor([-1 if r.allowed is None else s for s, r in zip(slots, rules)], dtype=torch.int32, device=dev)
        return RowRules(self.counts if counted else None, row_slot, penalties, bias, self.masks if masked else None, mask_row)

    def step(self, rows, greedy, **how):
        """Engine.step, with the pages that it needs and the rules of the rows' slots. A step that
        is refused, one that would write a page that another sequence holds too among them,
        changes nothing."""
        if not 0 < len(rows) <= self.max_rows:
            raise ValueError(f"a step has 1 to {self.max_rows} rows, not {len(rows)}")
        if not all(0 <= i < len(rows) for i in greedy):
            raise ValueError("greedy names a row that the step does not have")
        self.hold(rows)
        got = super().step(rows, greedy, rules=self.row_rules([rows[i][0] for i in greedy]), runs=longest_run(rows), **how)
        for i, (token, _) in zip(greedy, got):
            if token < 0:
                raise ValueError(f"slot {rows[i][0]}: no token can be chosen")
        return got

    def check(self) -> None:
        """Raises what the pool's calls reported (waits for the device)."""
        self.pool.check()


def longest_run(rows) -> int:
    """How many neighbouring rows are of one slot at most."""
    most = run = 0
    last = None
    for s, *_ in rows:
        run = run + 1 if s == last else 1
        last, most = s, max(most, run)
    return most
