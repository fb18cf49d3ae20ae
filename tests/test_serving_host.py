"""The serving engine's host side: the book of pages against a pool that is simulated entry by
entry, and the scheduler over a model that hashes what its rows see. No GPU."""
import types

import numpy as np
import pytest

from stride_amd import cli, engine, serving


class Table:
    """What kv_pool.KvPool does to table and counts, one entry at a time."""

    def __init__(self, slots, blocks, pages, page_tokens):
        self.table, self.refs, self.page = [[-1] * blocks for _ in range(slots)], [0] * pages, page_tokens
        self.tokens = [[None] * page_tokens for _ in range(pages)]

    def release(self, slot, first, end):
        for s, a, b in zip(slot, first, end):
            for i in range(a, b):
                if self.table[s][i] >= 0:
                    self.refs[self.table[s][i]] -= 1
                    self.table[s][i] = -1

    def reserve(self, slot, first, end):
        for s, a, b in zip(slot, first, end):
            for i in range(a, b):
                if self.table[s][i] < 0:
                    p = self.refs.index(0)  # ValueError: the book let too much through
                    self.refs[p], self.table[s][i] = 1, p

    def fork(self, src, dst, length):
        for s, d, n in zip(src, dst, length):
            for i in range(n // self.page):
                self.table[d][i] = self.table[s][i]
                if self.table[s][i] >= 0:
                    self.refs[self.table[s][i]] += 1
            i = n // self.page
            if n % self.page and self.table[s][i] >= 0:
                p = self.refs.index(0)
                self.refs[p], self.table[d][i] = 1, p
                self.tokens[p] = list(self.tokens[self.table[s][i]])

    def check(self):
        pass


class Model(serving.ServingEngine):
    """A ServingEngine whose token is a hash of the tokens that its row sees in the pages."""

    def __init__(self, slots, max_ctx, max_rows, page, pages, window=0, sinks=0):
        self.window, self.sinks, self.max_rows = window, sinks, max_rows
        blocks = -(-max_ctx // page)
        self.pool = Table(slots, blocks, pages or slots * blocks, page)
        self.kv = types.SimpleNamespace(slots=slots, capacity=blocks * page, page_tokens=page)
        self.book = serving.Pages(slots, len(self.pool.refs), page, window, sinks)
        self.rules = [None] * slots
        self.cfg = types.SimpleNamespace(vocab=1000)
        self.counts = self.masks = None
        self.work = self.most_used = 0

    def _ints(self, lists):
        return lists

    def step(self, rows, greedy, **how):
        assert len(rows) <= self.max_rows
        self.hold(rows)
        pool, out = self.pool, []
        assert self.book.used == sum(r > 0 for r in pool.refs)
        for s, held in enumerate(self.book.held):
            assert sorted(held) == [i for i, p in enumerate(pool.table[s]) if p >= 0]
            assert [held[i][0] for i in sorted(held)] == [pool.refs[p] for p in pool.table[s] if p >= 0]
        self.work += len(rows)
        self.most_used = max(self.most_used, self.book.used)
        for s, p, t in rows:
            at = pool.table[s][p // pool.page]
            assert pool.refs[at] == 1, "a shared page is written"
            pool.tokens[at][p % pool.page] = t
        for s, p, t in (rows[i] for i in greedy):
            h = engine.FNV_OFFSET
            for i in range(p + 1):
                if self.window <= 0 or p - i < self.window or i < self.sinks:
                    h = engine.fnv_mix(h, pool.tokens[pool.table[s][i // pool.page]][i % pool.page] + 1000 * i)
            out.append((h % 1000, h >> 32))
        return out


def prompts(seed, n, longest, shared):
    rng = np.random.default_rng(seed)
    base = rng.integers(0, 1000, longest).tolist()
    out = []
    for i in range(n):
        keep = int(rng.integers(0, longest)) if shared else 0
        out.append((i, base[:keep] + rng.integers(0, 1000, int(rng.integers(1, longest - keep + 1))).tolist()))
    return out


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 0), (20, 5), (33, 16), (200, 9)])
@pytest.mark.parametrize("page", [8, 16])
def test_scheduling_changes_no_ledger(window, sinks, page):
    todo = prompts(window + page, 14, 90, True)
    new, ctx = 12, 102
    alone = cli.Scheduler(Model(1, ctx, 128, page, 0, window, sinks), 1, new).run(todo)
    want = list(cli.ledger_lines(todo, alone))
    for seed, (slots, rows, pages) in enumerate([(3, 16, 0), (5, 40, 30), (14, 200, 60), (4, 7, 16)]):
        for share in (False, True):
            eng = Model(slots, ctx, rows, page, pages, window, sinks)
            if not all(eng.fits(len(t) + new) for _, t in todo):
                with pytest.raises(ValueError):
                    cli.Scheduler(eng, slots, new, share_prefixes=share).run(todo)
                continue
            got = list(cli.ledger_lines(todo, cli.Scheduler(eng, slots, new, row_shuffle=seed + 1, share_prefixes=share).run(todo)))
            assert got == want, (slots, rows, pages, share)
            assert eng.book.used == 0 and not any(eng.pool.refs)


def test_a_shared_prefix_is_processed_once():
    base = list(range(64))
    todo = [(i, base + [500 + i]) for i in range(6)]
    plain, shared = Model(6, 80, 100, 16, 0), Model(6, 80, 100, 16, 0)
    a = cli.Scheduler(plain, 6, 4).run(todo)
    b = cli.Scheduler(shared, 6, 4, share_prefixes=True).run(todo)
    assert list(cli.ledger_lines(todo, a)) == list(cli.ledger_lines(todo, b))
    assert plain.work - shared.work == 5 * 64 and shared.most_used == 4 + 6


def test_a_window_holds_its_pages_only():
    eng = Model(1, 400, 8, 16, 6, window=30, sinks=3)
    assert eng.fits(400) and not eng.fits(400, [400])
    cli.Scheduler(eng, 1, 40).run([(0, list(range(360)))])
    assert eng.most_used <= eng.book.most(400, 8) == 1 + 36 // 16 + 2


def test_book_refusals():
    book = serving.Pages(3, 4, 16, window=20)
    book.step([(0, p, 0) for p in range(40)])
    before = [dict(h) for h in book.held], book.used, list(book.gone), list(book.end)
    with pytest.raises(RuntimeError):  # 3 held, 1 passed, 3 wanted
        book.step([(0, 40, 0), (1, 16, 0), (2, 0, 0)])
    assert before == ([dict(h) for h in book.held], book.used, list(book.gone), list(book.end))
    assert book.step([(0, 70, 0)]) == ([(0, 0, 3)], [(0, 3, 5)])
    with pytest.raises(ValueError):
        book.step([(0, 40, 0)])
    assert book.shareable(0, 70) == 70 and book.shareable(0, 60) == 0 and book.shareable(0, 90) == 0 and book.shareable(1, 5) == 0
    with pytest.raises(ValueError):
        book.fork(0, 1, 60)
    with pytest.raises(ValueError):
        book.fork(0, 0, 70)
    book.step([(2, 0, 0), (1, 0, 0)])  # 2 held, 2 wanted
    with pytest.raises(RuntimeError):
        serving_book = serving.Pages(2, 1, 16)
        serving_book.step([(0, 3, 0)])
        serving_book.fork(0, 1, 4)
    with pytest.raises(ValueError):
        book.fork(0, 1, 70)  # slot 1 is in use
    assert book.finish(0) == 5 and book.finish(1) == 1 and book.finish(2) == 1 and book.used == 0


def test_rules_and_scheduler_refusals():
    for bad in (dict(repetition=0.0), dict(repetition=-1.0), dict(presence=float("nan")), dict(bias={3: float("inf")}), dict(allowed=[])):
        with pytest.raises(ValueError):
            serving.Rules(**bad)
    assert not serving.Rules(bias={1: 2.0}).counted and serving.Rules(presence=0.1).counted
    eng = Model(2, 64, 8, 16, 0)
    for rules in (serving.Rules(bias={1000: 1.0}), serving.Rules(allowed=[-1])):
        with pytest.raises(ValueError):
            eng.begin(0, [1], rules)
    eng.begin(0, [1])
    eng.step([(0, 0, 1)], [0])
    with pytest.raises(ValueError):
        eng.begin(0, [1])
    with pytest.raises(ValueError):
        cli.Scheduler(types.SimpleNamespace(), 1, 1, share_prefixes=True)
    with pytest.raises(ValueError):
        serving.ServingEngine(None, 1, 64, 8, window=0, sinks=4)
    for args in (["--window", "5"], ["--path", "serve", "--kv-shuffle", "3"]):
        with pytest.raises(SystemExit):
            cli.main(["--model", "m", "--input", "i", "--output", "o", *args])


def test_longest_run():
    assert serving.longest_run([]) == 0
    assert serving.longest_run([(s, 0, 0) for s in (1, 1, 2, 2, 2, 1)]) == 3


def test_slots_that_are_none():
    """Python's negative indices name the last slots: a branch of slot -1 was one of the last
    slot in the book and none on the device, whose pages the branch then lacked."""
    eng = Model(3, 64, 40, 16, 0)
    eng.begin(2, list(range(40)))
    eng.step([(2, p, p) for p in range(40)], [])
    before = eng.book.used, [dict(h) for h in eng.book.held]
    for source in (-1, -3, 3, 100):
        assert eng.shareable(source, 20) == 0
        with pytest.raises(ValueError):
            eng.begin(0, list(range(30)), None, source, 20)
    for shared in (-5, 31):
        with pytest.raises(ValueError):
            eng.begin(0, list(range(30)), None, 2, shared)
    with pytest.raises(ValueError):
        eng.book.fork(2, -2, 20)
    for slot in (-1, 3):
        with pytest.raises(ValueError):
            eng.finish(slot)
        with pytest.raises(ValueError):
            eng.begin(slot, [1])
    assert before == (eng.book.used, [dict(h) for h in eng.book.held])
    eng.begin(0, list(range(30)), None, 2, 20)
    assert eng.pool.table[0][:1] == eng.pool.table[2][:1]


@pytest.mark.parametrize("page", [8, 16])
def test_what_is_not_processed_is_not_shared(page):
    """A source that has processed part of a page: a branch at the page's end would share it with
    places that the source has yet to write."""
    eng = Model(3, 64, 40, page, 0)
    eng.begin(0, list(range(40)))
    eng.step([(0, p, p) for p in range(10)], [])
    for length in (11, 16, 17, 40):
        assert eng.shareable(0, length) == 0
        with pytest.raises(ValueError):
            eng.begin(1, list(range(40)), None, 0, length)
    assert [eng.shareable(0, n) for n in (1, 8, 10)] == [1, 8, 10] and eng.shareable(1, 1) == 0
    eng.begin(1, list(range(40)), None, 0, 10)
    assert eng.shareable(1, 10) == 10 and eng.shareable(1, 11) == 0  # a branch of a branch
    eng.step([(0, p, p) for p in range(10, 30)] + [(1, 10, 10)], [])
    assert eng.shareable(0, 30) == 30 and eng.shareable(0, 31) == 0 and eng.shareable(1, 11) == 11
    eng.finish(0)
    assert eng.shareable(0, 1) == 0
    eng.begin(0, [1, 2])
    assert eng.shareable(0, 1) == 0


def test_a_shared_page_is_not_written():
    """A position that was processed before, in a page that a branch holds too, by the source or
    the branch: its other holder would read the new token. In a page of its own it may come again."""
    eng = Model(3, 64, 40, 16, 0)
    eng.begin(0, list(range(40)))
    eng.step([(0, p, p) for p in range(40)], [])
    eng.begin(1, list(range(40)), None, 0, 36)
    before = eng.book.used, [dict(h) for h in eng.book.held], list(eng.book.end), list(eng.book.done)
    for rows in ([(0, 5, 9)], [(1, 31, 9)], [(0, 40, 1), (0, 16, 9)], [(2, 0, 1), (1, 0, 9), (1, 36, 9)]):
        with pytest.raises(ValueError, match="another sequence"):
            eng.step(rows, [])
    assert before == (eng.book.used, [dict(h) for h in eng.book.held], list(eng.book.end), list(eng.book.done))
    eng.step([(0, 35, 9), (0, 40, 9), (1, 36, 8), (1, 33, 8)], [])  # the part page was copied
    eng.finish(1)
    eng.step([(0, 5, 5)], [])


def test_a_refused_call_changes_no_book():
    """Too many rows, none, a greedy row that is none, a stream of set_kernel_stream's: refused
    before the book or the pool has changed."""
    from stride_amd import tc

    eng = Model(2, 64, 8, 16, 0)
    eng.begin(0, [1, 2, 3])
    eng.step([(0, 0, 1)], [])
    state = lambda: (eng.book.used, [sorted(h) for h in eng.book.held], list(eng.book.end), list(eng.book.done), [list(t) for t in eng.pool.table])
    before = state()
    real = serving.ServingEngine.step
    for rows, greedy in (([(0, p, 1) for p in range(1, 20)], []), ([], []), ([(0, 20, 1)], [1]), ([(0, 20, 1)], [-1])):
        with pytest.raises(ValueError):
            real(eng, rows, greedy)
        assert state() == before
    tc.set_kernel_stream(12345)
    try:
        for call in (lambda: real(eng, [(0, 20, 1)], [0]), lambda: eng.hold([(0, 20, 1)]), lambda: eng.begin(1, [1, 2], None, 0, 1),
                     lambda: eng.begin(1, [1, 2]), lambda: eng.finish(0)):
            with pytest.raises(ValueError, match="current stream"):
                call()
            assert state() == before
    finally:
        tc.set_kernel_stream(None)
    eng.hold([(0, 20, 1)])
    assert state() != before


def test_head_layouts():
    """The serving engine's attention has 1 to 16 query heads a group, the plain engine's four."""
    from stride_amd.weights import ModelConfig

    serve, plain = (e._check_heads for e in (serving.ServingEngine, engine.Engine))
    for heads, kv_heads, D, ok, four in ((8, 2, 64, True, True), (2, 2, 32, True, False), (16, 1, 128, True, False), (14, 2, 64, True, False),
                                         (17, 1, 64, False, False), (8, 2, 80, False, False), (7, 2, 64, False, False)):
        cfg = ModelConfig(heads=heads, kv_heads=kv_heads, head_dim=D)
        for check, served in ((serve, ok), (plain, four)):
            if served:
                check(None, cfg)
            else:
                with pytest.raises(ValueError, match="head_dim"):
                    check(None, cfg)
