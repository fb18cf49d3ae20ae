"""The page pool (stride_amd.kv_pool) against a plain model of it on the host: tables, counts
and every byte of the arena after each call; shared pages; refusals that leave all as it was;
capture; pages past 32 bits. Everything is whole numbers or copied bits: no tolerance."""
import numpy as np
import pytest
import torch

from stride_amd import harness, kv_pool, layout, tc
from stride_amd._lib import StrideTcError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def say(*a):
    print(*a, flush=True)


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


class Model:
    """What the calls mean, in lists and NumPy."""

    def __init__(self, pool):
        self.pt, self.pages = pool.page_tokens, pool.pages
        self.table = pool.table.cpu().numpy().copy()
        self.refs = pool.refs.cpu().numpy().copy()
        self.arena = pool.arena.cpu().numpy().reshape(pool.pages, pool.layers, 2, pool.kv_heads, pool.page_tokens, pool.head_dim).copy()

    def _take(self, count):
        free = np.flatnonzero(self.refs == 0)[:count]
        assert len(free) == count
        self.refs[free] = 1
        return free.tolist()

    def _drop(self, b):
        if b >= 0:
            self.refs[b] -= 1

    def reserve(self, slot, first, end):
        want = [(s, b) for s, a, e in zip(slot, first, end) for b in range(a, e) if self.table[s, b] < 0]
        for (s, b), page in zip(want, self._take(len(want))):
            self.table[s, b] = page

    def release(self, slot, first, end):
        for s, a, e in zip(slot, first, end):
            for b in range(max(a, 0), min(e, self.table.shape[1])):
                self._drop(self.table[s, b])
                self.table[s, b] = -1

    def fork(self, src, dst, length):
        part = [i for i, (s, n) in enumerate(zip(src, length)) if n % self.pt and self.table[s, n // self.pt] >= 0]
        fresh = dict(zip(part, self._take(len(part))))
        for i, (s, d, n) in enumerate(zip(src, dst, length)):
            old = self.table[d].copy()
            full = n // self.pt
            self.table[d] = -1
            for b in range(full):
                self.table[d, b] = self.table[s, b]
                if self.table[s, b] >= 0:
                    self.refs[self.table[s, b]] += 1
            if i in fresh:
                self.table[d, full] = fresh[i]
                self.arena[fresh[i], :, :, :, :n % self.pt] = self.arena[self.table[s, full], :, :, :, :n % self.pt]
            for b in old:
                self._drop(b)

    def compact(self, slot, first, count, keep):
        want = []
        for s, f, c in zip(slot, first, count):
            for b in range(f // self.pt, -(-(f + c) // self.pt) if c else f // self.pt):
                if self.table[s, b] < 0 or self.refs[self.table[s, b]] > 1:
                    want.append((s, b))
        fresh = dict(zip(want, self._take(len(want))))
        before, old = self.arena.copy(), self.table.copy()
        for s, f, c, ks in zip(slot, first, count, keep):
            moves = [(f + k, ks[k]) for k in range(c)]
            if c and (s, f // self.pt) in fresh:
                moves += [(t, t) for t in range(f // self.pt * self.pt, f) if old[s, f // self.pt] >= 0]
            for to, frm in moves:
                b = fresh.get((s, to // self.pt), old[s, to // self.pt])
                self.arena[b, :, :, :, to % self.pt] = before[old[s, frm // self.pt], :, :, :, frm % self.pt]
            for b in range(f // self.pt, self.table.shape[1]):
                if (s, b) in fresh:
                    self.table[s, b] = fresh[(s, b)]
                    self._drop(old[s, b])
                elif b >= -(-(f + c) // self.pt):
                    self._drop(self.table[s, b])
                    self.table[s, b] = -1


def same(pool, model):
    torch.cuda.synchronize()
    assert np.array_equal(pool.table.cpu().numpy(), model.table)
    assert np.array_equal(pool.refs.cpu().numpy(), model.refs)
    bits = pool.free_bits.cpu().numpy().view(np.uint8)
    assert np.array_equal(np.unpackbits(bits, bitorder="little")[:pool.pages].astype(bool), model.refs == 0)
    assert np.array_equal(pool.arena.cpu().numpy().reshape(model.arena.shape).view(np.uint8), model.arena.view(np.uint8))
    held = np.bincount(model.table[model.table >= 0], minlength=pool.pages)
    assert np.array_equal(held, model.refs), "the counts are the table's"


def make(seed, slots=6, max_ctx=200, pages=80, kv_heads=2, D=32, layers=3, pt=16, fp32=False):
    pool = kv_pool.KvPool.create(slots, max_ctx, pages, kv_heads, D, layers, pt, DEV, fp32=fp32)
    g = torch.Generator(device=DEV).manual_seed(seed)
    if fp32:
        pool.arena.normal_(generator=g)
    else:
        pool.arena.copy_(torch.randint(-32768, 32768, pool.arena.shape, generator=g, device=DEV, dtype=torch.int16))
    return pool, Model(pool)


def both(pool, model, call, *lists):
    getattr(pool, call)(*(i32(x) for x in lists))
    pool.check()
    getattr(model, call)(*lists)
    same(pool, model)


def compact(pool, model, slot, first, keep):
    count = [len(k) for k in keep]
    width = max(count + [1])
    pool.compact(i32(slot), i32(first), i32(count), torch.tensor([k + [0] * (width - len(k)) for k in keep], dtype=torch.int32, device=DEV))
    pool.check()
    model.compact(slot, first, count, keep)
    same(pool, model)


@pytest.mark.parametrize("pt,D,fp32", [(16, 32, False), (8, 64, False), (1, 32, False), (64, 128, False), (16, 64, True), (4, 24, False)])
def test_a_life(pt, D, fp32):
    """Prompts come, branch, branch again, diverge, shrink and go."""
    say("life", pt, D, fp32)
    pool, m = make(1, slots=7, max_ctx=100, pages=7 * -(-100 // pt) + 3, pt=pt, D=D, fp32=fp32)
    e = lambda n: -(-n // pt)
    both(pool, m, "reserve", [2, 0], [0, 0], [e(70), e(33)])
    both(pool, m, "reserve", [0, 2, 4], [e(33), 0, 1], [e(40), e(71), 1])   # nothing new, some, an empty range
    both(pool, m, "fork", [2, 0, 2], [1, 5, 3], [64, 33, 69])
    both(pool, m, "fork", [1, 2], [4, 6], [50, 0])                          # from a branch; of nothing
    both(pool, m, "reserve", [1, 4], [0, 0], [e(80), e(60)])
    both(pool, m, "fork", [3], [5], [17])                                   # over a branch that held pages
    both(pool, m, "release", [2, 2, 0], [0, 0, 0], [e(100), e(100), 1])     # twice, and a part
    compact(pool, m, [1], [10], [[10, 12, 30, 31, 32, 64, 79]])             # shared pages are replaced
    compact(pool, m, [4, 3], [0, 60], [list(range(5, 55)), []])             # everything moves; a tail goes
    both(pool, m, "release", [1, 3, 4, 5, 6, 0], [0] * 6, [1000] * 6)
    assert pool.free_pages() == pool.pages


def test_random_lives():
    for seed in range(4):
        rng = np.random.default_rng(seed)
        pool, m = make(seed, slots=8, max_ctx=160, pages=90, pt=16)
        length = [0] * 8
        for step in range(25):
            what = rng.integers(0, 4)
            order = rng.permutation(8).tolist()
            if what == 0:
                some = [s for s in order[:3] if length[s] < 140]
                grown = [min(160, length[s] + int(rng.integers(1, 60))) for s in some]
                need = sum(-(-g // 16) - int((m.table[s] >= 0).sum()) for s, g in zip(some, grown))
                if some and need <= int((m.refs == 0).sum()):
                    both(pool, m, "reserve", some, [0] * len(some), [-(-g // 16) for g in grown])
                    for s, g in zip(some, grown):
                        length[s] = g
            elif what == 1:
                src = [s for s in order[:2] if length[s]]
                dst = order[4:4 + len(src)]
                n = [int(rng.integers(0, length[s] + 1)) for s in src]
                if src and int((m.refs == 0).sum()) >= len(src):
                    both(pool, m, "fork", src, dst, n)
                    for d, x in zip(dst, n):
                        length[d] = x
            elif what == 2:
                some = [s for s in order[:3] if length[s]]
                if some and int((m.refs == 0).sum()) >= 30:
                    first = [int(rng.integers(0, length[s])) for s in some]
                    keep = [sorted(rng.choice(np.arange(f, length[s]), int(rng.integers(0, length[s] - f + 1)), replace=False).tolist())
                            for s, f in zip(some, first)]
                    compact(pool, m, some, first, keep)
                    for s, f, k in zip(some, first, keep):
                        length[s] = f + len(k)
            else:
                some = order[:2]
                both(pool, m, "release", some, [0, 0], [10, 10])
                for s in some:
                    length[s] = 0


def test_long_compaction_in_place():
    """Thousands of positions move within their own pages, by one and by many."""
    pool, m = make(3, slots=2, max_ctx=4096, pages=600, layers=1, D=64, pt=16)
    both(pool, m, "reserve", [0, 1], [0, 0], [256, 256])
    rng = np.random.default_rng(5)
    compact(pool, m, [1, 0], [4, 0], [sorted(rng.choice(np.arange(4, 4096), 3000, replace=False).tolist()), list(range(1, 4096))])


def test_two_branches_compact_their_shared_pages_at_once():
    pool, m = make(4, slots=4, max_ctx=96, pages=40)
    both(pool, m, "reserve", [0], [0], [6])
    both(pool, m, "fork", [0, 0], [1, 2], [96, 96])
    compact(pool, m, [1, 0, 2], [5, 5, 20], [[7, 50, 95], [6, 40, 41, 90], [21, 22, 60]])


def test_copy():
    pool, m = make(5)
    pool.copy(i32([3, 3, 8]), i32([10, 11, 79]), i32([5, 0, 16]))
    pool.check()
    m.arena[10, :, :, :, :5] = m.arena[3, :, :, :, :5]
    m.arena[79] = m.arena[8]
    same(pool, m)
    other, o = make(6, pages=40)
    pool.copy(i32([1, 2, 79]), i32([2, 1, 39]), into=other)
    pool.check()
    o.arena[2], o.arena[1], o.arena[39] = m.arena[1], m.arena[2], m.arena[79]
    same(other, o)
    same(pool, m)


def unchanged(pool, model, bit, call, *args):
    getattr(pool, call)(*args)
    with pytest.raises(StrideTcError, match=kv_pool.MESSAGES[bit][:20]):
        pool.check()
    same(pool, model)
    pool.check()


def test_calls_that_break_a_rule_change_nothing():
    pool, m = make(7, slots=6, pages=20)
    both(pool, m, "reserve", [0, 1], [0, 0], [5, 4])
    both(pool, m, "fork", [0], [2], [70])
    big = [2 ** 31 - 1, -2 ** 31]
    for s in [6, -1] + big:
        unchanged(pool, m, kv_pool.BAD_ITEM, "reserve", i32([1, s]), i32([0, 0]), i32([6, 6]))
        unchanged(pool, m, kv_pool.BAD_ITEM, "fork", i32([0, s]), i32([3, 4]), i32([5, 5]))
        unchanged(pool, m, kv_pool.BAD_ITEM, "fork", i32([0, 1]), i32([3, s]), i32([5, 5]))
        unchanged(pool, m, kv_pool.BAD_ITEM, "compact", i32([1, s]), i32([0, 0]), i32([1, 1]), torch.zeros((2, 1), dtype=torch.int32, device=DEV))
        unchanged(pool, m, kv_pool.BAD_ITEM, "release", i32([s]), i32([0]), i32([6]))
    for a, b in [(-1, 3), (0, 14)] + [(big[1], 3), (0, big[0])]:
        unchanged(pool, m, kv_pool.BAD_ITEM, "reserve", i32([1]), i32([a]), i32([b]))
    for n in [-1, 209] + big:
        unchanged(pool, m, kv_pool.BAD_ITEM, "fork", i32([0]), i32([3]), i32([n]))
    for f, c in [(-1, 1), (0, -1), (0, 3), (207, 2)] + [(big[0], 1), (big[1], 1), (0, big[0])]:
        unchanged(pool, m, kv_pool.BAD_ITEM, "compact", i32([1]), i32([f]), i32([c]), i32([1, 2]).reshape(1, 2))
    unchanged(pool, m, kv_pool.TWICE, "reserve", i32([3, 3]), i32([0, 1]), i32([1, 2]))
    unchanged(pool, m, kv_pool.TWICE, "fork", i32([0, 1]), i32([3, 3]), i32([5, 5]))
    unchanged(pool, m, kv_pool.TWICE, "fork", i32([0, 3]), i32([3, 4]), i32([5, 5]))
    unchanged(pool, m, kv_pool.TWICE, "fork", i32([0]), i32([0]), i32([5]))
    unchanged(pool, m, kv_pool.TWICE, "compact", i32([1, 1]), i32([0, 0]), i32([1, 1]), i32([3, 4]).reshape(2, 1))
    unchanged(pool, m, kv_pool.NO_PAGES, "reserve", i32([3, 4]), i32([0, 0]), i32([6, 6]))
    both(pool, m, "reserve", [3], [0], [10])  # ten of the ten that are left
    unchanged(pool, m, kv_pool.NO_PAGES, "fork", i32([0]), i32([4]), i32([5]))
    unchanged(pool, m, kv_pool.NO_PAGES, "compact", i32([2]), i32([3]), i32([1]), i32([9]).reshape(1, 1))
    for args in ((i32([20]), i32([1])), (i32([1]), i32([20])), (i32([-1]), i32([2])), (i32([1]), i32([big[1]]))):
        unchanged(pool, m, kv_pool.BAD_ITEM, "copy", *args)
    unchanged(pool, m, kv_pool.BAD_ITEM, "copy", i32([0]), i32([1]), i32([17]))
    unchanged(pool, m, kv_pool.TWICE, "copy", i32([0, 1]), i32([5, 5]))
    unchanged(pool, m, kv_pool.TWICE, "copy", i32([0, 1]), i32([1, 5]))


def test_lists_that_do_not_ascend_are_reported():
    pool, m = make(8)
    both(pool, m, "reserve", [0, 1], [0, 0], [6, 6])
    pool.compact(i32([0, 1]), i32([3, 3]), i32([3, 3]), i32([5, 9, 7, 4, 8, 90]).reshape(2, 3))
    with pytest.raises(StrideTcError, match="ascend"):
        pool.check()
    m.compact([1], [3], [3], [[4, 8, 90]])  # the other slot is right
    torch.cuda.synchronize()
    got = pool.arena.cpu().numpy().reshape(m.arena.shape)
    for t in range(6):
        b = int(pool.table[1, t // 16])
        assert np.array_equal(got[b, :, :, :, t % 16], m.arena[m.table[1, t // 16], :, :, :, t % 16])
    for keep, bit in (([2], "ascend"), ([2 ** 31 - 1], "ascend"), ([-5], "ascend"), ([150], "no page")):
        pool.compact(i32([1]), i32([3]), i32([1]), i32(keep).reshape(1, 1))
        with pytest.raises(StrideTcError, match=bit):
            pool.check()


def test_captured_and_replayed():
    """Reserve, fork, compact and release in one graph: every replay does its work anew."""
    pool, m = make(9, slots=4, max_ctx=96, pages=30)
    both(pool, m, "reserve", [0], [0], [5])
    src, dst, length = i32([0, 0]), i32([1, 2]), i32([70, 33])
    slot, first, count, keep = i32([1]), i32([60]), i32([2]), i32([61, 69]).reshape(1, 2)
    lo, hi = i32([0, 0]), i32([6, 6])

    def work():
        pool.release(dst, lo, hi)
        pool.fork(src, dst, length)
        pool.compact(slot, first, count, keep)
        pool.reserve(slot, lo[:1], hi[:1])

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for k in range(4):
        length.copy_(i32([70 + k, 33 + 2 * k]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        pool.check()
        m.release([1, 2], [0, 0], [6, 6])
        m.fork([0, 0], [1, 2], [70 + k, 33 + 2 * k])
        m.compact([1], [60], [2], [[61, 69]])
        m.reserve([1], [0], [6])
        same(pool, m)
        pool.arena[:1000].add_(k)  # eager work in between
        m.arena.reshape(-1)[:1000] += k


def test_many_pages_and_slots():
    """Prefix sums over more items than threads, bit maps of many words."""
    pool = kv_pool.KvPool.create(3000, 64, 9001, 1, 8, 1, 16, DEV)
    m = Model(pool)
    rng = np.random.default_rng(2)
    order = rng.permutation(3000)[:2500].tolist()
    both(pool, m, "reserve", order, [0] * 2500, rng.integers(0, 4, 2500).tolist())
    both(pool, m, "release", order[:1500], [0] * 1500, [2] * 1500)
    rest = [s for s in range(3000) if s not in set(order)]
    src = order[2000:2000 + len(rest)]
    both(pool, m, "fork", src, rest, rng.integers(0, 65, len(rest)).tolist())
    both(pool, m, "reserve", order[:1200], [0] * 1200, [2] * 1200)


def test_pages_past_32_bits():
    n_kv, D, pt, layers = 8, 128, 64, 4
    per = layers * 2 * n_kv * pt * D
    pages = (2 ** 32 + 2 ** 28) // per
    arena = torch.empty(pages * per, dtype=torch.int16, device=DEV)
    table = torch.full((3, 4), -1, dtype=torch.int32, device=DEV)
    refs = torch.ones(pages, dtype=torch.int32, device=DEV)  # held elsewhere, but for the last ones
    free = [2 ** 31 // per - 1, 2 ** 31 // per, 2 ** 32 // per - 1, 2 ** 32 // per, pages - 2, pages - 1]
    refs[free] = 0
    pool = kv_pool.KvPool(arena, table, refs, n_kv, D, layers, pt)
    pool.reserve(i32([0]), i32([0]), i32([4]))
    pool.check()
    assert pool.table[0].tolist() == free[:4]
    pagewise = arena.view(pages, layers * 2 * n_kv, pt, D)
    for b in free[:4]:
        pagewise[b].random_(-32768, 32768)
    before = {b: pagewise[b].clone() for b in free[:4]}
    pool.fork(i32([0]), i32([1]), i32([250]))
    pool.check()
    assert pool.table[1].tolist() == free[:3] + [free[4]]
    assert torch.equal(pagewise[free[4]][:, :58], before[free[3]][:, :58])
    pool.compact(i32([1]), i32([190]), i32([3]), i32([191, 200, 249]).reshape(1, 3))
    pool.check()
    assert pool.table[1].tolist() == free[:2] + [free[5], free[4]]  # the shared third page is replaced, the fourth is its own
    assert torch.equal(pagewise[free[5]][:, :62], before[free[2]][:, :62])
    assert torch.equal(pagewise[free[5]][:, 62], before[free[2]][:, 63])
    assert torch.equal(pagewise[free[5]][:, 63], before[free[3]][:, 8])
    assert torch.equal(pagewise[free[4]][:, 0], before[free[3]][:, 57])


def test_refusals():
    pool, _ = make(10)
    ok = i32([0])
    for call in (lambda: pool.reserve(ok.long(), ok, ok), lambda: pool.reserve(ok, i32([0, 1]), ok), lambda: pool.release(ok.cpu(), ok, ok),
                 lambda: pool.fork(ok, i32([1, 2, 3, 4]).reshape(2, 2)[:, 0], ok), lambda: pool.compact(ok, ok, ok, ok),
                 lambda: pool.compact(ok, ok, ok, torch.zeros((2, 1), dtype=torch.int32, device=DEV)),
                 lambda: pool.compact(ok, ok, ok, torch.zeros((1, 1), dtype=torch.int64, device=DEV)),
                 lambda: pool.copy(ok, ok, i32([1, 2])),
                 lambda: kv_pool.KvPool(pool.arena.to(torch.int32), pool.table, pool.refs, 2, 32, 3, 16),
                 lambda: kv_pool.KvPool(pool.arena, pool.table.long(), pool.refs, 2, 32, 3, 16),
                 lambda: kv_pool.KvPool(pool.arena, pool.table, pool.refs[:-1], 2, 32, 3, 16),
                 lambda: kv_pool.KvPool(pool.arena, pool.table.t(), pool.refs, 2, 32, 3, 16)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(StrideTcError, match="more items"):
        pool.reserve(i32(range(7)), i32([0] * 7), i32([0] * 7))
    empty = i32([])
    pool.reserve(empty, empty, empty)
    pool.fork(empty, empty, empty)
    pool.compact(i32([1]), i32([0]), i32([0]), torch.zeros((1, 0), dtype=torch.int32, device=DEV))
    pool.check()


@pytest.mark.parametrize("count", [1, 3, 70, 5000])
def test_a_kept_position_without_a_page_changes_nothing(count):
    """A position whose page was given up, one before its place, one behind the table, anywhere in
    a short or long list, the other items' lists being right: table, counts and arena are as
    they were, though the call wants fresh pages too."""
    pool, m = make(11, slots=6, max_ctx=6000, pages=900, layers=1, kv_heads=1, pt=16)
    both(pool, m, "reserve", [0, 1, 3], [0, 0, 0], [375, 375, 20])
    both(pool, m, "fork", [1], [4], [5984])  # slot 1's pages are shared
    both(pool, m, "release", [1], [300], [301])
    rng = np.random.default_rng(count)
    held = [t for t in range(40, 6000) if t // 16 != 300]
    good = sorted(rng.choice([t for t in held if t >= 40], count, replace=False).tolist())
    other = [21, 22, 300]
    width = max(count, 3)
    i32row = lambda k: k + [-9] * (width - len(k))
    for at in sorted({0, count // 2, count - 1}):
        for bad, bit in ((4800, kv_pool.MISSING), (4815, kv_pool.MISSING), (20 + at - 1, kv_pool.BAD_KEEP), (6000, kv_pool.BAD_KEEP),
                         (2 ** 31 - 1, kv_pool.BAD_KEEP), (-2 ** 31, kv_pool.BAD_KEEP)):
            keep = list(good)
            keep[at] = bad
            args = i32([0, 1, 3]), i32([20, 20, 20]), i32([3, count, 3]), torch.tensor([i32row(other), i32row(keep), i32row(other)], dtype=torch.int32, device=DEV)
            early = 0 <= bad < 20 + at  # place 20 + at may take positions from there on only
            unchanged(pool, m, kv_pool.BAD_KEEP if early else bit, "compact", *args)
    both(pool, m, "release", [4], [0], [375])  # (fresh pages for 5000 positions would be more than are left)
    compact(pool, m, [0, 1, 3], [20, 20, 20], [other, good, other])


def test_an_empty_list_leaves_a_shared_page():
    """count 0 cuts a sequence off and writes nothing: the page that it ends in stays shared."""
    pool, m = make(12)
    both(pool, m, "reserve", [0], [0], [6])
    both(pool, m, "fork", [0], [1], [96])
    compact(pool, m, [1], [40], [[]])
    assert int(pool.table[1, 2]) == int(pool.table[0, 2]) and pool.table[1, 3:].max() < 0
    compact(pool, m, [1], [40], [[40]])  # a kept position makes it the sequence's own
    assert int(pool.table[1, 2]) != int(pool.table[0, 2])


@pytest.mark.parametrize("how", ["current", "set"])
def test_check_waits_for_the_stream_of_the_calls(how):
    """Calls on a stream that is busy, which is no longer torch's current one, or never was, when
    check and free_pages ask."""
    pool, _ = make(13, slots=4, max_ctx=96, pages=30)
    slot, lo, hi, bad = i32([1]), i32([0]), i32([6]), i32([9])
    a = torch.ones((4096, 4096), device=DEV)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for call, refused, want in ((lambda: pool.reserve(slot, lo, hi), False, 24), (lambda: pool.reserve(bad, lo, hi), True, 24),
                                (lambda: pool.release(slot, lo, hi), False, 30)):
        with torch.cuda.stream(stream):
            for _ in range(40):  # some 40 ms of fp32 products
                b = a @ a
            if how == "current":
                call()
        if how == "set":
            tc.set_kernel_stream(stream)
            try:
                call()
            finally:
                tc.set_kernel_stream(None)
        if refused:
            with pytest.raises(StrideTcError, match="outside its bounds"):
                pool.check()
        assert pool.free_pages() == want
        pool.check()
    del b


@pytest.mark.parametrize("page,D", [(16, 64), (64, 128), (8, 32)])
def test_a_step_after_a_pool_had_no_page(page, D):
    """reserve finds too few pages on the device, when the step's other launches are on their way:
    qkv keeps the rows that have a page and writes nowhere else, and window_attention reads
    zeros for the others; check() says so afterwards."""
    n_kv, n_q, layers, H = 2, 4, 2, 256
    pool, m = make(14, slots=3, max_ctx=64 * 4, pages=64 // page + 2, kv_heads=n_kv, D=D, layers=layers, pt=page)
    g = torch.Generator(device=DEV).manual_seed(3)
    pool.reserve(i32([0]), i32([0]), i32([64 // page]))
    pool.check()
    m.reserve([0], [0], [64 // page])
    w = lambda n: (torch.randn((n // 16, H // 16, 16, 16), generator=g, device=DEV) * 0.05).to(torch.bfloat16).view(torch.int16)
    x = (torch.randn((2, H // 16, 16, 16), generator=g, device=DEV)).to(torch.bfloat16).view(torch.int16)
    rope = torch.randn((256, D // 2, 2), generator=g, device=DEV)
    wq, wk, wv = w(n_kv * n_q * D), w(n_kv * D), w(n_kv * D)
    slot = i32([0] * 10 + [1] * 10)
    pos = i32(list(range(10)) + list(range(10)))
    pool.reserve(i32([1, 2]), i32([0, 0]), i32([2, 200 // page]))  # too many: nobody gets one
    q = harness.qkv(wq, wk, wv, x, 20, D, rope, slot, pos, pool.kv, layer=1)
    out = harness.window_attention(q, pool.kv, slot, pos, n_kv, n_q, D, D ** -0.5, layer=1)
    with pytest.raises(StrideTcError, match="fewer pages"):
        pool.check()
    torch.cuda.synchronize()
    got = pool.arena.cpu().numpy().reshape(m.arena.shape)
    kept = np.zeros(m.arena.shape[:-1], dtype=bool)
    for t in range(10):
        kept[m.table[0, t // page], 1, :, :, t % page] = True
    assert np.array_equal(got[~kept], m.arena[~kept]) and not np.array_equal(got[kept], m.arena[kept])
    rows = layout.untile_lanes(out, 20)
    assert rows[:10].any(1).all() and not rows[10:].any()
    full = kv_pool.KvPool.create(3, 256, 100, n_kv, D, layers, page, DEV)  # the same with pages for all
    full.reserve(i32([0, 1]), i32([0, 0]), i32([64 // page, 2]))
    q2 = harness.qkv(wq, wk, wv, x, 20, D, rope, slot, pos, full.kv, layer=1)
    a = harness.window_attention(q2, full.kv, slot, pos, n_kv, n_q, D, D ** -0.5, layer=1)
    assert torch.equal(q, q2) and torch.equal(layout.untile_lanes(a, 20)[:10], rows[:10])
    old = harness.attention(q[:10], pool.kv, slot[:10], pos[:10], n_kv, D, D ** -0.5, layer=1, max_pages=4)
    assert torch.isfinite(layout.untile_lanes(old, 10).view(torch.bfloat16)).all()


def test_compaction_of_more_items_than_threads():
    """1500 lists of up to 40 kept positions, and one bad position in the last of them."""
    pool, m = make(15, slots=2000, max_ctx=64, pages=7000, kv_heads=1, layers=1, D=8, pt=16)
    rng = np.random.default_rng(6)
    slots = rng.permutation(2000)[:1500].tolist()
    both(pool, m, "reserve", slots, [0] * 1500, [4] * 1500)
    first = rng.integers(0, 20, 1500).tolist()
    keep = [sorted(rng.choice(np.arange(f, 64), int(rng.integers(0, 40)), replace=False).tolist()) for f in first]
    both(pool, m, "release", [slots[-1]], [3], [4])
    keep[-1] = [first[-1], 47]
    for bad, bit in ((48, kv_pool.MISSING), (64, kv_pool.BAD_KEEP)):
        rows = keep[:-1] + [[first[-1], bad]]
        unchanged(pool, m, bit, "compact", i32(slots), i32(first), i32([len(k) for k in rows]),
                  torch.tensor([k + [0] * (40 - len(k)) for k in rows], dtype=torch.int32, device=DEV))
    compact(pool, m, slots, first, keep)
