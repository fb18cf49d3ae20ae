"""stride_serve_window_attention against its definition in 64 bits: sights (window, first
tokens, empty), head layouts, pages, lengths from one position on, what lies in masked
places, batch invariance over every form, captured graphs, long caches, refusals.

Tolerance, for an output o = sum w_t v_t with A = sum w_t |v_t| (t over the visible ones):
  the query's 16 bits and the fp32 sums change a score by at most
      e = (2^-16 + 2^-22 (head_dim + 8)) * scale * max_t sum_d |q_d| |k_td|, a weight by a
      factor exp(+-e), and the sum of weights too: together 2 e A (e << 1)
  a weight's rounding to bf16: 2^-8 each, in numerator and denominator: 2 * 2^-8 A
  exp2's last place, fp32 sums over T positions: 2^-20 A is ample for T up to 2^16
  the result's rounding to bf16: 2^-8 (|o| + the above)
"""
import numpy as np
import pytest
import torch

from stride_amd import harness, layout, tc
from stride_amd._lib import StrideTcError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def say(*a):
    print(*a, flush=True)


class Case:
    """A cache of `slots` sequences over shuffled pages, filled with normal values."""

    def __init__(self, seed, slots, ctx, n_kv, n_q, D, page, layers=2, spread=1.25):
        g = self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.n_kv, self.n_q, self.D, self.page, self.layers, self.ctx = n_kv, n_q, D, page, layers, ctx
        mb = -(-ctx // page)
        self.table = torch.randperm(slots * mb, generator=g, device=DEV).reshape(slots, mb).to(torch.int32)
        self.arena = torch.empty((slots * mb, layers, 2, n_kv, page, D), device=DEV, dtype=torch.bfloat16).normal_(generator=g)
        self.spread = spread
        self.kv = harness.PagedKv.over(self.arena.view(torch.int16), self.table, n_kv, D, layers, page)
        self.scale = D ** -0.5

    def queries(self, rows):
        return torch.empty((rows, self.n_kv * self.n_q * self.D), device=DEV).normal_(generator=self.g) * self.spread

    def run(self, q, slot, pos, window=0, sinks=0, layer=1, **kw):
        i = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        return harness.window_attention(q, self.kv, i(slot), i(pos), self.n_kv, self.n_q, self.D, self.scale, window, sinks,
                                        layer=layer, **kw)

    def exact(self, q, slot, pos, window=0, sinks=0, layer=1):
        """(o, tolerance) in 64 bits, [rows][n_kv * n_q * D]."""
        D, out, tol = self.D, [], []
        for j in range(len(slot)):
            p = pos[j]
            t = torch.arange(max(p + 1, 0), device=DEV)
            see = t >= 0
            if window > 0:
                see = (p - t < window) | (t < sinks)
            t = t[see]
            if t.numel() == 0:
                out.append(torch.zeros(self.n_kv, self.n_q, D, dtype=torch.float64, device=DEV))
                tol.append(torch.zeros_like(out[-1]))
                continue
            blocks = self.table[slot[j]].long()[t // self.page]
            kv = self.arena[blocks, layer][torch.arange(t.numel(), device=DEV), :, :, t % self.page].double()  # [T][2][n_kv][D]
            k, v = kv[:, 0].permute(1, 2, 0).contiguous(), kv[:, 1].permute(1, 0, 2).contiguous()
            qj = q[j].double().reshape(self.n_kv, self.n_q, D)
            s = torch.matmul(qj, k) * self.scale
            w = torch.softmax(s, -1)
            o, a = torch.matmul(w, v), torch.matmul(w, v.abs())
            e = (2.0 ** -16 + 2.0 ** -22 * (D + 8)) * self.scale * torch.matmul(qj.abs(), k.abs()).amax(-1, keepdim=True)
            err = (2 * e + 2 * 2.0 ** -8 + 2.0 ** -20) * a
            out.append(o)
            tol.append(err + 2.0 ** -8 * (o.abs() + err) + 1e-30)
        return torch.stack(out).reshape(len(slot), -1), torch.stack(tol).reshape(len(slot), -1)

    def check(self, q, slot, pos, window=0, sinks=0, layer=1, **kw):
        tiles = self.run(q, slot, pos, window, sinks, layer, **kw)
        got = layout.untile_lanes(tiles, len(slot)).view(torch.bfloat16).double()
        want, tol = self.exact(q, slot, pos, window, sinks, layer)
        bad = ~((got - want).abs() <= tol)
        assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, rows {bad.any(1).nonzero()[:4, 0].tolist()}, "
                               f"worst {((got - want).abs() / tol).nan_to_num(1e9).max().item():.2f} of the tolerance")
        return tiles


POSITIONS = [0, 1, 15, 16, 62, 63, 64, 65, 127, 128, 254, 255, 256, 257, 300, 511, 512, 513, 600]


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (64, 4), (65, 0), (200, 300), (256, 1), (257, 64), (4000, 4), (63, 600)])
def test_sights(D, window, sinks):
    say("sights", D, window, sinks)
    c = Case(D + window + sinks, len(POSITIONS), 640, 2, 4, D, 16)
    c.check(c.queries(len(POSITIONS)), list(range(len(POSITIONS))), POSITIONS, window, sinks, runs=1)


@pytest.mark.parametrize("n_kv,n_q", [(1, 1), (1, 16), (3, 5), (8, 2), (2, 7), (1, 3)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_layouts(n_kv, n_q, D):
    if n_kv * n_q * D % 16:
        pytest.skip("columns come in tiles of 16")
    say("heads", n_kv, n_q, D)
    c = Case(n_kv * 100 + n_q, 5, 700, n_kv, n_q, D, 32)
    c.check(c.queries(5), [4, 0, 2, 1, 3], [699, 0, 333, 64, 511], 300, 2)
    c.check(c.queries(5), [4, 0, 2, 1, 3], [699, 0, 333, 64, 511])


@pytest.mark.parametrize("page", [8, 16, 64, 256, 1024])
@pytest.mark.parametrize("window", [0, 100])
def test_pages(page, window):
    say("pages", page, window)
    c = Case(page, 4, 1300, 2, 4, 64, page)
    c.check(c.queries(4), [2, 3, 0, 1], [1299, 1023, 257, 7], window, 3 if window else 0)


@pytest.mark.parametrize("seqs,rows,past", [(1, 2, 0), (1, 33, 0), (1, 130, 70), (3, 40, 250), (2, 65, 500), (5, 7, 300), (40, 3, 90)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4), (300, 0)])
@pytest.mark.parametrize("n_kv,D,n_q", [(2, 64, 4), (2, 128, 8), (2, 32, 1), (2, 64, 3), (16, 64, 4), (16, 128, 3), (16, 32, 2)])
def test_chunks_of_prompts(seqs, rows, past, window, sinks, n_kv, D, n_q):
    """Neighbouring rows of one sequence, and tiles in which several sequences meet."""
    say("chunks", seqs, rows, past, window, sinks, n_kv, D, n_q)
    c = Case(seqs * rows + past, seqs, past + rows, n_kv, n_q, D, 16)
    slot = [s for s in range(seqs) for _ in range(rows)]
    pos = [past + i for _ in range(seqs) for i in range(rows)]
    q = c.queries(len(slot))
    a = c.check(q, slot, pos, window, sinks, runs=rows)
    for runs in (0, 1):
        assert torch.equal(a, c.run(q, slot, pos, window, sinks, runs=runs)), runs


def test_rows_do_not_depend_on_their_batch():
    """Each row alone (split over its leaves), in a small batch, in a batch of hundreds (one
    workgroup a row), as part of its prompt (tiles), in any order: the same bits."""
    for D, n_q, window, sinks in ((64, 4, 0, 0), (64, 4, 333, 4), (128, 4, 0, 0), (128, 7, 500, 40), (32, 16, 100, 0)):
        say("invariance", D, n_q, window, sinks)
        c = Case(D + n_q, 6, 1500, 2, n_q, D, 16)
        slot = [s for s in range(6) for _ in range(120)]
        pos = [1379 - 200 * s + i for s in range(6) for i in range(120)]
        q = c.queries(720)
        base = layout.untile_lanes(c.run(q, slot, pos, window, sinks, runs=120), 720)
        for runs in (0, 1):
            assert torch.equal(base, layout.untile_lanes(c.run(q, slot, pos, window, sinks, runs=runs), 720)), runs
        order = torch.randperm(720, generator=torch.Generator().manual_seed(1)).tolist()
        got = layout.untile_lanes(c.run(q[order].contiguous(), [slot[i] for i in order], [pos[i] for i in order], window, sinks), 720)
        assert torch.equal(got, base[order]), "shuffled"
        for n in (1, 2, 3, 17, 40):
            some = order[:n]
            for runs in (0, 1):
                got = layout.untile_lanes(c.run(q[some].contiguous(), [slot[i] for i in some], [pos[i] for i in some], window, sinks, runs=runs), n)
                assert torch.equal(got, base[some]), (n, runs)
        part = list(range(130, 175))  # a piece of one prompt, cut elsewhere
        got = layout.untile_lanes(c.run(q[part].contiguous(), [slot[i] for i in part], [pos[i] for i in part], window, sinks, runs=45), 45)
        assert torch.equal(got, base[part])


@pytest.mark.parametrize("rows", [1, 5, 300])
def test_larger_capacity_changes_nothing(rows):
    """max_pages (and with it the split and its scratch) is a bound only."""
    c = Case(rows, 4, 2000, 2, 4, 64, 16)
    slot, pos = [i % 4 for i in range(rows)], [(37 * i) % 1900 for i in range(rows)]
    q = c.queries(rows)
    a = c.run(q, slot, pos, max_pages=30)
    assert torch.equal(a, c.run(q, slot, pos))
    assert torch.equal(a, c.run(q, slot, pos, max_pages=1 << 20))


@pytest.mark.parametrize("rows,n_kv", [(1, 2), (40, 2), (40, 16)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_masked_places_have_no_influence(rows, n_kv, poison):
    """Poison in every position that a row must not see: behind it, between sinks and window,
    in released pages; and in its neighbours' sights in the same tile."""
    say("poison", rows, n_kv, poison)
    window, sinks = 90, 3
    c = Case(7, 1, 700, n_kv, 4, 64, 16)
    pos = [560 + i for i in range(rows)]
    q = c.queries(rows)
    clean = c.run(q, [0] * rows, pos, window, sinks)
    see = torch.zeros(704, dtype=torch.bool, device=DEV)
    see[:sinks] = True
    see[pos[0] - window + 1:pos[-1] + 1] = True
    for t in (~see).nonzero()[:, 0].tolist():
        c.arena[int(c.table[0, t // 16]), :, :, :, t % 16] = poison
    assert torch.equal(clean, c.run(q, [0] * rows, pos, window, sinks))
    gone = [b for b in range(44) if not see[16 * b:16 * b + 16].any()]
    c.table[0, gone] = -1
    assert torch.equal(clean, c.run(q, [0] * rows, pos, window, sinks))


@pytest.mark.parametrize("n_kv", [2, 8])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_a_bad_token_reaches_only_the_rows_that_see_it(n_kv, which, poison):
    """A key or value that is not finite: rows before it and rows whose window has passed it
    are as they were, in tiles too, and for those that see it the plain formula decides what is
    not finite."""
    window, sinks, rows, at = 20, 0, 64, 330
    c = Case(8, 1, 500, n_kv, 4, 64, 16)
    pos = [300 + i for i in range(rows)]
    q = c.queries(rows)
    clean = layout.untile_lanes(c.run(q, [0] * rows, pos, window, sinks), rows)
    c.arena[int(c.table[0, at // 16]), 1, which, 1, at % 16, 5] = poison
    got = layout.untile_lanes(c.run(q, [0] * rows, pos, window, sinks, runs=rows), rows)
    sees = torch.tensor([at <= p < at + window for p in pos], device=DEV)
    assert torch.equal(got[~sees], clean[~sees])
    heads = got.reshape(rows, n_kv, 4, 64).view(torch.bfloat16)
    others = [g for g in range(n_kv) if g != 1]
    assert torch.equal(got.reshape(rows, n_kv, -1)[:, others], clean.reshape(rows, n_kv, -1)[:, others])
    if which == 1:  # a value: its dim alone
        assert torch.isfinite(heads[sees][:, 1, :, :5]).all() and torch.isfinite(heads[sees][:, 1, :, 6:]).all()
        assert not torch.isfinite(heads[sees][:, 1, :, 5]).any()
        if poison != poison:
            assert torch.isnan(heads[sees][:, 1, :, 5]).all()
        else:
            assert (heads[sees][:, 1, :, 5] == poison).all()
    elif poison != poison:  # a key: every dim of its heads
        assert torch.isnan(heads[sees][:, 1]).all()
    else:  # a score of +inf takes inf - inf, one of -inf is a weight of 0
        sign = torch.sign(q.reshape(rows, n_kv, 4, 64)[sees][:, 1, :, 5]) * (1 if poison > 0 else -1)
        assert torch.isnan(heads[sees][:, 1][sign > 0]).all() and torch.isfinite(heads[sees][:, 1][sign < 0]).all()
    for j in range(rows):  # and the same bits, or the same kind of value, row by row
        one = layout.untile_lanes(c.run(q[j:j + 1], [0], [pos[j]], window, sinks), 1)[0]
        a, b = one.view(torch.bfloat16), got[j].view(torch.bfloat16)
        assert torch.equal(a.nan_to_num(7e7), b.nan_to_num(7e7)), j


def test_a_bad_token_where_two_prompts_meet():
    """A tile of two sequences, the bad value in either, at an edge: its part alone is done
    another way, and no other row changes."""
    for at_slot in (0, 1):
        c = Case(20 + at_slot, 2, 400, 8, 4, 64, 16)
        slot = [0] * 80 + [1] * 80
        pos = [200 + i for i in range(80)] + [300 + i for i in range(80)]
        q = c.queries(160)
        clean = layout.untile_lanes(c.run(q, slot, pos, 150, 4, runs=80), 160)
        at = (230, 330)[at_slot]
        c.arena[int(c.table[at_slot, at // 16]), 1, 1, 3, at % 16, 40] = float("inf")
        got = layout.untile_lanes(c.run(q, slot, pos, 150, 4, runs=80), 160)
        touched = torch.tensor([s == at_slot and p >= at for s, p in zip(slot, pos)], device=DEV)
        assert torch.equal(got[~touched], clean[~touched])
        heads = got.reshape(160, 8, 4, 64).view(torch.bfloat16)
        assert torch.isinf(heads[touched][:, 3, :, 40]).all()
        heads[:, 3, :, 40] = clean.reshape(160, 8, 4, 64).view(torch.bfloat16)[:, 3, :, 40]
        assert torch.equal(heads.view(torch.int16).reshape(160, -1), clean)


@pytest.mark.parametrize("D,n_q", [(32, 1), (64, 4), (64, 3), (128, 8)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2100, 300), (2050, 0)])
@pytest.mark.parametrize("lengths", [(4,), (33,), (40, 25, 3, 30), (130, 7)])
def test_short_prompts_on_long_caches(D, n_q, window, sinks, lengths):
    """Few rows of few sequences over many leaves: tiles whose leaves are split among
    workgroups, short runs in them left to rows; one lane without a sequence, one with no
    position, capacities that change the split, and every row alone."""
    say("split tiles", D, n_q, window, sinks, lengths)
    c = Case(D + sum(lengths), len(lengths), 2900, 3, n_q, D, 16)
    slot = [s for s, n in enumerate(lengths) for _ in range(n)]
    pos = [(2899, 2600, 2304, 2047)[s] - n + 1 + i for s, n in enumerate(lengths) for i in range(n)]
    rows = len(slot)
    q = c.queries(rows)
    tiles = c.check(q, slot, pos, window, sinks, runs=max(lengths))
    a = layout.untile_lanes(tiles, rows)
    for runs in (0, 1, 2, rows):
        assert torch.equal(tiles, c.run(q, slot, pos, window, sinks, runs=runs)), runs
    assert torch.equal(tiles, c.run(q, slot, pos, window, sinks, runs=rows, max_pages=1 << 20))
    for j in (0, rows // 2, rows - 1):
        assert torch.equal(layout.untile_lanes(c.run(q[j:j + 1], [slot[j]], [pos[j]], window, sinks), 1)[0], a[j]), j
    slot[1], pos[2] = -1, -1
    got = layout.untile_lanes(c.run(q, slot, pos, window, sinks, runs=rows), rows)
    assert not got[1:3].any()
    keep = [j for j in range(rows) if j not in (1, 2)]
    assert torch.equal(got[keep], a[keep])


@pytest.mark.parametrize("D,n_q,each", [(64, 4, 8), (64, 4, 5), (128, 4, 4), (32, 1, 11), (64, 16, 4)])
@pytest.mark.parametrize("runs", [0, 1, 2])
def test_a_bad_token_where_many_prompts_meet(D, n_q, each, runs):
    """Tiles of several short runs, which workgroups take in turn: a bad value that only some
    rows of one prompt see makes that prompt's rows alone another way's work."""
    say("many prompts", D, n_q, each, runs)
    seqs = 24
    c = Case(D + each, seqs, 500, 2, n_q, D, 16)
    slot = [s for s in range(seqs) for _ in range(each)]
    pos = [300 + 7 * s + i for s in range(seqs) for i in range(each)]
    rows = len(slot)
    q = c.queries(rows)
    hint = (0, each, 1)[runs]
    clean = layout.untile_lanes(c.check(q, slot, pos, 130, 2, runs=hint), rows)
    assert torch.equal(clean, layout.untile_lanes(c.run(q, slot, pos, 130, 2, runs=1), rows))
    bad = {5: 300 + 35 + 2, 6: 300 + 42 + each, 13: 300 + 91 - 129, 20: 1}
    for s, at in bad.items():
        c.arena[int(c.table[s, at // 16]), 1, 1, 1, at % 16, 9] = float("inf")
    got = layout.untile_lanes(c.run(q, slot, pos, 130, 2, runs=hint), rows)
    sees = torch.tensor([s in bad and bad[s] <= p and (p - bad[s] < 130 or bad[s] < 2) for s, p in zip(slot, pos)], device=DEV)
    heads, was = (x.reshape(rows, 2, n_q, D).view(torch.bfloat16) for x in (got, clean))
    assert torch.isinf(heads[sees][:, 1, :, 9]).all() and torch.equal(got[~sees], clean[~sees])
    heads[:, 1, :, 9] = was[:, 1, :, 9]
    assert torch.equal(heads.view(torch.int16).reshape(rows, -1), clean)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("at", [5, 700, 2795, 2799])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_a_bad_token_on_a_long_cache(D, at, poison):
    """A bad value in one leaf of split tiles: among the sinks, where only some rows' windows
    begin, where only some rows end. Their leaves alone are done another way."""
    window, sinks, rows = 2101, 4, 30
    c = Case(30, 1, 2900, 3, 4, D, 16)
    pos = [2775 + i for i in range(rows)]
    q = c.queries(rows)
    clean = layout.untile_lanes(c.run(q, [0] * rows, pos, window, sinks, runs=rows), rows)
    c.arena[int(c.table[0, at // 16]), 1, 1, 2, at % 16, 7] = poison
    got = layout.untile_lanes(c.run(q, [0] * rows, pos, window, sinks, runs=rows), rows)
    sees = torch.tensor([at <= p < at + window for p in pos], device=DEV)
    heads, was = (x.reshape(rows, 3, 4, D).view(torch.bfloat16) for x in (got, clean))
    assert not torch.isfinite(heads[sees][:, 2, :, 7]).any() and torch.equal(got[~sees], clean[~sees])
    heads[:, 2, :, 7] = was[:, 2, :, 7]
    assert torch.equal(heads.view(torch.int16).reshape(rows, -1), clean)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("rows,ctx,window", [(40, 500, 0), (40, 500, 100), (30, 2900, 0), (300, 900, 77)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_a_bad_query_reaches_only_its_head(D, rows, ctx, window, poison):
    """Tiles in which one head's scores are not finite: it alone is NaN, the others are as they were."""
    say("query", D, rows, ctx, window, poison)
    c = Case(D + rows, 1, ctx, 2, 4, D, 16)
    pos = [ctx - rows + i for i in range(rows)]
    q = c.queries(rows)
    clean = layout.untile_lanes(c.run(q, [0] * rows, pos, window, 0, runs=rows), rows).reshape(rows, 8, D)
    q[rows // 2, 5 * D + 3] = poison
    got = layout.untile_lanes(c.run(q, [0] * rows, pos, window, 0, runs=rows), rows).reshape(rows, 8, D)
    assert torch.isnan(got[rows // 2, 5].view(torch.bfloat16)).all()
    got[rows // 2, 5] = clean[rows // 2, 5]
    assert torch.equal(got, clean)


def test_large_scores():
    """Scores that outrun exp's range, rising and falling along the cache, and weights that
    underflow: the references follow."""
    for D in (64, 128):
        c = Case(9, 3, 1200, 1, 4, D, 16, spread=1.0)
        ramp = torch.linspace(-60, 60, 1200, device=DEV)
        for s, r in enumerate((ramp, -ramp, ramp[torch.randperm(1200, generator=c.g, device=DEV)])):
            for t in range(1200):
                c.arena[int(c.table[s, t // 16]), 1, 0, 0, t % 16] = 0
            blocks = c.table[s].long()[torch.arange(1200, device=DEV) // 16]
            c.arena[blocks, 1, 0, 0, torch.arange(1200, device=DEV) % 16, 0] = r.to(torch.bfloat16)
        q = torch.zeros((3, 4 * D), device=DEV)
        q.view(3, 4, D)[:, :, 0] = torch.tensor([1.0, 8.0, -8.0, 100.0], device=DEV) / c.scale
        for slot in ([0, 1, 2], [2, 2, 0]):
            c.check(q, slot, [1199, 1150, 700])
        a = layout.untile_lanes(c.run(q, [0, 1, 2], [1199, 1150, 700]), 3)
        for j, (s, p) in enumerate(((0, 1199), (1, 1150), (2, 700))):
            rows = 40
            got = c.run(q[j:j + 1].expand(rows, -1).contiguous(), [s] * rows, [p] * rows, runs=rows)
            assert (layout.untile_lanes(got, rows) == a[j]).all()


def test_empty_rows_and_lanes_behind():
    c = Case(10, 3, 400, 2, 4, 64, 16)
    for rows, runs in ((5, 1), (5, 0), (37, 37)):
        q = c.queries(rows)
        q[1] = float("nan")
        pos = [-1 if i % 5 in (1, 4) else 100 + i for i in range(rows)]
        slot = [2] * rows
        out = torch.full(((rows + 15) // 16, 32, 16, 16), 0x1234, dtype=torch.int16, device=DEV)
        c.run(q, slot, pos, 0, 0, out_tiles=out, runs=runs)
        got = layout.untile_lanes(out, rows)
        for j in range(rows):
            if pos[j] < 0:
                assert not got[j].any()
        want, tol = c.exact(q, slot, pos)
        live = torch.tensor([p >= 0 for p in pos], device=DEV)
        assert ((got.view(torch.bfloat16).double() - want).abs() <= tol)[live].all()
        behind = layout.untile_lanes(out, (rows + 15) // 16 * 16)[rows:]
        assert (behind == 0x1234).all()


def test_rows_of_all_infinite_scores_are_empty():
    c = Case(11, 1, 100, 1, 4, 64, 16)
    c.arena[:, 1, 0] = 0
    c.arena[:, 1, 0, :, :, 0] = -float("inf")
    q = torch.zeros((2, 256), device=DEV)
    q.view(2, 4, 64)[:, :, 0] = 1.0
    assert not c.run(q, [0, 0], [0, 99]).any()


def test_strides_and_layers():
    c = Case(12, 2, 300, 2, 4, 64, 16, layers=3)
    wide = torch.full((9, 1024), float("nan"), device=DEV)
    q = c.queries(9)
    wide[:, 256:768] = q
    slot, pos = [0, 1] * 4 + [0], [290 - i for i in range(9)]
    for layer in (0, 1, 2):
        a = c.check(q, slot, pos, layer=layer)
        assert torch.equal(a, c.run(wide[:, 256:768], slot, pos, layer=layer))


def test_position_past_the_capacity_is_cut():
    """row_pos beyond the table, or beyond max_pages, reads nothing behind it."""
    c = Case(13, 2, 256, 1, 4, 64, 16)
    q = c.queries(2)
    a = c.run(q, [0, 1], [255, 255])
    assert torch.equal(a, c.run(q, [0, 1], [256, 2 ** 31 - 1]))
    assert torch.equal(c.run(q, [0, 1], [127, 127], 50), c.run(q, [0, 1], [200, 2 ** 30], 50, max_pages=2))


def test_cache_past_32_bits():
    """Pages whose elements lie beyond 2^31 and 2^32 from the arena's start."""
    n_kv, D, page = 8, 128, 64
    per = 2 * n_kv * page * D
    pages = (2 ** 32 + 2 ** 28) // per
    say("long cache", pages, "pages", pages * per * 2 / 2 ** 30, "GiB")
    c = Case(14, 1, 640, n_kv, 2, D, page, layers=1)
    arena = torch.empty(pages * per, dtype=torch.int16, device=DEV)
    high = [pages - 1 - 3 * i for i in range(5)] + [2 ** 31 // per, 2 ** 31 // per - 1, 2 ** 32 // per, 2 ** 32 // per - 1, 0]
    for i, b in enumerate(high):
        arena[b * per:(b + 1) * per] = c.arena[int(c.table[0, i])].view(torch.int16).reshape(-1)
    kv = harness.PagedKv.over(arena, torch.tensor([high], dtype=torch.int32, device=DEV), n_kv, D, 1, page)
    for rows in (1, 70):
        q = c.queries(rows)
        slot, pos = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.arange(639 - rows + 1, 640, dtype=torch.int32, device=DEV)
        a = harness.window_attention(q, c.kv, slot, pos, n_kv, 2, D, c.scale)
        assert torch.equal(a, harness.window_attention(q, kv, slot, pos, n_kv, 2, D, c.scale))


def test_captured_and_replayed():
    """A captured call follows its device arguments; two graphs with a scratch each; eager
    calls and synchronizations in between."""
    c = Case(15, 4, 1200, 2, 4, 64, 16)
    for rows, window in ((2, 0), (4, 300), (100, 0)):
        slot = torch.tensor([i % 4 for i in range(rows)], dtype=torch.int32, device=DEV)
        pos = torch.zeros(rows, dtype=torch.int32, device=DEV)
        q = c.queries(rows)
        out = torch.zeros(((rows + 15) // 16, 32, 16, 16), dtype=torch.int16, device=DEV)
        scratch = harness.window_attention_scratch(rows, 2, 4, 64, window, 2, 19, DEV)
        call = lambda o, s: harness.window_attention(q, c.kv, slot, pos, 2, 4, 64, c.scale, window, 2, layer=1, out_tiles=o, scratch=s)
        call(out, scratch)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(out, scratch)
        for k in range(4):
            pos.copy_(torch.tensor([(300 * k + 17 * i) % 1200 for i in range(rows)], dtype=torch.int32))
            q.copy_(c.queries(rows))
            want = call(torch.zeros_like(out), harness.window_attention_scratch(rows, 2, 4, 64, window, 2, 19, DEV))
            torch.cuda.synchronize()
            out.fill_(0x5555)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(layout.untile_lanes(out, rows), layout.untile_lanes(want, rows)), (rows, k)


def test_two_streams():
    c = Case(16, 2, 2000, 2, 4, 64, 16)
    q = c.queries(2)
    want = [c.run(q[i:i + 1], [i], [1999]) for i in range(2)]
    slots = [torch.tensor([i], dtype=torch.int32, device=DEV) for i in range(2)]
    pos = torch.tensor([1999], dtype=torch.int32, device=DEV)
    streams, outs, works = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for i in range(2):
        outs.append(torch.zeros((1, 32, 16, 16), dtype=torch.int16, device=DEV))
        works.append(harness.window_attention_scratch(1, 2, 4, 64, 0, 0, 32, DEV))
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                harness.window_attention(q[i:i + 1], c.kv, slots[i], pos, 2, 4, 64, c.scale, layer=1, out_tiles=outs[i], scratch=works[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i], want[i])


def test_refusals():
    c = Case(17, 2, 128, 2, 4, 64, 16)
    q = c.queries(2)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    call = lambda **kw: harness.window_attention(**{**dict(q=q, kv=c.kv, row_slot=i32(0, 1), row_pos=i32(5, 6), n_kv=2, n_q=4,
                                                           head_dim=64, scale=0.125), **kw})
    call()
    for kw in (dict(q=q.double()), dict(q=q[:, :256]), dict(q=q.t().contiguous().t()), dict(q=q[0]), dict(row_slot=i32(0)),
               dict(row_pos=i32(0)), dict(row_slot=i32(0, 1).long()), dict(row_pos=torch.zeros((2, 2), dtype=torch.int32, device=DEV)[:, 0]),
               dict(layer=2), dict(layer=-1), dict(n_kv=1, n_q=8), dict(out_tiles=torch.zeros((1, 16, 16, 16), dtype=torch.int16, device=DEV)),
               dict(out_tiles=torch.zeros((1, 32, 16, 16), device=DEV)), dict(scratch=torch.zeros(8, dtype=torch.float64, device=DEV)),
               dict(q=q.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            call(**kw)
    with pytest.raises(StrideTcError, match="sinks"):
        call(sinks=-1, scratch=torch.zeros(8, device=DEV))
    big = Case(18, 1, 1024, 1, 1, 64, 16)
    with pytest.raises(StrideTcError, match="scratch"):
        harness.window_attention(big.queries(1), big.kv, i32(0), i32(900), 1, 1, 64, 0.125, scratch=torch.zeros(16, device=DEV))
    tc.set_kernel_stream(torch.cuda.current_stream().cuda_stream)
    try:
        with pytest.raises(ValueError, match="scratch"):
            call()
    finally:
        tc.set_kernel_stream(None)


def test_no_rows():
    c = Case(19, 1, 64, 2, 4, 64, 16)
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert harness.window_attention(torch.zeros((0, 512), device=DEV), c.kv, e, e, 2, 4, 64, 0.125).numel() == 0


def test_arguments_of_another_device():
    """Each argument in host memory is refused before anything is launched."""
    c = Case(19, 2, 128, 2, 4, 64, 16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    good = dict(q=c.queries(2), kv=c.kv, row_slot=i32(0, 1), row_pos=i32(5, 6), n_kv=2, n_q=4, head_dim=64, scale=0.125,
                out_tiles=torch.zeros((1, 32, 16, 16), dtype=torch.int16, device=DEV), scratch=torch.zeros(4096, device=DEV))
    harness.window_attention(**good)
    host = dict(kv=harness.PagedKv.over(c.arena.view(torch.int16).cpu(), c.table.cpu(), 2, 64, 2, 16))
    for name in ("q", "row_slot", "row_pos", "out_tiles", "scratch"):
        host[name] = good[name].cpu()
    for name, value in host.items():
        with pytest.raises(ValueError, match="device"):
            harness.window_attention(**{**good, name: value})


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("kind", ["pairs", "mixed", "bad value"])
def test_units_that_share_a_workgroup(D, kind):
    """More rows that tiles leave than workgroups, so that each does several, of several leaves:
    hundreds of short runs; a prompt's chunk beside a large decode batch; tiles whose sums are
    not finite. The bits of the rows form, whose workgroups have one each."""
    n_kv, window, sinks = 8, 0, 0
    if kind == "pairs":
        seqs, each, first = 300, [2] * 300, lambda s: 990 + s % 50
    elif kind == "mixed":
        seqs, each, first = 241, [64] + [1] * 240, lambda s: 700 + 3 * (s % 100)
    else:
        seqs, each, first, window, sinks = 1, [300], lambda s: 740, 500, 3
    say("units", D, kind)
    c = Case(D + seqs, seqs, 1050, n_kv, 4, D, 16, layers=2)
    slot = [s for s in range(seqs) for _ in range(each[s])]
    pos = [first(s) + i for s in range(seqs) for i in range(each[s])]
    rows = len(slot)
    q = c.queries(rows)
    if kind == "bad value":  # in every group, seen by the earlier rows only
        c.arena[int(c.table[0, 300 // 16]), 1, 1, :, 300 % 16, 9] = float("inf")
    hint = {"pairs": 0, "mixed": 64, "bad value": rows}[kind]
    plain = c.run(q, slot, pos, window, sinks, runs=1)
    for _ in range(3):
        got = c.run(q, slot, pos, window, sinks, runs=hint)
        assert torch.equal(got, plain)
    some = list(range(0, rows, 37))
    if kind != "bad value":
        want, tol = c.exact(q[some], [slot[j] for j in some], [pos[j] for j in some], window, sinks)
        assert ((layout.untile_lanes(got, rows)[some].view(torch.bfloat16).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("seqs,each,ctx,n_kv,n_q,D", [(3, 62, 1969, 8, 4, 128), (4, 55, 1953, 8, 1, 32), (1, 64, 2900, 8, 4, 64), (2, 2, 500, 2, 4, 64)])
def test_a_scratch_sized_without_a_hint(seqs, each, ctx, n_kv, n_q, D):
    """One scratch of the size for "not known" serves a call with each hint, with the same bits."""
    c = Case(seqs * each, seqs, ctx, n_kv, n_q, D, 32)
    slot = [s for s in range(seqs) for _ in range(each)]
    pos = [ctx - each + i for _ in range(seqs) for i in range(each)]
    q = c.queries(len(slot))
    scratch = harness.window_attention_scratch(len(slot), n_kv, n_q, D, 0, 0, -(-ctx // 64), DEV)
    plain = c.run(q, slot, pos, runs=1)
    for runs in (0, 1, 2, 4, each, seqs * each, 1000):
        assert torch.equal(plain, c.run(q, slot, pos, runs=runs, scratch=scratch)), runs


@pytest.mark.parametrize("D,n_q", [(32, 2), (64, 4), (128, 7)])
@pytest.mark.parametrize("window,sinks,runs", [(64, 0, 40), (64, 20, 0), (600, 3, 80), (2100, 4, 80), (2060, 0, 120)])
def test_rows_of_one_sequence_far_apart(D, n_q, window, sinks, runs):
    """Two pieces of one sequence's rows in one tile, and pages between their windows that are
    gone or belong to others: no row sees them, and nothing changes."""
    say("far apart", D, n_q, window, sinks, runs)
    c = Case(D + window, 1, 5100, 2, n_q, D, 16)
    pos = list(range(10, 50)) + list(range(5040, 5080))
    slot, q = [0] * 80, c.queries(80)
    clean = c.check(q, slot, pos, window, sinks, runs=runs)
    assert torch.equal(clean, c.run(q, slot, pos, window, sinks, runs=1))
    see = torch.zeros(5104, dtype=torch.bool)
    for p in pos:
        see[max(0, p - window + 1):p + 1] = True
        see[:min(sinks, p + 1)] = True
    gone = [b for b in range(5100 // 16 + 1) if not see[16 * b:16 * b + 16].any()]
    assert len(gone) > 100
    for b in gone:
        c.arena[int(c.table[0, b])] = float("nan")
    assert torch.equal(clean, c.run(q, slot, pos, window, sinks, runs=runs))
    c.table[0, gone[::2]] = -1
    c.table[0, gone[1::2]] = c.table[0, 0].clone()
    assert torch.equal(clean, c.run(q, slot, pos, window, sinks, runs=runs))
    order = [j // 2 + 40 * (j % 2) for j in range(80)]  # and where they take turns
    got = c.run(q[order].contiguous(), slot, [pos[j] for j in order], window, sinks, runs=runs)
    assert torch.equal(layout.untile_lanes(got, 80), layout.untile_lanes(clean, 80)[order])


@pytest.mark.parametrize("rows,window", [(3, 0), (3, 50), (40, 50), (40, 0)])
def test_any_negative_position_is_none(rows, window):
    c = Case(21, 1, 300, 2, 4, 64, 16)
    q = c.queries(rows)
    pos = [200 + j for j in range(rows)]
    clean = layout.untile_lanes(c.run(q, [0] * rows, pos, window, 0), rows)
    for none in (-1, -2, -2 ** 31):
        pos[1] = none
        got = layout.untile_lanes(c.run(q, [0] * rows, pos, window, 0), rows)
        assert not got[1].any()
        assert torch.equal(got[[0] + list(range(2, rows))], clean[[0] + list(range(2, rows))])


def test_results_are_not_allocated_on_another_stream():
    """With a stream of set_kernel_stream's that is not torch's current one, what a runner would
    allocate would be filled beside the launch: it is to be passed."""
    c = Case(22, 2, 300, 2, 4, 64, 16)
    q, i = c.queries(3), torch.tensor([0, 1, 1], dtype=torch.int32, device=DEV)
    pos = torch.tensor([250, 3, 299], dtype=torch.int32, device=DEV)
    call = lambda **kw: harness.window_attention(q, c.kv, i, pos, 2, 4, 64, c.scale, layer=1, **kw)
    want = call()
    out, scratch = torch.zeros_like(want), torch.empty(1 << 20, device=DEV)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    tc.set_kernel_stream(stream)
    try:
        with pytest.raises(ValueError, match="out_tiles"):
            call(scratch=scratch)
        call(out_tiles=out, scratch=scratch)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        tc.set_kernel_stream(torch.cuda.current_stream())
        assert torch.equal(call(scratch=scratch), want)
    finally:
        tc.set_kernel_stream(None)
