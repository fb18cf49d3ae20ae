"""stride_amd.logits against NumPy: each step of the formula is one fp32 operation, so the
processed logits and the choice are equal bit for bit; counts; capture; refusals."""
import numpy as np
import pytest
import torch

from stride_amd import harness, layout, logits, synth, tc
from stride_amd._lib import StrideTcError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = np.float32(np.inf)


def say(*a):
    print(*a, flush=True)


def tiles_of(a, rows_padded=None):
    """[rows][vocab] fp32 -> lm_full's tiles; padding lanes and rows hold 77."""
    rows, vocab = a.shape
    T, rt = -(-rows // 16), -(-vocab // 16)
    wide = np.full((T * 16, rt * 16), 77, np.float32)
    wide[:rows, :vocab] = a
    return torch.from_numpy(np.ascontiguousarray(wide.reshape(T, 16, rt, 16).transpose(2, 0, 3, 1))).to(DEV)


def plain(l, word=None, pen=None, bias=None, allowed=None):
    """fp32 [rows][vocab] -> processed, (values, tokens)."""
    l = l.astype(np.float32).copy()
    with np.errstate(all="ignore"):
        if word is not None:
            n = (word & 0x7FFFFFFF).astype(np.float32)
            rep, pres, freq = (pen[:, k:k + 1].astype(np.float32) for k in range(3))
            l = np.where(word != 0, np.where(l > 0, l / rep, l * rep), l)
            l = np.where(n > 0, (l - freq * n) - pres, l)
        for j, d in enumerate(bias or []):
            for t, b in (d or {}).items():
                l[j, t] = l[j, t] + np.float32(b)
    if allowed is not None:
        l = np.where(allowed, l, -INF)
    best = np.where(np.isnan(l), -INF, l).max(1)
    index = np.array([int(np.flatnonzero(l[j] == best[j])[0]) if best[j] > -INF else -1 for j in range(l.shape[0])], np.int32)
    return l, best, index


def equal(a, b):
    """The same values (NaN as NaN, the zeros as one)."""
    assert np.array_equal(np.nan_to_num(a, nan=1e30) + 0.0, np.nan_to_num(b, nan=1e30) + 0.0) and np.array_equal(np.isnan(a), np.isnan(b))


def history(rng, slots, vocab, tokens):
    word = np.zeros((slots, vocab), np.int64)
    for s in range(slots):
        for t in rng.integers(0, vocab, tokens) // rng.integers(1, 20):
            word[s, t] += 1
        word[s, rng.integers(0, vocab, tokens)] |= 1 << 31
    return word


def counts_of(word):
    c = torch.from_numpy(np.where(word >= 1 << 31, word - (1 << 32), word).astype(np.int32)).to(DEV)
    return logits.TokenCounts(c, logits.pack_mask(word != 0, DEV))


@pytest.mark.parametrize("rows", [1, 3, 16, 17, 40])
@pytest.mark.parametrize("vocab", [1, 15, 31, 32, 33, 500, 511, 513, 5000, 32003])
def test_all_together(rows, vocab):
    say("logits", rows, vocab)
    rng = np.random.default_rng(rows * 100000 + vocab)
    l = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    l[:, rng.integers(0, vocab, 3)] = 0.0
    word = history(rng, rows + 2, vocab, 60)
    slot = rng.permutation(rows + 2)[:rows].astype(np.int32)
    pen = np.stack([1 + rng.random(rows), rng.standard_normal(rows), rng.random(rows)], 1).astype(np.float32)
    bias = [None if j % 3 == 0 else {int(t): float(np.float32(b)) for t, b in zip(rng.integers(0, vocab, 400 if j % 4 == 1 else 20), rng.standard_normal(400))}
            for j in range(rows)]
    masks = rng.random((3, vocab)) < np.array([0.02, 0.5, 0.98])[:, None]
    which = rng.integers(-1, 3, rows).astype(np.int32)
    allowed = np.where((which < 0)[:, None], True, masks[np.maximum(which, 0)])
    want, value, index = plain(l, word[slot], pen, bias, allowed)
    counts = counts_of(word)
    t = tiles_of(l)
    out = torch.full_like(t, 55.0)
    args = dict(counts=counts, row_slot=torch.from_numpy(slot).to(DEV), penalties=torch.from_numpy(pen).to(DEV),
                bias=logits.bias_lists(bias, DEV), mask=logits.pack_mask(masks, DEV), mask_row=torch.from_numpy(which).to(DEV))
    for k in range(3):  # with the processed logits, without them, and in place
        work = logits.scratch(rows, DEV)
        best = logits.process(t, rows, vocab, out=(out, None, t)[k], work=work, **args)
        v, i = harness.best_split(best)
        equal(v.numpy(), value)
        assert np.array_equal(i.numpy(), index)
        assert not work.any()
        if k != 1:
            got = layout.untile_logits((out, None, t)[k], rows, vocab).cpu().numpy()
            equal(got, want)
    pad = layout.untile_logits(out, out.shape[1] * 16, out.shape[0] * 16).cpu().numpy().copy()
    pad[:rows, :vocab] = 55.0
    assert (pad == 55.0).all(), "places behind the rows and the vocabulary are left alone"


@pytest.mark.parametrize("have", [(), ("counts",), ("bias",), ("mask",), ("counts", "mask"), ("bias", "mask")])
def test_each_alone(have):
    rng = np.random.default_rng(len(have))
    rows, vocab = 21, 3000
    l = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    word, pen, bias, allowed, args = None, None, None, None, {}
    if "counts" in have:
        word = history(rng, rows, vocab, 200)
        pen = np.tile(np.array([[1.3, 0.4, 0.2]], np.float32), (rows, 1))
        args.update(counts=counts_of(word), row_slot=torch.arange(rows, dtype=torch.int32, device=DEV), penalties=torch.from_numpy(pen).to(DEV))
    if "bias" in have:
        bias = [{int(t): 1.5 for t in rng.integers(0, vocab, 30)} for _ in range(rows)]
        args.update(bias=logits.bias_lists(bias, DEV))
    if "mask" in have:
        masks = rng.random((2, vocab)) < 0.1
        allowed = masks[np.arange(rows) % 2]
        args.update(mask=logits.pack_mask(masks, DEV), mask_row=(torch.arange(rows, device=DEV) % 2).to(torch.int32))
    want, value, index = plain(l, word, pen, bias, allowed)
    t = tiles_of(l)
    out = torch.zeros_like(t)
    v, i = harness.best_split(logits.process(t, rows, vocab, out=out, **args))
    equal(layout.untile_logits(out, rows, vocab).cpu().numpy(), want)
    equal(v.numpy(), value)
    assert np.array_equal(i.numpy(), index)


def test_nothing_allowed_ties_and_values_that_are_not_finite():
    rows, vocab = 8, 2000
    rng = np.random.default_rng(0)
    l = rng.standard_normal((rows, vocab)).astype(np.float32)
    l[1, [70, 1500, 900]] = 9.0           # a tie: the lowest
    l[2] = -INF
    l[3] = np.nan
    l[4, 33], l[4, 1200] = np.nan, 50.0
    l[5, 1999] = INF
    l[6] = -3.4e38
    l[6, 777] = np.finfo(np.float32).min / 2
    l[7] = -0.0
    l[7, 1234] = 0.0                      # the zeros are equal: token 0
    masks = np.zeros((2, vocab), bool)
    masks[1] = True
    masks[1, 70] = False
    for which in (None, 1, 0):
        kw = {} if which is None else dict(mask=logits.pack_mask(masks, DEV), mask_row=torch.full((rows,), which, dtype=torch.int32, device=DEV))
        _, value, index = plain(l, allowed=None if which is None else np.broadcast_to(masks[which], l.shape))
        v, i = harness.best_split(logits.process(tiles_of(l), rows, vocab, **kw))
        equal(v.numpy(), value)
        assert np.array_equal(i.numpy(), index)
    assert index.tolist() == [-1] * rows


def test_rows_do_not_depend_on_their_batch():
    rng = np.random.default_rng(4)
    vocab = 20000
    l = rng.standard_normal((50, vocab)).astype(np.float32)
    word = history(rng, 50, vocab, 500)
    counts = counts_of(word)
    pen = torch.tensor([[1.2, 0.3, 0.1]], device=DEV).repeat(50, 1)
    slots = torch.arange(50, dtype=torch.int32, device=DEV)
    base = logits.process(tiles_of(l), 50, vocab, counts, slots, pen).cpu()
    for j in (0, 17, 49):
        assert torch.equal(logits.process(tiles_of(l[j:j + 1]), 1, vocab, counts, slots[j:j + 1], pen[j:j + 1]).cpu()[0], base[j])


def test_slots_and_masks_out_of_range_have_none():
    rng = np.random.default_rng(5)
    rows, vocab = 6, 700
    l = rng.standard_normal((rows, vocab)).astype(np.float32)
    counts = counts_of(np.full((2, vocab), 3))
    pen = torch.tensor([[2.0, 1.0, 1.0]], device=DEV).repeat(rows, 1)
    slot = torch.tensor([0, -1, 2, 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    mask = logits.pack_mask(np.zeros((1, vocab), bool), DEV)
    mrow = torch.tensor([-1, -5, 1, 0, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    out = torch.zeros_like(tiles_of(l))
    best = logits.process(tiles_of(l), rows, vocab, counts, slot, pen, mask=mask, mask_row=mrow, out=out)
    word = np.zeros((rows, vocab), np.int64)
    word[[0, 3]] = 3
    allowed = np.ones((rows, vocab), bool)
    allowed[3] = False
    want, value, index = plain(l, word, pen.cpu().numpy(), None, allowed)
    equal(layout.untile_logits(out, rows, vocab).cpu().numpy(), want)
    assert np.array_equal(harness.best_split(best)[1].numpy(), index)


def test_bias_entries_out_of_range_and_equal_neighbours():
    rows, vocab = 2, 300
    l = np.zeros((rows, vocab), np.float32)
    off = torch.tensor([0, 5, 8], dtype=torch.int32, device=DEV)
    tok = torch.tensor([-7, 4, 4, 4, 2 ** 31 - 1, 10, 299, 300], dtype=torch.int32, device=DEV)
    val = torch.tensor([9.0, 1.0, 2.0, 3.0, 9.0, 5.0, 6.0, 9.0], device=DEV)
    out = torch.zeros_like(tiles_of(l))
    logits.process(tiles_of(l), rows, vocab, bias=(off, tok, val), out=out)
    want = l.copy()
    want[0, 4], want[1, 10], want[1, 299] = 3, 5, 6
    equal(layout.untile_logits(out, rows, vocab).cpu().numpy(), want)


def test_counts_record_reset_and_take_over():
    vocab, slots = 1003, 5
    c = logits.TokenCounts.create(slots, vocab, DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    word = np.zeros((slots, vocab), np.int64)
    rng = np.random.default_rng(3)
    for k in range(6):
        n = 300
        s, t = rng.integers(-1, slots + 1, n), rng.integers(-2, vocab + 2, n) // (1 + k)
        prompt = k % 2 == 0
        pairs = torch.stack([i32(t), i32(t)], 1)
        c.record(i32(s), pairs[:, 1] if k % 3 else i32(t), prompt=prompt)
        for a, b in zip(s, t):
            if 0 <= a < slots and 0 <= b < vocab:
                word[a, b] = word[a, b] | (1 << 31) if prompt else word[a, b] + 1
        if k == 3:
            c.reset(i32([4, -1, 9]))
            word[4] = 0
        if k == 4:
            c.reset(i32([0, 2, 4]), i32([1, 1, 7]))
            word[[0, 2]] = word[1]
        assert np.array_equal(c.counts.cpu().numpy().view(np.uint32), word.astype(np.uint32))
        assert torch.equal(c.seen.cpu(), logits.pack_mask(word != 0, "cpu"))
    c.record(i32([]), i32([]))
    c.reset(i32([]))


def test_captured_and_replayed():
    """A decode step's logit work in a graph: the choice enters the counts, and the next replay
    goes by them."""
    rng = np.random.default_rng(6)
    rows, vocab = 19, 4000
    l = rng.standard_normal((rows, vocab)).astype(np.float32)
    t = tiles_of(l)
    word = history(rng, rows, vocab, 50)
    counts = counts_of(word)
    slot = torch.arange(rows, dtype=torch.int32, device=DEV)
    pen = torch.tensor([[1.1, 0.5, 0.75]], device=DEV).repeat(rows, 1)
    best = torch.empty((rows, 2), dtype=torch.int32, device=DEV)
    work = logits.scratch(rows, DEV)

    def step():
        logits.process(t, rows, vocab, counts, slot, pen, best=best, work=work)
        counts.record(slot, best[:, 1])

    other = logits.TokenCounts.create(rows, vocab, DEV)
    logits.process(t, rows, vocab, other, slot, pen)  # eager work with a scratch of its own
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(5):
        graph.replay()
        torch.cuda.synchronize()
        _, value, index = plain(l, word, pen.cpu().numpy())
        v, i = harness.best_split(best)
        equal(v.numpy(), value)
        assert np.array_equal(i.numpy(), index), k
        word[np.arange(rows), index] += 1
        assert np.array_equal(counts.counts.cpu().numpy().view(np.uint32), word.astype(np.uint32))
        logits.process(t, rows, vocab, other, slot, pen)
        torch.cuda.synchronize()


def test_after_lm_full():
    """The same choice as the fused greedy head where nothing is asked for."""
    m, n, k = 37, 4096, 256
    w = layout.pack_tiles(torch.from_numpy(synth.bf16_normal(1, 3, n, k, 0.05).view(np.int16)).to(DEV))
    x = layout.lane_tiles(torch.from_numpy(synth.bf16_normal(1, 4, m, k, 1.0).view(np.int16)).to(DEV))
    best = harness.lm_greedy(w, x, m, 4001)
    assert torch.equal(best, logits.process(harness.lm_full(w, x, m), m, 4001))


def test_refusals():
    l = tiles_of(np.zeros((5, 100), np.float32))
    c = logits.TokenCounts.create(2, 100, DEV)
    slot, pen = torch.zeros(5, dtype=torch.int32, device=DEV), torch.ones((5, 3), device=DEV)
    mask = torch.zeros((1, 4), dtype=torch.int32, device=DEV)
    for kw in (dict(logits=l.double()), dict(logits=l[:, :, :, :8]), dict(logits=l.cpu()), dict(rows=17), dict(vocab=113),
               dict(counts=c), dict(counts=c, row_slot=slot), dict(counts=c, row_slot=slot[:4], penalties=pen),
               dict(counts=c, row_slot=slot.long(), penalties=pen), dict(counts=c, row_slot=slot, penalties=pen[:4]),
               dict(counts=c, row_slot=slot, penalties=pen, vocab=99), dict(mask=mask), dict(mask=mask[:, :3], mask_row=slot),
               dict(mask=mask, mask_row=slot[:2]), dict(bias=(slot[:3], slot, pen[:, 0])), dict(bias=(slot, slot, pen)),
               dict(out=l[:3]), dict(best=torch.zeros((5, 1), dtype=torch.int32, device=DEV)), dict(work=torch.zeros(3, device=DEV))):
        with pytest.raises((ValueError, RuntimeError)):
            logits.process(**{**dict(logits=l, rows=5, vocab=100), **kw})
    for bad in (lambda: logits.TokenCounts(c.counts.long(), c.seen), lambda: logits.TokenCounts(c.counts, c.seen[:, :3]),
                lambda: logits.TokenCounts(c.counts.t(), c.seen), lambda: c.record(slot.long(), slot), lambda: c.record(slot, slot[:3]),
                lambda: c.record(slot.cpu(), slot.cpu()), lambda: c.reset(slot.long())):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    empty = logits.process(torch.zeros((7, 0, 16, 16), device=DEV), 0, 100)
    assert empty.shape == (0, 2)


def test_arguments_of_another_device():
    """Each argument in host memory is refused before anything is launched."""
    l = tiles_of(np.zeros((5, 100), np.float32))
    c = logits.TokenCounts.create(2, 100, DEV)
    slot = torch.zeros(5, dtype=torch.int32, device=DEV)
    good = dict(logits=l, rows=5, vocab=100, counts=c, row_slot=slot, penalties=torch.ones((5, 3), device=DEV),
                bias=logits.bias_lists([{1: 2.0}] * 5, DEV), mask=torch.full((1, 4), -1, dtype=torch.int32, device=DEV), mask_row=slot.clone(),
                out=torch.zeros_like(l), best=torch.zeros((5, 2), dtype=torch.int32, device=DEV), work=logits.scratch(5, DEV))
    logits.process(**good)
    host = {k: v.cpu() for k, v in good.items() if isinstance(v, torch.Tensor)}
    host["counts"] = logits.TokenCounts.create(2, 100, "cpu")
    host["bias"] = tuple(t.cpu() for t in good["bias"])
    for name, value in host.items():
        with pytest.raises(ValueError):
            logits.process(**{**good, name: value})


def test_results_are_not_allocated_on_another_stream():
    """With a stream of set_kernel_stream's that is not torch's current one, best and work are to be passed."""
    l = tiles_of(np.random.default_rng(3).normal(size=(5, 100)).astype(np.float32))
    want = logits.process(l, 5, 100)
    best, work = torch.zeros_like(want), logits.scratch(5, DEV)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    tc.set_kernel_stream(stream)
    try:
        with pytest.raises(ValueError, match="best"):
            logits.process(l, 5, 100, work=work)
        logits.process(l, 5, 100, best=best, work=work)
        torch.cuda.synchronize()
        assert torch.equal(best, want)
        tc.set_kernel_stream(torch.cuda.current_stream())
        assert torch.equal(logits.process(l, 5, 100, work=work), want)
    finally:
        tc.set_kernel_stream(None)
