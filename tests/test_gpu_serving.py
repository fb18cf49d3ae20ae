"""The serving operators together, as stride_amd.serving runs them on a tiny checkpoint: window
attention over a pool's pages that sequences share and give up, and tokens chosen by rules."""
import json
import types

import numpy as np
import pytest
import torch

from stride_amd import cli, engine, harness, layout, logits, serving, tc, weights
from stride_amd.kv_pool import KvPool
import llama_tiny

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def say(*a):
    print(*a, flush=True)


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    path = tmp_path_factory.mktemp("m")
    llama_tiny.write(str(path), seed=5)
    return str(path), weights.Weights.load(str(path), DEV, max_positions=512)


def family(seed, n, longest):
    """Prompts of which many begin alike."""
    rng = np.random.default_rng(seed)
    base = rng.integers(0, 1000, longest).tolist()
    out = []
    for i in range(n):
        keep = int(rng.integers(0, longest))
        out.append((i, base[:keep] + rng.integers(0, 1000, int(rng.integers(1, longest - keep + 1))).tolist()))
    return out


RULES = {0: serving.Rules(1.3, 0.2, 0.1), 2: serving.Rules(bias={5: 3.0, 17: -2.0}), 3: serving.Rules(allowed=range(100, 140)),
         4: serving.Rules(0.8, -0.1, 0.3, {7: 1.0}, range(50))}


def test_ledger_identical_across_scheduling(model, tmp_path):
    """The command's ledger with a window, sinks, penalties, biases and allowed tokens: one
    sequence at a time, and several in a small pool with shared prefixes and shuffled rows."""
    with open(tmp_path / "p.jsonl", "w") as f:
        for pid, tokens in family(1, 9, 120):
            extra = {} if pid % 3 else {"bias": {"5": 2.5}, "allowed": list(range(400))}
            f.write(json.dumps({"id": pid, "tokens": tokens, **extra}) + "\n")
    base = ["--model", model[0], "--input", str(tmp_path / "p.jsonl"), "--max-new", "9", "--path", "serve", "--window", "50", "--sinks",
            "3", "--repetition-penalty", "1.2", "--frequency-penalty", "0.1"]
    out = []
    for k, more in enumerate(([], ["--concurrency", "4", "--max-rows", "24", "--row-shuffle", "5", "--kv-pages", "33", "--share-prefixes"],
                              ["--concurrency", "9", "--max-rows", "300", "--page-tokens", "8", "--share-prefixes"])):
        say("ledger", more)
        assert cli.main([*base, "--output", str(tmp_path / f"{k}.jsonl"), *more]) == 0
        out.append((tmp_path / f"{k}.jsonl").read_text())
    assert out[0] == out[1] == out[2]
    for line in out[0].splitlines():
        rec = json.loads(line)
        assert rec["id"] % 3 or max(rec["tokens"]) < 400


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_attention_of_the_engine(model, monkeypatch, window, sinks):
    """Each layer's call against the formula in 64 bits on the same queries and cache: a score's
    error from queries of 16 bits and sums in fp32, two roundings of a weight, one of the result."""
    w, cfg = model[1], model[1].cfg
    D, real, worst = cfg.head_dim, harness.window_attention, []

    def checked(q, kv, slot, pos, n_kv, n_q, head_dim, scale, win, snk, layer, pages, out_tiles, scratch, runs):
        tiles = real(q, kv, slot, pos, n_kv, n_q, head_dim, scale, win, snk, layer, pages, out_tiles=out_tiles, scratch=scratch, runs=runs)
        rows = q.shape[0]
        got = layout.untile_lanes(tiles, rows).view(torch.bfloat16).double()
        for j in range(0, rows, 7):
            s, p = int(slot[j]), int(pos[j])
            see = [t for t in range(p + 1) if win == 0 or p - t < win or t < snk]
            k, v = (kv.gather(layer, which, [s] * len(see), see, n_kv, D).view(torch.bfloat16).double().reshape(-1, n_kv, D)
                    for which in (0, 1))
            qj = q[j].double().reshape(n_kv, n_q, D)
            x = torch.matmul(qj, k.permute(1, 2, 0).contiguous()) * scale
            vt = v.permute(1, 0, 2).contiguous()
            weight = torch.softmax(x, -1)
            o, a = torch.matmul(weight, vt), torch.matmul(weight, vt.abs())
            e = (2.0 ** -16 + 2.0 ** -22 * (D + 8)) * scale * torch.matmul(qj.abs(), k.abs().permute(1, 2, 0).contiguous()).amax(-1, keepdim=True)
            err = (2 * e + 2 * 2.0 ** -8 + 2.0 ** -20) * a
            tol = err + 2.0 ** -8 * (o.abs() + err) + 1e-30
            worst.append(((got[j] - o.reshape(-1)).abs() / tol.reshape(-1)).max().item())
            assert worst[-1] <= 1, (layer, s, p, worst[-1])
        return tiles

    monkeypatch.setattr(harness, "window_attention", checked)
    todo = family(2, 3, 90)
    eng = serving.ServingEngine(w, 3, 100, 64, window=window, sinks=sinks)
    done = cli.Scheduler(eng, 3, 5, share_prefixes=True).run(todo)
    assert len(done) == 3 and len(worst) > 20


@pytest.mark.parametrize("heads,kv_heads,D", [(2, 2, 32), (6, 2, 64), (8, 1, 64), (16, 1, 32), (4, 2, 128)])
def test_head_layouts_of_the_engine(monkeypatch, heads, kv_heads, D):
    """Models of 1 to 16 query heads a group: each layer's attention against the formula in 64 bits
    (the tolerance of test_attention_of_the_engine), and the same ledger alone and together."""
    cfg = weights.ModelConfig(hidden=256, mlp=512, layers=2, heads=heads, kv_heads=kv_heads, head_dim=D, vocab=1000)
    w = weights.Weights.random(cfg, DEV, seed=heads, max_positions=256)
    n_q, real, worst = heads // kv_heads, harness.window_attention, []

    def checked(q, kv, slot, pos, n_kv, nq, head_dim, scale, win, snk, layer, pages, **kw):
        tiles = real(q, kv, slot, pos, n_kv, nq, head_dim, scale, win, snk, layer, pages, **kw)
        assert (n_kv, nq, head_dim) == (kv_heads, n_q, D)
        got = layout.untile_lanes(tiles, q.shape[0]).view(torch.bfloat16).double()
        for j in range(0, q.shape[0], 5):
            s, p = int(slot[j]), int(pos[j])
            see = [t for t in range(p + 1) if p - t < win or t < snk]
            k, v = (kv.gather(layer, which, [s] * len(see), see, n_kv, D).view(torch.bfloat16).double().reshape(-1, n_kv, D)
                    for which in (0, 1))
            qj = q[j].double().reshape(n_kv, n_q, D)
            kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
            weight = torch.softmax(torch.matmul(qj, kt) * scale, -1)
            o, a = torch.matmul(weight, vt), torch.matmul(weight, vt.abs())
            e = (2.0 ** -16 + 2.0 ** -22 * (D + 8)) * scale * torch.matmul(qj.abs(), kt.abs()).amax(-1, keepdim=True)
            err = (2 * e + 2 * 2.0 ** -8 + 2.0 ** -20) * a
            tol = err + 2.0 ** -8 * (o.abs() + err) + 1e-30
            worst.append(((got[j] - o.reshape(-1)).abs() / tol.reshape(-1)).max().item())
            assert worst[-1] <= 1, (layer, s, p, worst[-1])
        return tiles

    todo = family(heads, 4, 50)
    monkeypatch.setattr(harness, "window_attention", checked)
    alone = cli.Scheduler(serving.ServingEngine(w, 1, 64, 64, window=20, sinks=2), 1, 4).run(todo)
    monkeypatch.undo()
    assert len(worst) > 20
    eng = serving.ServingEngine(w, 4, 64, 24, window=20, sinks=2)
    together = cli.Scheduler(eng, 4, 4, row_shuffle=3, share_prefixes=True).run(todo)
    assert list(cli.ledger_lines(todo, alone)) == list(cli.ledger_lines(todo, together))


def test_rules_that_allow_everything_are_greedy(model):
    w = model[1]
    todo = family(3, 4, 60)
    ledgers = []
    for rules in ({}, {pid: serving.Rules(allowed=range(w.cfg.vocab)) for pid, _ in todo}):
        eng = serving.ServingEngine(w, 4, 80, 64)
        ledgers.append(list(cli.ledger_lines(todo, cli.Scheduler(eng, 4, 8, rules=rules).run(todo))))
    assert ledgers[0] == ledgers[1]


def test_rules_of_the_engine(model, monkeypatch):
    """Every choice against the formula on the step's own logits, with the tokens that the host
    knows the sequence has: at most five roundings of fp32 (a quotient or product, a product,
    three sums), each of a value no larger than the sum of the magnitudes."""
    w, vocab = model[1], model[1].cfg.vocab
    todo, real, state = family(4, 6, 70), logits.process, types.SimpleNamespace(checked=0)
    eng = serving.ServingEngine(w, 6, 90, 64, window=64, sinks=2)
    pid_of, made = {}, {}

    def begin(slot, prompt, rules=None, source=-1, shared=0):
        pid_of[slot] = next(p for p, t in todo if t == prompt)
        made[pid_of[slot]] = []
        serving.ServingEngine.begin(eng, slot, prompt, rules, source, shared)

    def checked(tiles, rows, *args, **kw):
        plain = layout.untile_logits(tiles, rows, vocab).clone()
        best = real(tiles, rows, *args, **kw)
        got = best.cpu()
        for j, slot in enumerate(args[2].tolist()):
            pid = pid_of[slot]
            r, n = RULES.get(pid, serving.Rules()), made[pid]
            l = plain[j].double().cpu().numpy()
            size, has = np.abs(l), np.zeros(vocab, dtype=bool)
            has[todo[pid][1] + n] = True
            times = np.bincount(n, minlength=vocab) if n else np.zeros(vocab)
            rep, pres, freq = (float(np.float32(x)) for x in (r.repetition, r.presence, r.frequency))
            l = np.where(has, np.where(l > 0, l / rep, l * rep), l)
            size = size * max(rep, 1 / rep, 1) + abs(freq) * times + abs(pres)
            l = l - freq * times - pres * (times > 0)
            for t, b in (r.bias or {}).items():
                l[t], size[t] = l[t] + b, size[t] + abs(b)
            tol = 5 * 2.0 ** -24 * size
            if r.allowed is not None:
                off = np.ones(vocab, dtype=bool)
                off[list(r.allowed)] = False
                l[off] = -np.inf
            value, token = float(got[j, 0:1].view(torch.float32)), int(got[j, 1])
            assert abs(value - l[token]) <= tol[token], (pid, token)
            assert l[token] + 2 * tol[token] >= (l - 2 * tol).max(), (pid, token)
            n.append(token)
            state.checked += 1
        return best

    monkeypatch.setattr(logits, "process", checked)
    monkeypatch.setattr(eng, "begin", begin)
    done = cli.Scheduler(eng, 6, 8, rules=RULES, share_prefixes=True).run(todo)
    assert state.checked >= 4 * 8 and all(done[p][0].tokens == made[p] for p in RULES)
    counts = eng.counts.counts.cpu().numpy()
    for slot, pid in pid_of.items():
        if RULES.get(pid, serving.Rules()).counted:
            assert np.array_equal(counts[slot] & 0x7FFFFFFF, np.bincount(done[pid][0].tokens, minlength=vocab))
            assert np.array_equal(np.flatnonzero(counts[slot] < 0), np.unique(todo[pid][1]))


def test_pages_come_back(model):
    eng = serving.ServingEngine(model[1], 3, 300, 32, pages=20, window=33, sinks=1)
    todo = [(i, t * 3) for i, t in family(5, 7, 60)]
    cli.Scheduler(eng, 3, 20, share_prefixes=True).run(todo)
    assert eng.pool.free_pages() == 20 and (eng.pool.table == -1).all() and eng.book.used == 0
    eng.step([(0, p, 1) for p in range(32)], [])
    eng.pool.reserve(*eng._ints([[1], [0], [19]]))  # behind the book's back: more than there is
    with pytest.raises(Exception, match="kv pool"):
        eng.check()


def test_engine_refusals(model):
    eng = serving.ServingEngine(model[1], 2, 64, 16)
    for rows in ([(2, 0, 1)], [(-1, 0, 1)], [(0, 64, 1)], [(0, -1, 1)]):
        with pytest.raises(ValueError):
            eng.step(rows, [0])
    tc.set_kernel_stream(torch.cuda.current_stream().cuda_stream)
    try:
        with pytest.raises(ValueError, match="current stream"):
            eng.step([(0, 0, 1)], [0])
    finally:
        tc.set_kernel_stream(None)
    plain = engine.Engine(model[1], 1, 64, 16)
    with pytest.raises(ValueError, match="ServingEngine"):
        plain.step([(0, 0, 1)], [0], rules=eng)


def test_captured_decode(model):
    """A captured step with rules and a window, replayed with new rows, positions and tokens and
    with pages taken and given up between the replays, against eager steps."""
    w = model[1]
    engs = [serving.ServingEngine(w, 3, 200, 64, window=40, sinks=2) for _ in range(2)]
    prompts = [t for _, t in family(6, 3, 20)]
    rules = [serving.Rules(1.3, 0.2, 0.1), None, serving.Rules(bias={9: 1.5}, allowed=range(300))]
    last = []
    for e in engs:
        for s in range(3):
            e.begin(s, prompts[s], rules[s])
        last.append([e.step([(s, p, t) for p, t in enumerate(prompts[s])], [len(prompts[s]) - 1])[0][0] for s in range(3)])
    assert last[0] == last[1]
    eager, captured = engs
    n = [len(p) for p in prompts]
    rows = [(s, n[s], last[0][s]) for s in range(3)]
    slot, pos, tok, _ = captured.device_rows(rows)
    best = torch.empty((3, 2), dtype=torch.int32, device=DEV)
    rr = captured.row_rules([0, 1, 2])
    counts = captured.counts.counts.clone(), captured.counts.seen.clone()
    captured.hold(rows)
    captured.launch(3, slot, pos, tok, None, best=best, rules=rr, runs=1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.launch(3, slot, pos, tok, None, best=best, rules=rr, runs=1)
    captured.counts.counts.copy_(counts[0])
    captured.counts.seen.copy_(counts[1])
    for k in range(60):
        rows = [(s, n[s] + k, last[0][s]) for s in range(3)]
        want = eager.step(rows, [0, 1, 2])
        captured.hold(rows)
        pos.copy_(torch.tensor([r[1] for r in rows], dtype=torch.int32))
        tok.copy_(torch.tensor([r[2] for r in rows], dtype=torch.int32))
        graph.replay()
        b = best.cpu().numpy().view(np.uint32)
        assert [(int(x[1]), int(x[0])) for x in b] == want, k
        last[0] = [t for t, _ in want]
    for e in engs:
        e.check()
    assert torch.equal(eager.counts.counts, captured.counts.counts)


def test_cache_operators_between_attentions():
    """A cache that is written, branched, moved out and back, evicted from and read again: each
    attention has the bits of one over a plain cache with the same entries."""
    n_kv, n_q, D, layers, page = 2, 4, 64, 2, 16
    g = torch.Generator(device=DEV).manual_seed(8)
    pool = KvPool.create(4, 700, 100, n_kv, D, layers, page, DEV)
    away = KvPool.create(4, 700, 50, n_kv, D, layers, page, DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    dense = torch.empty((3, layers, 2, 700, n_kv, D), device=DEV, dtype=torch.bfloat16).normal_(generator=g)  # what slots hold
    view = pool.arena.view(100, layers, 2, n_kv, page, D)

    def write(slot, first, end):
        for t in range(first, end):
            view[int(pool.table[slot, t // page]), :, :, :, t % page] = dense[slot, :, :, t].view(torch.int16)

    def attend(slots, pos, window=0, sinks=0, runs=0):
        q = torch.empty((len(pos), n_kv * n_q * D), device=DEV).normal_(generator=g)
        call = lambda kv, layer: layout.untile_lanes(harness.window_attention(q, kv, i32(*slots), i32(*pos), n_kv, n_q, D, 0.125, window,
                                                                              sinks, layer, runs=runs), len(pos))
        plain = torch.zeros((3, 44, layers, 2, n_kv, page, D), dtype=torch.int16, device=DEV)
        for t in range(700):
            plain[:, t // page, :, :, :, t % page] = dense[:, :, :, t].view(torch.int16)
        kv = harness.PagedKv.over(plain, torch.arange(132, device=DEV, dtype=torch.int32).reshape(3, 44), n_kv, D, layers, page)
        for layer in range(layers):
            assert torch.equal(call(pool.kv, layer), call(kv, layer)), (slots, pos, layer)

    pool.reserve(i32(0, 1), i32(0, 0), i32(38, 5))
    write(0, 0, 600)
    write(1, 0, 70)
    attend([0, 1], [599, 69], runs=1)
    attend([0] * 40, list(range(560, 600)), 200, 4, runs=40)
    pool.fork(i32(0), i32(2), i32(500))  # a branch, which goes on in its own way
    dense[2, :, :, :500] = dense[0, :, :, :500]
    pool.reserve(i32(2), i32(0), i32(37))
    write(2, 500, 580)
    attend([0, 2, 1, 2], [599, 579, 50, 501])
    keep = torch.sort(torch.randperm(540, generator=torch.Generator().manual_seed(2))[:300]).values + 20  # evicted from
    pool.compact(i32(2), i32(20), i32(300), keep.to(torch.int32).to(DEV)[None])
    dense[2, :, :, 20:320] = dense[2, :, :, keep.to(DEV)].clone()
    attend([2] * 30 + [0], list(range(290, 320)) + [599], runs=30)
    held = pool.table[0, :38].clone()  # slot 0 moves out, its pages serve another, and back
    away.reserve(i32(1), i32(0), i32(38))
    pool.copy(held, away.table[1, :38].contiguous(), into=away)
    pool.release(i32(0), i32(0), i32(44))
    pool.reserve(i32(3), i32(0), i32(44))
    for t in range(44):
        view[int(pool.table[3, t])] = 0x7F81
    pool.release(i32(3), i32(0), i32(44))
    pool.reserve(i32(0), i32(0), i32(38))
    away.copy(away.table[1, :38].contiguous(), pool.table[0, :38].contiguous(), into=pool)
    attend([0, 2], [599, 319])
    pool.check(), away.check()
    pool.release(i32(0, 1, 2), i32(0, 0, 0), i32(44, 44, 44))
    assert pool.free_pages() == 100
