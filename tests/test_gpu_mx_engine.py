"""Models in microscaled weights through the engines and the command: each operator of a step against
its formula in 64 bits on what it was given, ledgers that no scheduling changes, a captured step."""
import json

import numpy as np
import pytest
import torch

import llama_tiny
import mx_plain
from stride_amd import cli, engine, layout, mx, serving, weights

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    path = tmp_path_factory.mktemp("m")
    llama_tiny.write(str(path), seed=6)
    return str(path), weights.Weights.load(str(path), DEV, max_positions=512)


def prompts(seed, n, longest):
    rng = np.random.default_rng(seed)
    return [(i, rng.integers(0, 1000, int(rng.integers(1, longest))).tolist()) for i in range(n)]


def rows_of(tiles, n):
    return layout.untile_lanes(tiles.cpu(), n).double().numpy() if tiles.dtype != torch.int16 else \
        layout.untile_lanes(tiles.view(torch.bfloat16).cpu(), n).double().numpy()


def within(got, want, tol):
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


def test_weights_in_blocks(model):
    w = model[1]
    m = w.microscaled()
    assert (w.bits, m.bits) == (16, 4) and m.microscaled() is m and m.embed is w.embed
    for L, Q in zip(w.layers, m.layers):
        for k, t in L.items():
            if k.startswith("norm"):
                assert Q[k] is t
                continue
            rows = layout.unpack_rows(t).view(torch.bfloat16).cpu().double().numpy()
            code, byte = mx_plain.encode(rows, 4)
            codes, scales = mx_plain.pack(code, byte, 4)
            assert np.array_equal(Q[k].codes.cpu().numpy(), codes) and np.array_equal(Q[k].scales.cpu().numpy(), scales)
    matrices = sum(t.numel() for L in w.layers for k, t in L.items() if not k.startswith("norm"))
    head = w.cfg.vocab * w.cfg.hidden * 2
    assert m.bytes_per_pass - head < 1.1 * matrices * 17 / 32 * 2  # hidden 256 is filled up to 512
    assert w.bytes_per_pass - head == 2 * matrices


@pytest.mark.parametrize("kind", ["tc", "serve"])
def test_each_operator_of_a_step(model, monkeypatch, kind):
    """Tolerances: those of tests/test_gpu_mx.py (half a step of the result's type, the instruction's
    cut-offs, fp32 sums)."""
    m = model[1].microscaled()
    real = {k: getattr(mx, k) for k in ("norm", "quantize", "gemm", "mlp13")}
    calls = dict.fromkeys(real, 0)

    def eight(t, n, want, e):
        code, byte = mx_plain.unpack(t.codes.cpu().numpy(), t.scales.cpu().numpy(), 8)
        got, scale = mx_plain.decode(code, byte, 8), np.repeat(2.0 ** (byte - 127.0), 32, 1)
        within(got[:n, : t.cols], want, e + np.maximum(2.0 ** -4 * (np.abs(want) + e), 2.0 ** -10 * scale[:n, : t.cols]))
        assert (got[:n, t.cols:] == 0).all()

    def norm(h, n, weight, eps, add=None, out=None, bits=8):
        before = rows_of(h, n)
        delta = 0 if add is None else rows_of(add, n)
        t = real["norm"](h, n, weight, eps, add=add, out=out, bits=bits)
        after = (before.astype(np.float32) + np.asarray(delta, np.float32)).astype(np.float64)
        assert np.array_equal(rows_of(h, n), after)
        want = after / np.sqrt((after * after).mean(1, keepdims=True) + eps) * weight.cpu().double().numpy()
        e = 30 * 2.0 ** -24 * np.abs(want)  # a sum of 256 squares: 8 a lane and 20 more, halved by the root, six roundings around
        eight(t, n, want, e) if bits == 8 else within(rows_of(t, n), want, e + 2.0 ** -8 * (np.abs(want) + e))
        calls["norm"] += 1
        return t

    def quantize(tiles, n, bits, out):
        t = real["quantize"](tiles, n, bits=bits, out=out)
        code, byte = mx_plain.encode(rows_of(tiles, n), bits)
        got = mx_plain.unpack(t.codes.cpu().numpy(), t.scales.cpu().numpy(), bits)
        assert np.array_equal(got[0][:n], code[:n]) and np.array_equal(got[1][:n], byte[:n])
        calls["quantize"] += 1
        return t

    def gemm(w, x, n, out):
        t = real["gemm"](w, x, n, out=out)
        wv, xv = mx_plain.values(w, w.rows, w.cols), mx_plain.values(x, n, x.cols)
        want, e = xv @ wv.T, mx_plain.products_bound(wv, xv)
        within(rows_of(t, n), want, e + 2.0 ** -8 * (np.abs(want) + e))
        calls["gemm"] += 1
        return t

    def mlp13(w1, w3, x, n, out):
        t = real["mlp13"](w1, w3, x, n, out=out)
        v1, v3, xv = mx_plain.values(w1, w1.rows, w1.cols), mx_plain.values(w3, w3.rows, w3.cols), mx_plain.values(x, n, x.cols)
        g, u, eg, eu = xv @ v1.T, xv @ v3.T, mx_plain.products_bound(v1, xv), mx_plain.products_bound(v3, xv)
        silu = g / (1 + np.exp(-g))
        eight(t, n, silu * u, 1.1 * eg * (np.abs(u) + eu) + np.abs(silu) * eu + 2.0 ** -20 * np.abs(silu * u))
        calls["mlp13"] += 1
        return t

    for k, f in (("norm", norm), ("quantize", quantize), ("gemm", gemm), ("mlp13", mlp13)):
        monkeypatch.setattr(mx, k, f)
    todo = prompts(3, 3, 20)
    if kind == "tc":
        eng = engine.Engine(m, 3, 40, 16)
    else:
        eng = serving.ServingEngine(m, 3, 40, 16, window=12, sinks=2)
    done = cli.Scheduler(eng, 3, 3).run(todo)
    assert len(done) == 3 and all(len(s.tokens) == 3 for s, _ in done.values())
    layers = len(m.layers)
    assert calls["gemm"] == 2 * calls["mlp13"] == 2 * calls["quantize"] and calls["norm"] == calls["gemm"] // (2 * layers) * (2 * layers + 1)


@pytest.mark.parametrize("more", [["--path", "tc"], ["--path", "serve", "--window", "50", "--sinks", "3", "--repetition-penalty", "1.2"]])
def test_ledger_identical_across_scheduling(model, tmp_path, more):
    with open(tmp_path / "p.jsonl", "w") as f:
        for pid, tokens in prompts(4, 8, 100):
            f.write(json.dumps({"id": pid, "tokens": tokens}) + "\n")
    base = ["--model", model[0], "--input", str(tmp_path / "p.jsonl"), "--max-new", "9", "--weights", "mx4", *more]
    shuffle = ["--kv-shuffle", "3"] if "tc" in more else ["--share-prefixes"]
    out = []
    for k, how in enumerate(([], ["--concurrency", "4", "--max-rows", "24", "--row-shuffle", "5", *shuffle],
                             ["--concurrency", "8", "--max-rows", "300", "--page-tokens", "8"])):
        print("ledger", more, how, flush=True)
        assert cli.main([*base, "--output", str(tmp_path / f"{k}.jsonl"), *how]) == 0
        out.append((tmp_path / f"{k}.jsonl").read_text())
    assert out[0] == out[1] == out[2]
    assert cli.main([a for a in base if a not in ("--weights", "mx4")] + ["--output", str(tmp_path / "b.jsonl")]) == 0
    assert (tmp_path / "b.jsonl").read_text() != out[0], "bf16 weights have another ledger"


def test_step_captured_and_replayed(model):
    """A decode step in a HIP graph, with eager steps between the replays."""
    m = model[1].microscaled()
    todo = [p for _, p in prompts(5, 4, 30)]

    def ready():
        eng = engine.Engine(m, 4, 60, 64, attention_one_kernel=True)
        seqs = [engine.Sequence(i, p) for i, p in enumerate(todo)]
        eng.prefill(seqs)
        return eng, seqs

    want_eng, want = ready()
    want_eng.decode(want, 5)
    eng, seqs = ready()
    other, other_seqs = ready()
    rows = [(s.slot, s.length - 1, s.tokens[-1]) for s in seqs]
    slot, pos, tok, items = eng.device_rows(rows)
    best = torch.zeros((4, 2), dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eng.launch(4, slot, pos, tok, items, best=best)
    for k in range(5):
        fresh = eng.device_rows([(s.slot, s.length - 1, s.tokens[-1]) for s in seqs])
        for a, b in zip((slot, pos, tok), fresh):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = best.cpu().numpy()
        for i, s in enumerate(seqs):
            eng._record(s, int(got[i, 1]), int(got[i, 0]) & 0xFFFFFFFF)
        other.decode(other_seqs, 1)
    for a, b in zip(seqs, want):
        assert a.tokens == b.tokens and a.fingerprint == b.fingerprint


def test_exact_path_has_no_such_weights(capsys):
    with pytest.raises(SystemExit):
        cli.main(["--model", "random:0", "--input", "none", "--output", "none", "--path", "exact", "--weights", "mx4"])
    assert "mx4" in capsys.readouterr().err
