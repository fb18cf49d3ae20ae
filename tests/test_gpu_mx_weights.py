"""Models in microscaled weights as they are made: on torch's stream whatever the kernels' is, and without
the bf16 model beside them."""

import json

import pytest
import torch

import llama_tiny
from stride_amd import cli, mx, tc, weights

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def same_model(a, b):
    assert a.bits == b.bits == 4 and a.bytes_per_pass == b.bytes_per_pass and a.cfg == b.cfg
    assert torch.equal(a.embed, b.embed) and torch.equal(a.lm, b.lm) and torch.equal(a.norm_final, b.norm_final) and torch.equal(a.rope, b.rope)
    for L, Q in zip(a.layers, b.layers, strict=True):
        assert L.keys() == Q.keys()
        for k in L:
            for p, q in (((L[k].codes, Q[k].codes), (L[k].scales, Q[k].scales)) if isinstance(L[k], mx.Tiles) else ((L[k], Q[k]),)):
                assert torch.equal(p, q), k


def test_made_beside_another_kernel_stream(tmp_path):
    """The matrices are packed on torch's current stream, so their blocks are made there too."""
    llama_tiny.write(str(tmp_path), seed=8)
    w = weights.Weights.load(str(tmp_path), DEV, max_positions=64)
    want = w.microscaled()
    stream = torch.cuda.Stream()
    tc.set_kernel_stream(stream)
    try:
        got = w.microscaled()
    finally:
        tc.set_kernel_stream(None)
    torch.cuda.synchronize()
    same_model(got, want)
    with torch.cuda.stream(stream):
        got = w.microscaled()
    torch.cuda.synchronize()
    same_model(got, want)


def test_made_a_matrix_at_a_time(tmp_path, monkeypatch):
    """load(bits=4) and random(bits=4) are the blocks of the bf16 model, and never hold it: beside what
    they keep there are a matrix's rows, its tiles and the values that it is made from (8 bytes of a
    bf16 one's 2 while a random one is drawn), and not a layer's share of the others."""
    shape = dict(llama_tiny.TINY, num_hidden_layers=12, vocab_size=400)
    llama_tiny.write(str(tmp_path), seed=9, cfg=shape)
    cfg = weights.ModelConfig.load(str(tmp_path))
    for make in (lambda bits: weights.Weights.load(str(tmp_path), DEV, max_positions=64, bits=bits),
                 lambda bits: weights.Weights.random(cfg, DEV, 3, 64, bits)):
        full = make(16)
        want = full.microscaled()
        matrices = [2 * t.numel() for L in full.layers for k, t in L.items() if not k.startswith("norm")]
        del full
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        got = make(4)
        kept, most = torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before
        same_model(got, want)
        assert most < kept + 8 * max(matrices + [2 * cfg.vocab * cfg.hidden]) < kept + sum(matrices) * 3 // 4, (kept, most, sum(matrices))
        del got, want
    with pytest.raises(ValueError, match="4 or 16"):
        weights.Weights.load(str(tmp_path), DEV, bits=8)
    with pytest.raises(ValueError, match="4 or 16"):
        weights.Weights.random(cfg, DEV, bits=0)


def test_command_makes_a_matrix_at_a_time(tmp_path, monkeypatch):
    """--weights mx4 without a bf16 model, and the ledger of one made from it."""
    llama_tiny.write(str(tmp_path), seed=10)
    (tmp_path / "p.jsonl").write_text("".join(json.dumps({"id": i, "tokens": [5 * i + 1, 2, 3]}) + "\n" for i in range(3)))

    def ledger(name):
        assert cli.main(["--model", str(tmp_path), "--input", str(tmp_path / "p.jsonl"), "--output", str(tmp_path / name), "--max-new", "5",
                         "--weights", "mx4"]) == 0
        return (tmp_path / name).read_text()

    with monkeypatch.context() as m:
        load = weights.Weights.load
        m.setattr(weights.Weights, "load", staticmethod(lambda *a, bits=16, **k: load(*a, **k).microscaled() if bits == 4 else load(*a, **k)))
        want = ledger("a.jsonl")
    monkeypatch.setattr(weights.Weights, "microscaled", lambda self: pytest.fail("the bf16 model was made first"))
    assert ledger("b.jsonl") == want
