"""Models in microscaled weights as they are made: on torch's stream whatever the kernels' is, and without
the bf16 model beside them."""

import pytest
import torch

import llama_tiny
from stride_amd import mx, tc, weights

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
