"""Calls of the microscaled operators that have to be refused, or that have to leave rows alone, without
a GPU: what the C ABI refuses before a launch."""
import pytest
import torch

from stride_amd import _lib, harness, mx

BUF = 0x7F0000000000  # an address that nothing may touch: every call here is refused


def tiles(tiles=1, cols=512, codes=BUF, scales=BUF):
    return mx._TILES(codes, scales, tiles, cols)


def err():
    return _lib.load().stride_tc_last_error().decode()


@pytest.mark.parametrize("slots,positions", [(-1, 8), (8, -1), (-2 ** 31, -2 ** 31)])
def test_qkv_within_refuses(slots, positions):
    ref = bytes(_lib.KvRef(BUF, BUF, 2048, 2048, 1024, 1024, 8, 64))
    block = mx._QKV(5, 1, 0, 0, tiles(), tiles(4), tiles(4), tiles(4), BUF, 64, ref, BUF, BUF, BUF, 0, 64)
    lib = _lib.packed()
    assert lib.stride_mx_qkv_within(block, slots, positions, None) == _lib.EINVAL and "counts" in err()
    assert lib.stride_mx_qkv_within(None, 8, 8, None) == _lib.EINVAL and "null" in err()
    empty = mx._QKV(0, 0, 0, 0, tiles(0), tiles(0), tiles(0), tiles(0), 0, 64, ref, 0, 0, 0, 0, 64)
    assert lib.stride_mx_qkv_within(empty, 8, 8, None) == 0


def code(tiles, cols, bits):
    return tiles * _lib.load().stride_mx_code_bytes(cols, bits)


def span(tiles, cols, bits, at, scales=None):
    """Tiles at `at`, their scales behind their codes (or at `scales`)."""
    return mx._TILES(at, at + code(tiles, cols, bits) if scales is None else scales, tiles, cols)


FAR = BUF + (1 << 40)
ROWS, LT, COLS = 37, 3, 528  # two groups
VALUES = LT * 33 * 256
X8, Z8 = code(LT, COLS, 8), code(LT, 2 * COLS, 8)
W = 2 * COLS // 16


@pytest.mark.parametrize("name,block", [
    # each result on the last byte of an operand, or an operand's first on the result's last
    *(("quantize", mx._QUANTIZE(ROWS, LT, 0, 0, FAR, t, 8, 4)) for t in (
        span(LT, COLS, 8, FAR + VALUES * 4 - 16), span(LT, COLS, 8, FAR - X8 + 16), span(LT, COLS, 8, BUF, FAR + 64))),
    *(("dequantize", mx._DEQUANTIZE(ROWS, LT, 0, 0, span(LT, COLS, 4, BUF, FAR), out, 544, 4, 2)) for out in (
        BUF, BUF + code(LT, COLS, 4) - 16, FAR, BUF - (36 * 544 + COLS) * 2 + 16)),
    *(("norm", mx._NORM(ROWS, LT, 0, 0, h, add, gain, out, x, COLS, 1e-5)) for h, add, gain, out, x in (
        (BUF, BUF + 16, FAR, span(LT, COLS, 8, FAR + (1 << 20)), 0), (BUF, 0, BUF + VALUES * 4 - 16, span(LT, COLS, 8, FAR), 0),
        (BUF, 0, FAR, span(LT, COLS, 8, BUF + 64), 0), (BUF, FAR, FAR + (1 << 30), span(LT, COLS, 8, FAR + 32), 0),
        (BUF, 0, FAR, span(LT, COLS, 8, FAR + 64), 0), (BUF, 0, FAR, mx._NONE, BUF + VALUES * 4 - 16), (BUF, FAR + 16, FAR + (1 << 30), mx._NONE, FAR),
        (BUF, 0, FAR, span(LT, COLS, 8, FAR + (1 << 30), BUF + 4), 0))),
    *(("gemm", mx._GEMM(ROWS, LT, 0, 0, span(LT, COLS, 8, BUF), span(W, COLS, 4, FAR), y)) for y in (
        BUF, BUF + X8 - 16, BUF + X8, FAR + code(W, COLS, 4) - 16, FAR + code(W, COLS, 4), FAR - 16)),
    *(("mlp13", mx._MLP13(ROWS, LT, 0, 0, span(LT, COLS, 8, BUF), span(W, COLS, 4, FAR), span(W, COLS, 4, FAR + (1 << 30)), z)) for z in (
        span(LT, 2 * COLS, 8, BUF + 16), span(LT, 2 * COLS, 8, BUF - Z8 + 16), span(LT, 2 * COLS, 8, FAR + (2 << 30), BUF + X8 + 4),
        span(LT, 2 * COLS, 8, FAR + 4096), span(LT, 2 * COLS, 8, FAR + (1 << 30) + 64), span(LT, 2 * COLS, 8, BUF + (1 << 30), FAR + 8))),
    # as many rows as each of the other forms of the products takes
    *(("gemm", mx._GEMM(16 * t, t, 0, 0, span(t, COLS, 8, BUF), span(w, COLS, 4, FAR), FAR)) for t, w in (
        (24, 33), (64, 66), (128, 66), (256, 64), (256, 128))),
])
def test_results_that_lie_on_an_operand(name, block):
    assert getattr(_lib.packed(), "stride_mx_" + name)(block, None) == _lib.EINVAL and "overlap" in err(), err()


@pytest.mark.parametrize("q_out,slot", [(BUF, FAR), (FAR + 64, FAR + (3 << 30)), (FAR + (2 << 30), FAR + (2 << 30) + 36 * 64 * 4 * 4)])
def test_qkv_results_that_lie_on_an_operand(q_out, slot):
    ref = bytes(_lib.KvRef(FAR + (4 << 30), FAR + (5 << 30), 2048, 2048, 1024, 1024, 8, 64))
    block = mx._QKV(ROWS, LT, 0, 0, span(LT, COLS, 8, BUF), span(16, COLS, 4, FAR), span(4, COLS, 4, FAR + (1 << 24)), span(4, COLS, 4, FAR + (1 << 25)),
                    q_out, 256, ref, FAR + (6 << 30), slot, FAR + (7 << 30), 0, 64)
    for call in (lambda: _lib.packed().stride_mx_qkv(block, None), lambda: _lib.packed().stride_mx_qkv_within(block, 8, 8, None)):
        assert call() == _lib.EINVAL and "overlap" in err(), err()


def test_arguments_of_another_kind_are_refused_by_a_message():
    """What trips over a missing attribute is no refusal: a tensor where Tiles belong and the other way."""
    x, w, t = mx.Tiles.create(20, 512, 8, "cpu"), mx.Tiles.create(64, 512, 4, "cpu"), torch.zeros((2, 32, 16, 16))
    kv = harness.PagedKv.create(1, 16, 1, 32, 1, 16, "cpu")
    for bad, name in ((lambda: mx.gemm(w, t, 20), "x"), (lambda: mx.gemm(w, None, 20), "x"), (lambda: mx.mlp13(w, w, t, 20), "x"),
                      (lambda: mx.qkv(w, w, w, t, 20, 32, t, t, t, kv), "x"), (lambda: mx.dequantize(t), "t"), (lambda: mx.quantize(x), "tiles"),
                      (lambda: mx.quantize([1.0]), "tiles"), (lambda: mx.norm(x, 20, t, 1e-5), "h"), (lambda: mx.norm(None, 20, t, 1e-5), "h")):
        with pytest.raises(ValueError, match=f"^{name} must"):
            bad()
