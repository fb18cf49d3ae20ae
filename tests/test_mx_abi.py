"""The microscaled operators' C ABI (include/stride_mx.h) without a GPU: exports, struct layouts,
packed blocks, sizes, and every refusal that comes before a launch; the plain forms of the tests."""
import copy
import ctypes as C
import os
import pickle
import re
import struct
import subprocess

import numpy as np
import pytest
import torch

import mx_plain
from stride_amd import _lib, mx

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "stride_mx.h")
BUF = 0x7F0000000000  # an address that nothing may touch: every call here is refused or empty
LAYOUTS = {"StrideMxTiles": "<2Q2i", "StrideMxQuantizeParams": "<4iQ24s2i", "StrideMxDequantizeParams": "<4i24sQq2i",
           "StrideMxNormParams": "<4i3Q24sQif", "StrideMxGemmParams": "<4i24s24sQ", "StrideMxMlp13Params": "<4i24s24s24s24s",
           "StrideMxQkvParams": "<4i24s24s24s24sQq56s3Q2i"}


def test_exports_match_header():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"\b(stride_mx_\w+)\s*\(", text))
    assert declared == set(_lib.MX_ENTRIES)
    for name in declared:
        assert hasattr(_lib.load(), name), name


def test_struct_layout(tmp_path):
    """The C compiler's sizes are those of the blocks that the runners pack, without padding."""
    src = tmp_path / "probe.c"
    src.write_text(f'#include "{HEADER}"\n#include <stdio.h>\nint main(void) {{\n' +
                   "".join(f'printf("%zu\\n", sizeof({name}));\n' for name in LAYOUTS) + "return 0;}\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [struct.calcsize(f) for f in LAYOUTS.values()]


def test_sizes():
    lib = _lib.load()
    for cols, groups in ((16, 1), (512, 1), (528, 2), (2048, 4), (1 << 20, 2048)):
        assert lib.stride_mx_code_bytes(cols, 4) == groups * 4096 and lib.stride_mx_code_bytes(cols, 8) == groups * 8192
        assert lib.stride_mx_scale_bytes(cols) == groups * 256
    for cols in (0, -16, 8, 24, (1 << 20) + 16):
        assert lib.stride_mx_code_bytes(cols, 4) == lib.stride_mx_scale_bytes(cols) == -1
    assert lib.stride_mx_code_bytes(512, 6) == -1


def tiles(tiles=1, cols=512, codes=BUF, scales=BUF):
    return mx._TILES(codes, scales, tiles, cols)


def call(name, block):
    return getattr(_lib.packed(), "stride_mx_" + name)(block, None)


def err():
    return _lib.load().stride_tc_last_error().decode()


BAD_TILES = [(dict(cols=0), "cols"), (dict(cols=24), "cols"), (dict(cols=1 << 21), "cols"), (dict(tiles=0), "too few"),
             (dict(codes=0), "missing"), (dict(scales=0), "missing"), (dict(codes=BUF + 8), "aligned"), (dict(scales=BUF + 2), "aligned")]


@pytest.mark.parametrize("bad,why", BAD_TILES)
def test_tiles_that_are_refused(bad, why):
    t, ok = tiles(**bad), tiles()
    for name, block in (("quantize", mx._QUANTIZE(5, 1, 0, 0, BUF, t, 4, 2)), ("dequantize", mx._DEQUANTIZE(5, 1, 0, 0, t, BUF, 1 << 21, 4, 2)),
                        ("gemm", mx._GEMM(5, 1, 0, 0, t, ok, BUF)), ("gemm", mx._GEMM(5, 1, 0, 0, ok, t, BUF)),
                        ("mlp13", mx._MLP13(5, 1, 0, 0, t, ok, ok, tiles(cols=16))), ("mlp13", mx._MLP13(5, 1, 0, 0, ok, ok, t, tiles(cols=16)))):
        assert call(name, block) == _lib.EINVAL, name
        assert why in err() or "equal tiles" in err() or "cols differ" in err(), (name, err())


@pytest.mark.parametrize("rows,groups", [(-1, 0), (5, 2), (17, 1), (2 ** 31 - 1, 1)])
def test_lanes_that_are_refused(rows, groups):
    t, kv = tiles(1 << 28), bytes(_lib.KvRef())
    for name, block in (("quantize", mx._QUANTIZE(rows, groups, 0, 0, BUF, t, 4, 2)), ("dequantize", mx._DEQUANTIZE(rows, groups, 0, 0, t, BUF, 512, 4, 2)),
                        ("norm", mx._NORM(rows, groups, 0, 0, BUF, 0, BUF, t, 0, 512, 1e-5)), ("gemm", mx._GEMM(rows, groups, 0, 0, t, t, BUF)),
                        ("mlp13", mx._MLP13(rows, groups, 0, 0, t, t, t, t)), ("qkv", mx._QKV(rows, groups, 0, 0, t, t, t, t, BUF, 16, kv, BUF, BUF, BUF, 0, 16))):
        assert call(name, block) == _lib.EINVAL and "lane_groups" in err(), name


def test_nothing_to_do_and_nothing_given():
    t, kv = tiles(0, codes=0, scales=0), bytes(_lib.KvRef())
    for name, block in (("quantize", mx._QUANTIZE(0, 0, 0, 0, 0, t, 4, 2)), ("dequantize", mx._DEQUANTIZE(0, 0, 0, 0, t, 0, 512, 4, 2)),
                        ("norm", mx._NORM(0, 0, 0, 0, 0, 0, 0, t, 0, 512, 1e-5)), ("gemm", mx._GEMM(0, 0, 0, 0, t, t, 0)),
                        ("mlp13", mx._MLP13(0, 0, 0, 0, t, t, t, t)), ("qkv", mx._QKV(0, 0, 0, 0, t, t, t, t, 0, 16, kv, 0, 0, 0, 0, 16))):
        assert call(name, block) == 0, name
        assert call(name, None) == _lib.EINVAL and "null" in err()


def test_copies_of_tiles_have_their_own_memory():
    """What a copied, pickled or loaded Tiles hands to a call is its own memory's address, and the
    tensors behind an address are not exchanged."""
    t = mx.Tiles.create(20, 528, 4, "cpu")
    t.codes.fill_(3)
    for other in (copy.deepcopy(t), pickle.loads(pickle.dumps(t)), copy.copy(t)):
        assert other._ref == mx._TILES(other.codes.data_ptr(), other.scales.data_ptr(), 2, 528)
        assert torch.equal(other.codes, t.codes) and (other.cols, other.bits, other.rows) == (528, 4, 32)
    assert copy.deepcopy(t).codes.data_ptr() != t.codes.data_ptr()
    for name in ("codes", "scales", "cols", "bits"):
        with pytest.raises(AttributeError):
            setattr(t, name, getattr(t, name))


def test_launches_beyond_32_bits_of_threads():
    """A launch counts its threads in 32 bits: what would not fit is refused."""
    rows = 2 ** 31 - 16
    t, w = tiles(1 << 27, 1 << 20), tiles(1 << 10, 1 << 20)
    for name, block in (("quantize", mx._QUANTIZE(rows, rows // 16, 0, 0, BUF, t, 4, 2)), ("dequantize", mx._DEQUANTIZE(rows, rows // 16, 0, 0, t, BUF, 1 << 20, 4, 2)),
                        ("norm", mx._NORM(rows, rows // 16, 0, 0, BUF, 0, BUF, tiles(1 << 27), 0, 512, 1e-5)), ("gemm", mx._GEMM(rows, rows // 16, 0, 0, t, w, BUF)),
                        ("mlp13", mx._MLP13(rows, rows // 16, 0, 0, t, w, w, tiles(1 << 27, 1 << 14, BUF + 64)))):
        assert call(name, block) == _lib.EINVAL and "too " in err(), name


@pytest.mark.parametrize("block,why", [
    (mx._QUANTIZE(5, 1, 0, 0, BUF, tiles(), 6, 2), "bits"), (mx._QUANTIZE(5, 1, 0, 0, BUF, tiles(), 4, 3), "bytes"),
    (mx._QUANTIZE(5, 1, 0, 0, 0, tiles(), 4, 2), "src"), (mx._QUANTIZE(5, 1, 0, 0, BUF + 8, tiles(), 4, 2), "src"),
])
def test_quantize_refuses(block, why):
    assert call("quantize", block) == _lib.EINVAL and why in err()


@pytest.mark.parametrize("block,why", [
    (mx._DEQUANTIZE(5, 1, 0, 0, tiles(), BUF, 512, 5, 2), "bits"), (mx._DEQUANTIZE(5, 1, 0, 0, tiles(), BUF, 512, 4, 8), "bytes"),
    (mx._DEQUANTIZE(5, 1, 0, 0, tiles(), 0, 512, 4, 2), "out"), (mx._DEQUANTIZE(5, 1, 0, 0, tiles(), BUF, 504, 4, 2), "out_stride"),
    (mx._DEQUANTIZE(5, 1, 0, 0, tiles(), BUF, 516, 4, 2), "out_stride"),
])
def test_dequantize_refuses(block, why):
    assert call("dequantize", block) == _lib.EINVAL and why in err()


@pytest.mark.parametrize("over,why", [
    (dict(dim=0), "dim"), (dict(dim=24), "dim"), (dict(dim=1 << 17), "dim"), (dict(h=0), "need h"), (dict(weight=0), "need h"),
    (dict(x=BUF), "one of"), (dict(out=mx._NONE), "one of"), (dict(out=tiles(cols=528)), "cols"), (dict(out=tiles(0)), "too few"),
    (dict(h=BUF + 4), "aligned"), (dict(add=BUF + 2), "aligned"), (dict(weight=BUF + 4), "aligned"), (dict(out=mx._NONE, x=BUF + 8), "aligned"),
])
def test_norm_refuses(over, why):
    a = {**dict(h=BUF, add=0, weight=BUF, out=tiles(), x=0, dim=512), **over}
    assert call("norm", mx._NORM(5, 1, 0, 0, *a.values(), 1e-5)) == _lib.EINVAL and why in err()


@pytest.mark.parametrize("name,block,why", [
    ("gemm", mx._GEMM(5, 1, 0, 0, tiles(), tiles(), 0), "y"), ("gemm", mx._GEMM(5, 1, 0, 0, tiles(), tiles(), BUF + 8), "y"),
    ("gemm", mx._GEMM(5, 1, 0, 0, tiles(), tiles(cols=528), BUF), "cols"), ("gemm", mx._GEMM(17, 2, 0, 0, tiles(), tiles(), BUF), "too few"),
    ("mlp13", mx._MLP13(5, 1, 0, 0, tiles(), tiles(2), tiles(3), tiles(cols=32, codes=BUF + 64)), "equal tiles"),
    ("mlp13", mx._MLP13(5, 1, 0, 0, tiles(), tiles(2), tiles(2), tiles(cols=48, codes=BUF + 64)), "cols"),
    ("mlp13", mx._MLP13(17, 2, 0, 0, tiles(2), tiles(2), tiles(2), tiles(cols=32, codes=BUF + 64)), "too few"),
    ("mlp13", mx._MLP13(5, 1, 0, 0, tiles(), tiles(32), tiles(32), tiles()), "z must not be x"),
    ("mlp13", mx._MLP13(5, 1, 0, 0, tiles(), tiles(1 << 17), tiles(1 << 17), tiles(cols=1 << 20)), "row tiles"),
])
def test_products_refuse(name, block, why):
    assert call(name, block) == _lib.EINVAL and why in err()


def qkv(q=4, kv=1, head_dim=64, q_stride=64, layer=0, rope=BUF, pos=BUF, **ref):
    r = _lib.KvRef(BUF, BUF, 2 * 1024, 2 * 1024, 1024, 1024, 8, 64)
    for k, v in ref.items():
        setattr(r, k, v)
    return mx._QKV(5, 1, 0, 0, tiles(), tiles(q), tiles(4 * kv), tiles(4), BUF, q_stride, bytes(r), rope, BUF, pos, layer, head_dim)


@pytest.mark.parametrize("over,why", [
    (dict(kv=2), "equal tiles"), (dict(head_dim=24), "head_dim"), (dict(head_dim=128), "head_dim"), (dict(q=3), "head_dim"),
    (dict(rope=0), "missing"), (dict(pos=0), "missing"), (dict(q_stride=48), "q_stride"), (dict(layer=-1), "layer"), (dict(max_blocks=0), "max_blocks"),
    (dict(arena=0), "missing"), (dict(table=0), "missing"), (dict(group_elems=24 * 64), "power of two"), (dict(group_elems=1000), "group_elems"),
])
def test_qkv_refuses(over, why):
    assert call("qkv", qkv(**over)) == _lib.EINVAL and why in err()


def test_tiles_are_checked():
    t = mx.Tiles.create(20, 528, 4, "cpu")
    assert (t.tiles, t.rows, t.cols, t.nbytes) == (2, 32, 528, 2 * 2 * (4096 + 256))
    for bad in (lambda: mx.Tiles(t.codes, t.scales, 528, 8), lambda: mx.Tiles(t.codes, t.scales, 1040, 4), lambda: mx.Tiles(t.codes, t.scales[:1], 528, 4),
                lambda: mx.Tiles(t.codes.to(torch.int8), t.scales, 528, 4), lambda: mx.Tiles(t.codes, t.scales, 520, 4),
                lambda: mx.Tiles(t.codes.transpose(3, 4), t.scales, 528, 4), lambda: mx.Tiles.create(3, 64, 6, "cpu"), lambda: mx.Tiles.create(-1, 64, 4, "cpu")):
        with pytest.raises(ValueError):
            bad()
    assert mx.Tiles.create(0, 64, 4, "cpu").tiles == 0


@pytest.mark.parametrize("bits", [4, 8])
def test_plain_form_is_the_nearest(bits):
    """The oracle's elements against a search over all values of the format, its scales against the
    smallest power of two that cuts nothing off, and its layout against its inverse."""
    rng = np.random.default_rng(bits)
    a = rng.standard_normal((7, 560)) * 2.0 ** rng.integers(-30, 30, (7, 1))
    code, byte = mx_plain.encode(a, bits)
    v, w = mx_plain.decode(code, byte, bits), mx_plain.wide(a)
    table = mx_plain.E2M1 if bits == 4 else mx_plain.E4M3
    every = np.concatenate([-table, table])
    scale = np.repeat(2.0 ** (byte - 127.0), 32, 1)
    for r in range(7):
        best = np.abs(w[r][:, None] / scale[r][:, None] - every).min(1)
        assert np.array_equal(np.abs(w[r] - v[r]) / scale[r], best)
    top, half = (6.0, 1.0) if bits == 4 else (448.0, 16.0)
    most, s = np.abs(w).reshape(16, -1, 32).max(-1), 2.0 ** (byte - 127.0)
    live = most > 0
    assert (most[live] <= (top + half) * s[live]).all() and (most[live] > (top + half) * s[live] / 2 - (bits == 4) * 1e-300).all()
    assert all(np.array_equal(p, q) for p, q in zip(mx_plain.unpack(*mx_plain.pack(code, byte, bits), bits), (code, byte)))
