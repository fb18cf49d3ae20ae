"""The serving operators' C ABI (include/stride_serve.h) without a GPU: exports, struct
layouts, packed blocks, the scratch sizes, and every refusal that comes before a launch."""
import ctypes as C
import os
import re
import struct
import subprocess

import pytest

from stride_amd import _lib, harness, logits

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "stride_serve.h")
BUF = 0x7F0000000000  # an address that nothing may touch: every call here is refused or empty


def err():
    return _lib.load().stride_tc_last_error().decode()


def test_exports_match_header():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"\b(stride_(?:serve|kv|logits)_\w+)\s*\(", text))
    assert declared == set(_lib.SERVE_ENTRIES)
    lib = _lib.load()
    for name in declared:
        assert hasattr(lib, name), name


def test_struct_layout(tmp_path):
    pairs = {"StrideWindowAttentionParams": _lib.WindowAttentionParams, "StrideKvPool": _lib.KvPoolParams,
             "StrideLogitsParams": _lib.LogitsParams, "StrideTokenCounts": _lib.TokenCountsParams}
    lines = []
    for cname, cls in pairs.items():
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        lines += [f'printf("%zu\\n", offsetof({cname}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "probe.cpp"
    src.write_text(f'#include <cstddef>\n#include <cstdio>\n#include "{HEADER}"\nint main() {{\n' + "\n".join(lines) + "\n}\n")
    subprocess.run(["g++", "-std=c++17", str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for cls in pairs.values():
        want.append(C.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want
    assert struct.calcsize("<4iQqQ56sQQQq9if") == C.sizeof(_lib.WindowAttentionParams)
    assert struct.calcsize("<4i13Q3i4x") == C.sizeof(_lib.LogitsParams)


def test_header_is_c(tmp_path):
    src = tmp_path / "probe.c"
    src.write_text(f'#include "{HEADER}"\nint main(void) {{ return sizeof(StrideKvPool) == 120 ? 0 : 1; }}\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(src), "-o", str(tmp_path / "probe")], check=True)
    assert subprocess.run([str(tmp_path / "probe")]).returncode == 0


def attention(**over):
    p = _lib.WindowAttentionParams()
    p.l = _lib.Lanes(4, 1, 0, 0)
    p.q = p.out = p.row_slot = p.row_pos = p.scratch = BUF
    p.q_stride = p.out_cols = 8 * 4 * 64
    p.kv = _lib.KvRef(BUF, BUF, 2 * 8 * 16 * 64, 2 * 8 * 16 * 64, 8 * 16 * 64, 16 * 64, 64, 64)
    p.scratch_floats = 1 << 40
    p.max_pages, p.n_kv, p.n_q, p.head_dim, p.scale = 16, 8, 4, 64, 0.125
    for k, v in over.items():
        obj = p
        *path, last = k.split("__")
        for x in path:
            obj = getattr(obj, x)
        setattr(obj, last, v)
    return p


@pytest.mark.parametrize("over,why", [
    (dict(l__rows=-1), "rows >= 0"), (dict(l__lane_groups=2), "lane_groups"),
    (dict(head_dim=48), "head_dim"), (dict(kv__head_dim=128), "head_dim"), (dict(head_dim=256, kv__head_dim=256), "head_dim"),
    (dict(n_q=0), "query heads"), (dict(n_q=17), "query heads"), (dict(n_kv=0), "n_kv"), (dict(layer=-1), "layer"),
    (dict(max_pages=0), "max_pages"), (dict(sinks=-1), "sinks"), (dict(runs=-1), "runs"), (dict(kv__max_blocks=0), "max_blocks"),
    (dict(kv__group_elems=4 * 64), "power of two"), (dict(kv__group_elems=24 * 64), "power of two"),
    (dict(kv__group_elems=16 * 64 + 8), "power of two"), (dict(kv__block_elems=12), "strides"), (dict(kv__which_elems=4), "strides"),
    (dict(out_cols=2040), "out_cols"), (dict(out_cols=1024), "out_cols"), (dict(q_stride=2046), "q_stride"),
    (dict(q_stride=1024), "q_stride"), (dict(q=0), "missing pointer"), (dict(out=0), "missing pointer"),
    (dict(kv__arena=0), "missing pointer"), (dict(kv__table=0), "missing pointer"), (dict(row_slot=0), "missing pointer"),
    (dict(row_pos=0), "missing pointer"), (dict(q=BUF + 4), "aligned"), (dict(out=BUF + 2), "aligned"),
    (dict(kv__arena=BUF + 8), "aligned"), (dict(scratch=0), "scratch"), (dict(scratch_floats=16), "scratch"),
    (dict(scratch=BUF + 4), "aligned"),
])
def test_attention_refuses(over, why):
    assert _lib.load().stride_serve_window_attention(C.byref(attention(**over)), None) == _lib.EINVAL
    assert why in err()


def test_attention_empty_and_null():
    lib = _lib.load()
    p = attention(l__rows=0, l__lane_groups=0, q=0, out=0)
    assert lib.stride_serve_window_attention(C.byref(p), None) == 0
    assert lib.stride_serve_window_attention(None, None) == _lib.EINVAL
    assert lib.stride_serve_window_attention_scratch(None) == -1
    assert lib.stride_serve_window_attention_scratch(C.byref(attention(n_q=17))) == -1


def test_attention_scratch_is_bounded_by_the_sight():
    """A window bounds the leaves that a row sees, and with them the scratch."""
    size = lambda **o: _lib.load().stride_serve_window_attention_scratch(C.byref(attention(runs=1, **o)))
    everything = size(max_pages=512, kv__max_blocks=2048)
    assert everything > 0 and everything % (4 * 8 * 128) == 0  # 32768 positions: 128 leaves of 4 rows and 8 groups
    one = everything // 128
    assert size(max_pages=512, kv__max_blocks=2048, window=1) == 0  # one leaf: nothing to join
    assert size(max_pages=512, kv__max_blocks=2048, window=257) == 0  # two: the row goes through them itself
    assert size(max_pages=512, kv__max_blocks=2048, window=258) == 3 * one  # two borders can lie in it
    assert size(max_pages=512, kv__max_blocks=2048, window=257, sinks=4) == 3 * one
    assert size(max_pages=512, kv__max_blocks=64) == 4 * one  # 1024 positions are all there is
    assert size(max_pages=1 << 30, kv__max_blocks=2048) == everything


def pool(**over):
    p = _lib.KvPoolParams()
    p.kv = _lib.KvRef(BUF, BUF, 2 * 2 * 8 * 16 * 64, 2 * 8 * 16 * 64, 8 * 16 * 64, 16 * 64, 64, 64)
    p.refs = p.free_bits = p.errors = p.work = BUF
    p.pages, p.slots, p.layers, p.n_kv, p.elem_bytes = 100, 8, 2, 8, 2
    p.work_ints = _lib.load().stride_kv_work_ints(8, 64, 100)
    for k, v in over.items():
        obj = p
        *path, last = k.split("__")
        for x in path:
            obj = getattr(obj, x)
        setattr(obj, last, v)
    return p


POOL_CALLS = {
    "reserve": lambda lib, p, n=2, a=BUF: lib.stride_kv_reserve(p, a, BUF, BUF, n, None),
    "release": lambda lib, p, n=2, a=BUF: lib.stride_kv_release(p, a, BUF, BUF, n, None),
    "fork": lambda lib, p, n=2, a=BUF: lib.stride_kv_fork(p, a, BUF, BUF, n, None),
    "compact": lambda lib, p, n=2, a=BUF: lib.stride_kv_compact(p, a, BUF, BUF, BUF, 4, 4, n, None),
    "copy": lambda lib, p, n=2, a=BUF: lib.stride_kv_copy(p, None, a, BUF, None, n, None),
}


@pytest.mark.parametrize("call", POOL_CALLS)
@pytest.mark.parametrize("over", [
    dict(elem_bytes=1), dict(pages=0), dict(slots=0), dict(slots=131073), dict(layers=0), dict(n_kv=0), dict(kv__max_blocks=0),
    dict(kv__group_elems=24 * 64), dict(kv__group_elems=0), dict(kv__head_dim=4, kv__group_elems=64), dict(kv__block_elems=12),
    dict(kv__layer_elems=4), dict(kv__which_elems=2), dict(kv__max_blocks=1 << 27), dict(layers=65536), dict(kv__arena=0),
    dict(kv__table=0), dict(refs=0), dict(free_bits=0), dict(errors=0), dict(work=0), dict(work_ints=100), dict(kv__arena=BUF + 8),
])
def test_pool_refuses(call, over):
    lib = _lib.load()
    p = pool(**over)
    assert POOL_CALLS[call](lib, C.byref(p)) == _lib.EINVAL, err()
    assert "kv_" + call in err()


@pytest.mark.parametrize("call", POOL_CALLS)
def test_pool_items(call):
    lib = _lib.load()
    p = pool()
    at = C.byref(p)
    assert POOL_CALLS[call](lib, at, n=0) == 0
    assert POOL_CALLS[call](lib, at, n=-1) == _lib.EINVAL
    assert POOL_CALLS[call](lib, at, a=None) == _lib.EINVAL and "missing pointer" in err()
    assert POOL_CALLS[call](lib, None) == _lib.EINVAL
    if call in ("reserve", "fork", "compact"):
        assert POOL_CALLS[call](lib, at, n=9) == _lib.EINVAL and "more items than slots" in err()


def test_pool_copy_between_unlike_pools_is_refused():
    lib = _lib.load()
    p, q = pool(), pool(layers=1, kv__block_elems=2 * 8 * 16 * 64)
    assert lib.stride_kv_copy(C.byref(p), C.byref(q), BUF, BUF, None, 1, None) == _lib.EINVAL and "shape" in err()
    q = pool(pages=100000, work_ints=10**9)
    assert lib.stride_kv_copy(C.byref(p), C.byref(q), BUF, BUF, None, 1, None) == _lib.EINVAL and "too large" in err()
    assert lib.stride_kv_work_ints(0, 1, 1) == -1 and lib.stride_kv_work_ints(1, 1, 0) == -1


def process(**over):
    p = _lib.LogitsParams()
    p.l = _lib.Lanes(20, 2, 0, 0)
    p.logits = p.best = p.scratch = BUF
    p.vocab = 1000
    for k, v in over.items():
        obj = p
        *path, last = k.split("__")
        for x in path:
            obj = getattr(obj, x)
        setattr(obj, last, v)
    return p


@pytest.mark.parametrize("over,why", [
    (dict(l__rows=-1), "rows >= 0"), (dict(l__lane_groups=1), "lane_groups"), (dict(vocab=0), "vocab"), (dict(logits=0), "missing"),
    (dict(best=0), "missing"), (dict(scratch=0), "missing"), (dict(counts=BUF), "counts need"),
    (dict(counts=BUF, seen=BUF, row_slot=BUF, penalties=BUF), "counts need"), (dict(bias_offsets=BUF), "bias_offsets need"),
    (dict(mask=BUF), "a mask needs"), (dict(mask=BUF, mask_row=BUF), "a mask needs"), (dict(logits=BUF + 4), "aligned"),
    (dict(out=BUF + 8), "aligned"), (dict(vocab=2**31 - 1), "vocab"),
])
def test_logits_refuse(over, why):
    assert _lib.load().stride_logits_process(C.byref(process(**over)), None) == _lib.EINVAL
    assert why in err()


def test_logits_empty_and_sizes():
    lib = _lib.load()
    p = process(l__rows=0, l__lane_groups=0, logits=0)
    assert lib.stride_logits_process(C.byref(p), None) == 0
    assert lib.stride_logits_process(None, None) == _lib.EINVAL
    assert [lib.stride_logits_scratch(n) for n in (-1, 0, 1, 16, 17)] == [-1, 0, logits.UNIT, logits.UNIT, 2 * logits.UNIT]
    c = _lib.TokenCountsParams(BUF, BUF, 4, 1000)
    assert lib.stride_logits_record(C.byref(c), None, None, 1, 0, 0, None) == 0
    assert lib.stride_logits_record(C.byref(c), BUF, BUF, -1, 1, 0, None) == _lib.EINVAL
    assert lib.stride_logits_record(None, BUF, BUF, 1, 1, 0, None) == _lib.EINVAL
    assert lib.stride_logits_reset(C.byref(c), None, None, 1, None) == _lib.EINVAL
    assert lib.stride_logits_reset(C.byref(_lib.TokenCountsParams(BUF, BUF, 0, 10)), BUF, None, 1, None) == _lib.EINVAL


def test_bias_lists_and_masks():
    o, t, v = logits.bias_lists([{7: 1.5, 2: -1.0}, None, {}, {5: 0.25}], "cpu")
    assert o.tolist() == [0, 2, 2, 2, 3] and t.tolist() == [2, 7, 5] and v.tolist() == [-1.0, 1.5, 0.25]
    o, t, v = logits.bias_lists([None], "cpu")
    assert o.tolist() == [0, 0]
    m = logits.mask_of([[0, 31, 32], [], [33]], 34, "cpu")
    assert m.tolist() == [[1 - (1 << 31), 1], [0, 0], [0, 2]]
    assert m.shape == (3, logits.words(34))


def test_existing_arena_is_checked():
    import torch

    arena, table = torch.zeros(4 * 2 * 2 * 16 * 32, dtype=torch.int16), torch.zeros((2, 2), dtype=torch.int32)
    kv = harness.PagedKv.over(arena, table, 2, 32, 1, 16)
    assert kv.slots == 2 and kv.capacity == 32 and kv.ref.block_elems == 2 * 2 * 16 * 32
    for a, t in ((arena[1:], table), (arena.float(), table), (arena, table.long()), (arena, table.t()), (arena, table[0])):
        with pytest.raises(ValueError):
            harness.PagedKv.over(a, t, 2, 32, 1, 16)


def test_scratch_without_a_hint_serves_every_hint():
    """The size for runs = 0 is no smaller than the one for any hint, over every form: short and
    long contexts, few and many rows, tiles split or whole."""
    size = _lib.load().stride_serve_window_attention_scratch
    wider = 0
    for rows in (1, 3, 4, 5, 16, 62, 100, 186, 220, 333, 1000, 2048):
        for n_kv, n_q, D in ((8, 4, 64), (8, 4, 128), (8, 1, 32), (2, 16, 64), (1, 7, 128), (16, 2, 32)):
            for ctx, window, sinks in ((200, 0, 0), (1500, 0, 0), (1969, 0, 0), (8192, 0, 0), (8192, 2100, 300), (40000, 0, 0), (40000, 64, 4)):
                for page in (8, 16, 64):
                    p = attention(l__rows=rows, l__lane_groups=(rows + 15) // 16, n_kv=n_kv, n_q=n_q, head_dim=D, kv__head_dim=D,
                                  kv__group_elems=page * D, kv__max_blocks=-(-ctx // page), max_pages=-(-ctx // 64), window=window,
                                  sinks=sinks, q_stride=n_kv * n_q * D, out_cols=n_kv * n_q * D)
                    at = C.byref(p)
                    most = size(at)
                    for runs in (1, 2, 3, 4, 5, 7, 8, 16, 31, 55, 62, 64, 200, rows - 1, rows, rows + 1, 2 ** 31 - 1):
                        if runs < 1:
                            continue
                        p.runs = runs
                        assert size(at) <= most, (rows, n_kv, n_q, D, ctx, window, page, runs)
                        wider += size(at) < most
    assert wider  # a hint may want less


@pytest.mark.parametrize("D,tokens,ok", [(128, 1 << 24, True), (128, 1 << 25, False), (32, 1 << 26, True), (32, 1 << 27, False), (64, 1 << 30, False)])
def test_attention_pages_whose_offsets_pass_32_bits(D, tokens, ok):
    """A row's offset in a head's part of a page is an int."""
    p = attention(head_dim=D, kv__head_dim=D, kv__group_elems=tokens * D, kv__which_elems=8 * tokens * D, kv__layer_elems=16 * tokens * D,
                  kv__block_elems=16 * tokens * D, kv__max_blocks=1, q_stride=32 * D, out_cols=32 * D)
    want = _lib.load().stride_serve_window_attention_scratch(C.byref(p))
    assert (want >= 0) == ok
    if not ok:
        assert _lib.load().stride_serve_window_attention(C.byref(p), None) == _lib.EINVAL and "2^31" in err()


@pytest.mark.parametrize("call", POOL_CALLS)
@pytest.mark.parametrize("D,elem,tokens,ok", [(64, 2, 1 << 23, True), (64, 2, 1 << 24, False), (64, 4, 1 << 22, True), (64, 4, 1 << 23, False)])
def test_pool_pages_whose_bytes_pass_32_bits(call, D, elem, tokens, ok):
    """Bytes of a head's part of a page are an int, and a copy's loop runs up to 1 KiB past them."""
    group = tokens * D
    p = pool(kv__head_dim=D, kv__group_elems=group, kv__which_elems=8 * group, kv__layer_elems=16 * group, kv__block_elems=32 * group,
             elem_bytes=elem, kv__max_blocks=8)
    assert POOL_CALLS[call](_lib.load(), C.byref(p), n=0) == (0 if ok else _lib.EINVAL)
    if not ok:
        assert "2^30" in err()
