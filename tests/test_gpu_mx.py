"""stride_amd.mx against plain forms in 64 bits (mx_plain): blocks bit for bit, the norm and the
products within the roundings that they take; rows that do not depend on their batch; capture,
streams, refusals."""

import numpy as np
import pytest
import torch

import mx_plain
from stride_amd import harness, layout, mx, tc
from stride_amd._lib import StrideTcError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def say(*a):
    print(*a, flush=True)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def bf16(a):
    """float64 -> the nearest bf16, as float64."""
    return torch.from_numpy(np.asarray(a, np.float32)).to(torch.bfloat16).double().numpy()


def tiles_of(a, dtype):
    """float64 [rows][cols] -> device tiles; lanes behind the rows hold 99."""
    rows, cols = a.shape
    full = np.full((-(-rows // 16) * 16, cols), 99.0)
    full[:rows] = a
    return layout.lane_tiles(torch.from_numpy(full).to(dtype)).to(DEV)


def marked(rows, cols, bits, fill=0xA5):
    t = mx.Tiles.create(rows, cols, bits, DEV)
    t.codes.fill_(fill)
    t.scales.fill_(fill)
    return t


def held(a, bits):
    """float64 [rows][cols] -> Tiles, its rows behind the last marked as a buffer's may be."""
    code, byte = mx_plain.encode(a, bits)
    codes, scales = mx_plain.pack(code, byte, bits)
    t = mx.Tiles(dev(codes), dev(scales), a.shape[1], bits)
    if a.shape[0] % 16:
        last = t.codes[-1].reshape(t.codes.shape[1], -1, 16, 16)
        last[:, :, a.shape[0] % 16:] = 0xFF
        t.scales[-1][:, :, a.shape[0] % 16:] = 0xFF
    return t


def same_blocks(t, a, rows):
    """Codes, scales and filling are those of `a`; rows behind are as marked."""
    codes, scales = mx_plain.pack(*mx_plain.encode(a, t.bits), t.bits)
    got_c, got_s = t.codes.cpu().numpy(), t.scales.cpu().numpy()
    full = rows % 16 == 0
    n = got_c.shape[0] if full else got_c.shape[0] - 1
    n = min(n, rows // 16)
    assert np.array_equal(got_c[:n], codes[:n]) and np.array_equal(got_s[:n], scales[:n])
    if not full:
        k = rows % 16
        c, w = (x[rows // 16].reshape(x.shape[1], -1, 16, 16) for x in (got_c, codes))
        assert np.array_equal(c[:, :, :k], w[:, :, :k]) and (c[:, :, k:] == 0xA5).all()
        assert np.array_equal(got_s[rows // 16][:, :, :k], scales[rows // 16][:, :, :k]) and (got_s[rows // 16][:, :, k:] == 0xA5).all()


def weights_of(rng, n, k):
    return bf16(rng.standard_normal((n, k)) * 0.02)


def acts_of(rng, m, k):
    a = rng.standard_normal((m, k))
    a[:, rng.random(k) < 0.01] *= 10
    return a


# --- blocks -----------------------------------------------------------------

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 16), (3, 32), (15, 48), (16, 512), (17, 528), (33, 2064), (130, 1040)])
def test_quantize(bits, dtype, rows, cols):
    say("quantize", bits, dtype, rows, cols)
    rng = np.random.default_rng(rows * 10000 + cols + bits)
    a = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-20, 20, (rows, 1))
    a[rng.random((rows, cols)) < 0.2] = 0
    a[:, : cols // 3] = 0
    a = torch.from_numpy(a).to(dtype).double().numpy()
    out = marked(rows, cols, bits)
    src = tiles_of(a, dtype)
    assert mx.quantize(src, rows, bits=bits, out=out) is out
    same_blocks(out, a, rows)
    for to in (torch.bfloat16, torch.float32):
        v = mx.dequantize(out, rows, dtype=to)
        want = torch.from_numpy(mx_plain.values(out, rows, cols)).to(to)
        assert v.dtype == to and torch.equal(v.cpu(), want)
    fresh = mx.quantize(src.view(torch.int16) if dtype == torch.bfloat16 else src, rows, bits=bits)
    assert torch.equal(fresh.codes.cpu()[: rows // 16], out.codes.cpu()[: rows // 16])


@pytest.mark.parametrize("bits", [4, 8])
def test_borders_of_the_formats(bits):
    """Each tie of the elements and of the scale rule, the smallest and largest numbers, zeros of both
    signs, and blocks that are not finite."""
    f32 = np.float32
    top, up = (6.0, 7.0) if bits == 4 else (448.0, 464.0)
    table = mx_plain.E2M1 if bits == 4 else mx_plain.E4M3
    rows = []
    for most in (top, np.nextafter(f32(up), f32(0)), up, np.nextafter(f32(up), f32(1e9)), top * 4 / 3):
        for e in (-126, -30, 0, 30):
            ties = (table[1:] + table[:-1]) / 2
            r = np.resize(np.concatenate([table, ties, np.nextafter(ties.astype(f32), f32(0)), np.nextafter(ties.astype(f32), f32(1e9))]), 512)
            r = np.where(r < most, r, 0.0).reshape(16, 32)
            r[:, 5] = -most
            r[:, 7] = -0.0
            rows.append(r.reshape(-1) * 2.0 ** e)
    tiny = np.zeros(512)
    tiny[:64] = 2.0 ** -149 * np.arange(64)
    tiny[64:96] = 2.0 ** -127
    tiny[96:128] = np.finfo(f32).max
    tiny[128:160] = np.finfo(f32).min
    tiny[160:192] = 2.0 ** -126 * np.linspace(1, 500, 32)
    rows.append(tiny)
    for bad in (np.inf, -np.inf, np.nan):
        r = np.ones(512)
        r[[3, 300]] = bad
        rows.append(r)
    a = np.array(rows).astype(f32).astype(np.float64)
    out = marked(a.shape[0], 512, bits)
    mx.quantize(tiles_of(a, torch.float32), a.shape[0], bits=bits, out=out)
    same_blocks(out, a, a.shape[0])
    v = mx.dequantize(out, a.shape[0], dtype=torch.float32).cpu().numpy()
    want = mx_plain.values(out, a.shape[0], 512)
    assert np.array_equal(np.isnan(v), np.isnan(want)) and np.isnan(v[-3:, :32]).all() and (v[-3:, 32:256] == 1).all()
    assert np.array_equal(np.nan_to_num(v.astype(np.float64)), np.nan_to_num(want.astype(f32).astype(np.float64)))


def test_dequantize_into_strided_rows():
    rng = np.random.default_rng(3)
    a = acts_of(rng, 21, 208)
    t = held(a, 8)
    wide = torch.full((30, 256), 7.0, device=DEV)
    mx.dequantize(t, 21, dtype=torch.float32, out=wide[:, :208])
    assert np.array_equal(wide[:21, :208].cpu().numpy().astype(np.float64), mx_plain.values(t, 21, 208))
    assert (wide[21:] == 7).all() and (wide[:, 208:] == 7).all()


# --- the norm -----------------------------------------------------------------

def norm_want(h, add, gain, eps):
    h = h if add is None else (h.astype(np.float32) + add.astype(np.float32)).astype(np.float64)
    return h, h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * gain


@pytest.mark.parametrize("with_add", [False, True])
@pytest.mark.parametrize("rows,dim", [(1, 16), (2, 48), (16, 256), (5, 512), (17, 528), (33, 2048), (3, 2064), (9, 4096), (6, 8192), (2, 8208), (3, 17424)])
def test_norm(rows, dim, with_add):
    """h is exact. An element is off by half a step of e4m3 at its scale (2^-4 of it, or 2^-10 of the
    scale), and the value that is rounded by what fp32 loses: a sum of dim / (64 waves) squares a lane
    and 27 more additions, each 2^-24 of it, half of that after the root; six roundings around it."""
    say("norm", rows, dim, with_add)
    rng = np.random.default_rng(rows * 100000 + dim)
    h = acts_of(rng, rows, dim).astype(np.float32).astype(np.float64) * 3
    add = bf16(rng.standard_normal((rows, dim))) if with_add else None
    gain = (1 + 0.2 * rng.standard_normal(dim)).astype(np.float32).astype(np.float64)
    h2, want = norm_want(h.astype(np.float32).astype(np.float64), add, gain, 1e-5)
    e = ((dim / 1024 * 8 + 16 + 27) / 2 + 6) * 2.0 ** -24
    results = []
    for bits in (8, 16):
        ht = tiles_of(h, torch.float32)
        at = tiles_of(add, torch.bfloat16) if with_add else None
        out = marked(rows, dim, 8) if bits == 8 else tiles_of(np.zeros((rows, dim)), torch.bfloat16)
        assert mx.norm(ht, rows, dev(gain.astype(np.float32)), 1e-5, add=at, out=out, bits=bits) is out
        back = layout.untile_lanes(ht.cpu(), ht.shape[0] * 16)
        assert np.array_equal(back[:rows].numpy().astype(np.float64), h2) and (back[rows:] == 99).all()
        if bits == 8:
            code, byte = mx_plain.unpack(out.codes.cpu().numpy(), out.scales.cpu().numpy(), 8)
            low, high = (mx_plain.scale_bytes(mx_plain.wide(want * f), 8) for f in (1 - e, 1 + e))
            assert ((byte == low) | (byte == high))[:rows].all()
            got = mx_plain.decode(code, byte, 8)[:rows]
            assert (got[:, dim:] == 0).all() and (byte[rows:] == 0xA5).all() and (code[rows:] == 0xA5).all()
            got, scale = got[:, :dim], np.repeat(2.0 ** (byte[:rows] - 127.0), 32, 1)[:, :dim]
            tol = e * np.abs(want) + np.maximum(2.0 ** -4 * np.abs(want) * (1 + e), 2.0 ** -10 * scale)
        else:
            full = layout.untile_lanes(out.cpu(), out.shape[0] * 16).double().numpy()
            got, tol = full[:rows], (e + 2.0 ** -8 * (1 + e)) * np.abs(want) + 1e-38
            assert (full[rows:] == 99).all()
        assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
        results.append(out)
    # both are the same fp32 values: the 8-bit ones round to at most half a step from the bf16 ones' interval
    again = mx.norm(tiles_of(h2, torch.float32), rows, dev(gain.astype(np.float32)), 1e-5)
    assert torch.equal(again.codes[: rows // 16], results[0].codes[: rows // 16])


def test_norm_rows_that_are_zero_or_not_finite():
    h = np.ones((6, 512))
    h[1] = 0
    h[2, 100] = np.inf
    h[3, 7] = np.nan
    h[4] = 1e30  # the sum of squares is beyond fp32: the row's scale is 0
    got = mx_plain.values(mx.norm(tiles_of(h, torch.float32), 6, torch.ones(512, device=DEV), 1e-5), 6, 512)
    assert (got[0] == got[5]).all() and (got[1] == 0).all() and (got[4] == 0).all() and np.isnan(got[3]).all()
    assert np.isnan(got[2, 96:128]).all() and (got[2, :96] == 0).all()


def test_norm_of_any_nan():
    """NaN of every payload and sign stays NaN in both results, in its own row."""
    bits = torch.tensor([0x7FFFFFFF, -1, 0x7F800001, 0x7FC00000, -0x3FFFFF], dtype=torch.int32, device=DEV)
    h = torch.ones((1, 32, 16, 16), device=DEV)
    h.view(torch.int32)[0, 3, :5, 7] = bits
    for b in (8, 16):
        t = mx.norm(h, 16, torch.ones(512, device=DEV), 1e-5, bits=b)
        v = mx.dequantize(t).float() if b == 8 else layout.untile_lanes(t, 16).view(torch.bfloat16).float()
        assert v[:5].isnan().all() and (v[5:] == 1).all()


# --- products -----------------------------------------------------------------

SHAPES = [(1, 16, 16), (1, 256, 512), (16, 48, 528), (17, 512, 2048), (33, 1040, 1040), (5, 2048, 8192), (64, 512, 2560), (130, 256, 4112),
          (290, 528, 2048), (700, 272, 1536)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm(m, n, k):
    say("gemm", m, n, k)
    rng = np.random.default_rng(m + n + k)
    w, x = held(weights_of(rng, n, k), 4), held(acts_of(rng, m, k), 8)
    wv, xv = mx_plain.values(w, n, k), mx_plain.values(x, m, k)
    out = tiles_of(np.zeros((m, n)), torch.bfloat16)
    assert mx.gemm(w, x, m, out=out) is out
    full = layout.untile_lanes(out.cpu(), out.shape[0] * 16).double().numpy()
    want, e = xv @ wv.T, mx_plain.products_bound(wv, xv)
    tol = e + 2.0 ** -8 * (np.abs(want) + e)
    assert (np.abs(full[:m] - want) <= tol).all(), (np.abs(full[:m] - want) / tol).max()
    assert (full[m:] == 99).all()


@pytest.mark.parametrize("m,n,k", [(1, 16, 16), (3, 48, 512), (17, 512, 2048), (33, 528, 1040), (130, 1040, 2064), (290, 272, 2048), (513, 512, 512)])
def test_mlp13(m, n, k):
    """The error of both products through silu(g) u (|silu'| <= 1.1, |silu(g)| <= |g|), fp32 roundings,
    then half a step of e4m3."""
    say("mlp13", m, n, k)
    rng = np.random.default_rng(m + n + k)
    w1, w3, x = held(weights_of(rng, n, k), 4), held(weights_of(rng, n, k), 4), held(acts_of(rng, m, k), 8)
    v1, v3, xv = mx_plain.values(w1, n, k), mx_plain.values(w3, n, k), mx_plain.values(x, m, k)
    out = marked(m, n, 8)
    assert mx.mlp13(w1, w3, x, m, out=out) is out
    code, byte = mx_plain.unpack(out.codes.cpu().numpy(), out.scales.cpu().numpy(), 8)
    g, u = xv @ v1.T, xv @ v3.T
    eg, eu = mx_plain.products_bound(v1, xv), mx_plain.products_bound(v3, xv)
    silu = g / (1 + np.exp(-g))
    want = silu * u
    e = 1.1 * eg * (np.abs(u) + eu) + np.abs(silu) * eu + 2.0 ** -20 * np.abs(want)
    got, scale = mx_plain.decode(code, byte, 8), np.repeat(2.0 ** (byte - 127.0), 32, 1)
    assert (got[:m, n:] == 0).all() and (code[m:] == 0xA5).all() and (byte[m:] == 0xA5).all()
    got, scale = got[:m, :n], scale[:m, :n]
    tol = e + np.maximum(2.0 ** -4 * (np.abs(want) + e), 2.0 ** -10 * scale)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
    most = np.abs(mx_plain.wide(np.abs(want) + e)).reshape(-1, out.codes.shape[1] * 4, 32).max(-1)[:m]
    assert (2.0 ** (byte[:m] - 127.0) <= np.maximum(most / 230, 2.0 ** -127)).all(), "no scale is larger than it has to be"


def qkv_case(rng, m, heads, kv_heads, D, k, page=16, slots=3, ctx=200):
    nq, nkv = heads * D, kv_heads * D
    order = [layout.rope_rows(nq, D), layout.rope_rows(nkv, D), layout.rope_rows(nkv, D)]
    raw = [weights_of(rng, len(o), k) for o in order]
    ws = [held(r[o], 4) for r, o in zip(raw, order)]
    vals = []
    for w, o in zip(ws, order):
        v = np.empty((len(o), k))
        v[o] = mx_plain.values(w, len(o), k)
        vals.append(v)
    x = held(acts_of(rng, m, k), 8)
    kv = harness.PagedKv.create(slots, ctx, kv_heads, D, 2, page, DEV, shuffle_seed=5)
    at = rng.permutation(slots * ctx)[:m]
    slot, pos = (at // ctx).astype(np.int32), (at % ctx).astype(np.int32)
    angle = np.arange(ctx)[:, None] * 10000.0 ** (-np.arange(D // 2) * 2 / D)
    rope = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    return ws, vals, x, kv, slot, pos, rope


def rotated(y, pos, rope, D):
    y = y.reshape(y.shape[0], -1, D)
    c, s = (rope[pos][:, None, :, i].astype(np.float64) for i in range(2))
    a, b = y[..., : D // 2], y[..., D // 2:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1).reshape(y.shape[0], -1)


@pytest.mark.parametrize("m,heads,kv_heads,D,k,page", [(1, 4, 1, 32, 64, 16), (5, 8, 2, 64, 512, 16), (37, 4, 4, 128, 1040, 64), (130, 16, 4, 64, 2048, 8),
                                                        (300, 8, 2, 64, 1536, 16)])
def test_qkv(m, heads, kv_heads, D, k, page):
    """q in fp32, K and V rounded once to bf16; besides the bound of each sum, Gaussian data's 2-norm
    error, which is that of many independent cut-offs: below 2e-5."""
    say("qkv", m, heads, kv_heads, D, k)
    rng = np.random.default_rng(m + D)
    ws, vals, x, kv, slot, pos, rope = qkv_case(rng, m, heads, kv_heads, D, k, page)
    q = torch.full((m + 2, heads * D), 99.0, device=DEV)
    before = kv.arena.clone()
    mx.qkv(*ws, x, m, D, dev(rope), dev(slot), dev(pos), kv, layer=1, q_out=q)
    xv = mx_plain.values(x, m, k)
    bound = [mx_plain.products_bound(v, xv) for v in vals]
    mate = lambda e: e + np.roll(e.reshape(m, -1, D), D // 2, 2).reshape(m, -1)  # a pair's errors add up
    want = rotated(xv @ vals[0].T, pos, rope, D)
    got = q[:m].cpu().numpy().astype(np.float64)
    far = np.abs(xv) @ np.abs(vals[0]).T
    assert (np.abs(got - want) <= mate(bound[0] + 2.0 ** -22 * far)).all() and (q[m:] == 99).all()
    if k >= 512:
        assert np.linalg.norm(got - want) <= 2e-5 * np.linalg.norm(want)
    for which, (v, b) in enumerate(zip(vals[1:], bound[1:])):
        got = kv.gather(1, which, slot, pos, kv_heads, D).view(torch.bfloat16).cpu().double().numpy()
        y = xv @ v.T
        want, e = (rotated(y, pos, rope, D), mate(b + 2.0 ** -22 * np.abs(xv) @ np.abs(v).T)) if which == 0 else (y, b)
        assert (np.abs(got - want) <= e + 2.0 ** -8 * (np.abs(want) + e) + 1e-38).all()
    rest = kv.arena.clone().view(-1, 2, kv.ref.layer_elems)
    assert torch.equal(rest[:, 0], before.view(-1, 2, kv.ref.layer_elems)[:, 0]), "the other layer is left alone"
    for which in (0, 1):
        kv.fill_dense(1, which, torch.zeros((3, kv_heads, 200, D), dtype=torch.int16, device=DEV))
    assert torch.equal(kv.arena, before)


@pytest.mark.parametrize("m", [5, 200, 1500])
def test_qkv_rows_without_a_place(m):
    """Padding rows of a captured batch (slot or position below 0), positions behind the table and
    entries without a page: the others' bits are as without them, in the cache and in q."""
    rng = np.random.default_rng(m)
    ws, _, x, kv, slot, pos, rope = qkv_case(rng, m, 8, 2, 64, 512, slots=8)
    rope = np.concatenate([rope, rope])
    q = torch.full((m, 512), 99.0, device=DEV)
    mx.qkv(*ws, x, m, 64, dev(rope), dev(slot), dev(pos), kv, layer=1, q_out=q)
    want_q, want = q.clone(), kv.arena.clone()
    bad = rng.permutation(m)[: m // 2]
    slot2, pos2 = slot.copy(), pos.copy()
    for i, j in enumerate(bad):
        if i % 4 == 0:
            slot2[j] = -1 - i
        elif i % 4 == 1:
            pos2[j] = -2 ** 31 + i
        elif i % 4 == 2:
            pos2[j] = 208 + i % 100
        else:
            slot2[j], pos2[j] = -2 ** 31, 2 ** 31 - 1
    kv.arena.zero_()
    q.fill_(99.0)
    args = (*ws, x, m, 64, dev(rope), dev(slot2), dev(pos2), kv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mx.qkv(*args, layer=1, q_out=q)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        mx.gemm(ws[0], x, m)
        rest = np.setdiff1d(np.arange(m), bad)
        assert torch.equal(q[dev(rest)], want_q[dev(rest)]) and (q[dev(bad)] == 99).all()
    for j in bad:  # what the whole call kept of them, taken away
        base = int(kv.table[slot[j], pos[j] // 16]) * kv.ref.block_elems + kv.ref.layer_elems + int(pos[j] % 16) * 64
        for which in (0, 1):
            for h in (0, 1):
                at = base + which * kv.ref.which_elems + h * kv.ref.group_elems
                want[at:at + 64] = 0
    assert torch.equal(kv.arena, want)
    kv.table.fill_(-1)
    kv.arena.zero_()
    mx.qkv(*ws, x, m, 64, dev(rope), dev(slot), dev(pos), kv, layer=1, q_out=q)
    assert torch.equal(q, want_q) and not kv.arena.any()


def test_rows_do_not_depend_on_their_batch():
    """The same bits alone, in any batch and in any order, over every form that a call can take."""
    rng = np.random.default_rng(11)
    for n, k in ((512, 2048), (2048, 2560)):
        m = 1100
        w, w3, a = held(weights_of(rng, n, k), 4), held(weights_of(rng, n, k), 4), acts_of(rng, m, k)
        x = held(a, 8)
        base = layout.untile_lanes(mx.gemm(w, x, m).cpu(), m)
        z = mx.mlp13(w, w3, x, m)
        zc, zs = mx_plain.unpack(z.codes.cpu().numpy(), z.scales.cpu().numpy(), 8)
        code, byte = mx_plain.encode(a, 8)
        for rows in (1, 5, 16, 17, 33, 64, 70, 128, 130, 200, 257, 300, 520, 700, 1030):
            say("batch", n, k, rows)
            pick = rng.permutation(m)[:rows]
            part_code, part_byte = np.zeros((-(-rows // 16) * 16, code.shape[1]), np.int64), np.zeros((-(-rows // 16) * 16, byte.shape[1]), np.int64)
            part_code[:rows], part_byte[:rows] = code[pick], byte[pick]
            px = mx.Tiles(*(dev(p) for p in mx_plain.pack(part_code, part_byte, 8)), k, 8)
            assert torch.equal(layout.untile_lanes(mx.gemm(w, px, rows).cpu(), rows), base[pick]), rows
            pz = mx.mlp13(w, w3, px, rows)
            c, s = mx_plain.unpack(pz.codes.cpu().numpy(), pz.scales.cpu().numpy(), 8)
            assert np.array_equal(c[:rows], zc[pick]) and np.array_equal(s[:rows], zs[pick]), rows


def test_rows_that_are_not_finite_keep_to_themselves():
    rng = np.random.default_rng(12)
    w, a = held(weights_of(rng, 512, 1024), 4), acts_of(rng, 40, 1024)
    good = layout.untile_lanes(mx.gemm(w, held(a, 8), 40).cpu(), 40)
    a[7, 3], a[20, 1000] = np.nan, np.inf
    x = held(a, 8)
    got = layout.untile_lanes(mx.gemm(w, x, 40).cpu(), 40)
    bad = [7, 20]
    rest = [i for i in range(40) if i not in bad]
    nan = got.view(torch.bfloat16).isnan()
    assert nan[bad].all() and torch.equal(got[rest], good[rest])
    z = mx_plain.values(mx.mlp13(w, w, x, 40), 40, 512)
    assert np.isnan(z[bad]).all() and np.isfinite(z[rest]).all()
    wv = weights_of(rng, 512, 1024)
    wv[9, 100] = np.nan
    y = layout.untile_lanes(mx.gemm(held(wv, 4), held(acts_of(rng, 40, 1024), 8), 40).cpu(), 40).view(torch.bfloat16)
    assert y[:, 9].isnan().all() and not torch.cat([y[:, :9], y[:, 10:]], 1).isnan().any()


# --- together -----------------------------------------------------------------

def layer_of(rng, H, F):
    return dict(w1=held(weights_of(rng, F, H), 4), w3=held(weights_of(rng, F, H), 4), w2=held(weights_of(rng, H, F), 4),
                gain=dev((1 + 0.1 * rng.standard_normal(H)).astype(np.float32)))


def test_mlp_half_captured_and_replayed():
    """Norm, gate and up, down, and the norm that adds it, in a graph: each replay, with eager work
    between them, has the eager call's bits."""
    rng = np.random.default_rng(13)
    m, H, F = 37, 512, 1040
    L = layer_of(rng, H, F)
    start = tiles_of(acts_of(rng, m, H), torch.float32)
    bufs = lambda: (start.clone(), mx.Tiles.create(m, H, 8, DEV), mx.Tiles.create(m, F, 8, DEV), torch.zeros((3, H // 16, 16, 16), dtype=torch.int16, device=DEV),
                    torch.zeros((3, H // 16, 16, 16), dtype=torch.int16, device=DEV))

    def half(h, x, z, y, out):
        mx.norm(h, m, L["gain"], 1e-5, out=x)
        mx.mlp13(L["w1"], L["w3"], x, m, out=z)
        mx.gemm(L["w2"], z, m, out=y)
        mx.norm(h, m, L["gain"], 1e-5, add=y, out=out, bits=16)

    eager, b = bufs(), bufs()
    half(*eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        half(*b)
    for k in range(4):
        b[0].copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(b, eager):
            assert all(torch.equal(s, t) for s, t in (((p.codes, q.codes), (p.scales, q.scales)) if isinstance(p, mx.Tiles) else ((p, q),))), k
        other = bufs()
        half(*other)
        torch.cuda.synchronize()


def test_streams():
    """Two streams at once, and a stream set by set_kernel_stream, for which results are passed."""
    rng = np.random.default_rng(14)
    w, x = held(weights_of(rng, 2048, 2048), 4), held(acts_of(rng, 64, 2048), 8)
    want = mx.gemm(w, x, 64)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(want) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                mx.gemm(w, x, 64, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    tc.set_kernel_stream(streams[0])
    try:
        for call in (lambda: mx.gemm(w, x, 64), lambda: mx.mlp13(w, w, x, 64), lambda: mx.quantize(want, 64), lambda: mx.dequantize(x),
                     lambda: mx.norm(torch.zeros((4, 128, 16, 16), device=DEV), 64, torch.ones(2048, device=DEV), 1e-5)):
            with pytest.raises(ValueError, match="pass out"):
                call()
        outs[0].zero_()
        torch.cuda.synchronize()
        mx.gemm(w, x, 64, out=outs[0])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want)
    finally:
        tc.set_kernel_stream(None)


def test_refusals():
    rng = np.random.default_rng(15)
    w, x = held(weights_of(rng, 64, 512), 4), held(acts_of(rng, 20, 512), 8)
    w2, narrow = held(weights_of(rng, 80, 512), 4), held(weights_of(rng, 64, 1024), 4)
    h, gain = torch.zeros((2, 32, 16, 16), device=DEV), torch.ones(512, device=DEV)
    half = torch.zeros((2, 32, 16, 16), dtype=torch.int16, device=DEV)
    y = torch.zeros((2, 4, 16, 16), dtype=torch.int16, device=DEV)
    host = mx.Tiles.create(20, 512, 8, "cpu")
    host_w = mx.Tiles.create(64, 512, 4, "cpu")
    for bad in (lambda: mx.gemm(w, w, 20), lambda: mx.gemm(x, x, 20), lambda: mx.gemm(narrow, x, 20), lambda: mx.gemm(w, x, 33),
                lambda: mx.gemm(w, host, 20), lambda: mx.gemm(host_w, x, 20), lambda: mx.gemm(w, x, 20, out=y[:1]), lambda: mx.gemm(w, x, 20, out=half),
                lambda: mx.gemm(w, x, 20, out=y.float()), lambda: mx.gemm(w, x, 20, out=y.cpu()), lambda: mx.gemm(w, x, -1),
                lambda: mx.mlp13(w, w2, x, 20), lambda: mx.mlp13(w2, w, x, 20), lambda: mx.mlp13(w, w, x, 20, out=mx.Tiles.create(20, 80, 8, DEV)),
                lambda: mx.mlp13(w, w, x, 20, out=mx.Tiles.create(16, 64, 8, DEV)), lambda: mx.mlp13(w, w, x, 20, out=mx.Tiles.create(20, 64, 4, DEV)),
                lambda: mx.quantize(h.double()), lambda: mx.quantize(h[:, :, :8]), lambda: mx.quantize(h.transpose(0, 1)), lambda: mx.quantize(h.cpu()),
                lambda: mx.quantize(h, 33), lambda: mx.quantize(h, bits=6), lambda: mx.quantize(h, out=x), lambda: mx.quantize(h, 20, bits=8, out=narrow),
                lambda: mx.dequantize(x, 33), lambda: mx.dequantize(x, dtype=torch.float16), lambda: mx.dequantize(x, out=torch.zeros((32, 512), device=DEV)),
                lambda: mx.dequantize(host), lambda: mx.norm(half, 20, gain, 1e-5), lambda: mx.norm(h, 33, gain, 1e-5), lambda: mx.norm(h, 20, gain[:500], 1e-5),
                lambda: mx.norm(h, 20, gain.double(), 1e-5), lambda: mx.norm(h, 20, gain.cpu(), 1e-5), lambda: mx.norm(h, 20, gain, 1e-5, add=h),
                lambda: mx.norm(h, 20, gain, 1e-5, add=half[:, :16].contiguous()), lambda: mx.norm(h, 20, gain, 1e-5, bits=4),
                lambda: mx.norm(h, 20, gain, 1e-5, out=half), lambda: mx.norm(h, 20, gain, 1e-5, bits=16, out=x), lambda: mx.norm(h.cpu(), 20, gain.cpu(), 1e-5)):
        with pytest.raises((ValueError, StrideTcError, AttributeError)):
            bad()
    ws, _, x, kv, slot, pos, rope = qkv_case(rng, 5, 4, 1, 32, 64)
    good = dict(wq=ws[0], wk=ws[1], wv=ws[2], x=x, rows=5, head_dim=32, rope=dev(rope), row_slot=dev(slot), row_pos=dev(pos), kv=kv, layer=1)
    mx.qkv(**good)
    for over in (dict(layer=2), dict(layer=-1), dict(rows=17), dict(head_dim=64), dict(rope=dev(rope).double()), dict(row_slot=dev(slot).long()),
                 dict(row_pos=dev(pos)[:3]), dict(row_pos=dev(pos).cpu()), dict(wk=ws[0]), dict(wv=ws[0]), dict(wq=x), dict(q_out=torch.zeros((5, 64), device=DEV)),
                 dict(q_out=torch.zeros((4, 128), device=DEV)), dict(q_out=torch.zeros((5, 128)))):
        with pytest.raises((ValueError, StrideTcError)):
            mx.qkv(**{**good, **over})


def test_no_rows():
    x = mx.Tiles.create(0, 512, 8, DEV)
    w = mx.Tiles.create(64, 512, 4, DEV)
    assert mx.gemm(w, x, 0).shape == (0, 4, 16, 16) and mx.mlp13(w, w, x, 0).tiles == 0
    h = torch.zeros((0, 32, 16, 16), device=DEV)
    assert mx.norm(h, 0, torch.ones(512, device=DEV), 1e-5).tiles == 0 and mx.quantize(h).tiles == 0 and mx.dequantize(x).shape == (0, 512)


def rows_alone(x, first, n):
    """Rows first * 16 .. of Tiles, as Tiles of their own."""
    return mx.Tiles(x.codes[first:first + n].contiguous(), x.scales[first:first + n].contiguous(), x.cols, x.bits)


@pytest.mark.parametrize("m,n,k", [
    (40, 2048, 512), (100, 256, 8192), (150, 2048, 4096), (200, 1024, 1024), (600, 2048, 1024), (1000, 1552, 528),
    (1400, 4096, 512), (1400, 2064, 2064), (2100, 4096, 8192), (440, 2064, 528), (870, 2064, 1040), (2600, 2064, 4112)])
def test_each_form_has_the_same_bits(m, n, k):
    """From waves of their own to 256 x 128 tiles, ragged ones among them: every row as in a batch of
    16, which is a wave's of its own; lanes behind the rows stay as they were."""
    say("forms", m, n, k)
    gen = torch.Generator(device=DEV).manual_seed(m + n + k)
    rand = lambda *s: torch.randn(s, generator=gen, device=DEV)
    ws = [mx.quantize(layout.lane_tiles((rand(n, k) * 0.05).to(torch.bfloat16))) for _ in range(2)]
    x = mx.quantize(layout.lane_tiles(rand(m, k).to(torch.bfloat16)), m, bits=8)
    T = (m + 15) // 16
    y = torch.full((T, n // 16, 16, 16), 99, dtype=torch.int16, device=DEV)
    z = marked(m, n, 8)
    mx.gemm(ws[0], x, m, out=y)
    mx.mlp13(*ws, x, m, out=z)
    D, kv_heads = 32, n // 64
    slots = torch.zeros(m, dtype=torch.int32, device=DEV)
    pos = torch.randperm(m, generator=gen, device=DEV).to(torch.int32)
    rope = rand(m, D // 2, 2)
    caches = [harness.PagedKv.create(1, m, kv_heads, D, 1, 16, DEV) for _ in range(2)]
    w_qkv = (ws[0], *(mx.Tiles(w.codes[: kv_heads * 2].contiguous(), w.scales[: kv_heads * 2].contiguous(), k, 4) for w in ws))
    q = torch.zeros((m, n), device=DEV) if n % D == 0 else None
    if q is not None:
        mx.qkv(*w_qkv, x, m, D, rope, slots, pos, caches[0], q_out=q)
    for t in range(T):
        rows = min(16, m - 16 * t)
        part = rows_alone(x, t, 1)
        y1 = torch.full((1, n // 16, 16, 16), 99, dtype=torch.int16, device=DEV)
        z1 = marked(rows, n, 8)
        mx.gemm(ws[0], part, rows, out=y1)
        mx.mlp13(*ws, part, rows, out=z1)
        assert torch.equal(y[t], y1[0]) and torch.equal(z.codes[t], z1.codes[0]) and torch.equal(z.scales[t], z1.scales[0]), t
        if q is not None:
            q1 = mx.qkv(*w_qkv, part, rows, D, rope, slots[:rows], pos[16 * t:16 * t + rows].contiguous(), caches[1])
            assert torch.equal(q[16 * t:16 * t + rows], q1), t
    assert torch.equal(caches[0].arena, caches[1].arena)


LONG = 2 ** 18 + 37  # rows of 16384 values: offsets beyond 32 bits, in bytes and in elements


def random_tiles(rows, cols, bits):
    t = mx.Tiles.create(rows, cols, bits, DEV)
    t.codes.random_(0, 256 if bits == 4 else 0x70)
    t.scales.random_(115, 125)
    return t


def tail(t, first):
    """The last tiles of a tensor or Tiles, in memory of their own."""
    if isinstance(t, mx.Tiles):
        return mx.Tiles(t.codes[first:].clone(), t.scales[first:].clone(), t.cols, t.bits)
    return t[first:].clone()


def same_ends(whole, part, first):
    """The last tiles of a long result are those of a call on these rows alone."""
    for a, b in ([(whole.codes, part.codes), (whole.scales, part.scales)] if isinstance(whole, mx.Tiles) else [(whole, part)]):
        assert torch.equal(a[first:], b)


def test_long_products():
    first, rows = 2 ** 14 - 3, 37 + 48
    say("x of 4 GiB")
    x, w = random_tiles(LONG, 16384, 8), random_tiles(48, 16384, 4)
    same_ends(mx.gemm(w, x, LONG), mx.gemm(w, tail(x, first), rows), first)
    say("y of 8 GiB")
    x, w = random_tiles(LONG, 512, 8), random_tiles(16384, 512, 4)
    same_ends(mx.gemm(w, x, LONG), mx.gemm(w, tail(x, first), rows), first)
    say("z of 4 GiB")
    w3 = random_tiles(16384, 512, 4)
    same_ends(mx.mlp13(w, w3, x, LONG), mx.mlp13(w, w3, tail(x, first), rows), first)


def test_long_values():
    first, rows = 2 ** 14 - 3, 37 + 48
    say("h of 16 GiB")
    h = torch.empty((2 ** 14 + 3, 1024, 16, 16), dtype=torch.float32, device=DEV).normal_()
    add = torch.empty(h.shape, dtype=torch.bfloat16, device=DEV).normal_()
    gains = torch.rand(16384, device=DEV)
    part = tail(h, first)
    same_ends(mx.norm(h, LONG, gains, 1e-5, add=add), mx.norm(part, rows, gains, 1e-5, add=tail(add, first)), first)
    live = torch.arange(h[first:].numel(), device=DEV).view(part.shape)
    live = (live // (1024 * 256) * 16 + live // 16 % 16) < rows
    assert torch.equal(h[first:][live], part[live])
    del h, part, live
    for bits in (4, 8):
        say("to", bits, "bits")
        t = mx.quantize(add, LONG, bits=bits)
        small = mx.quantize(tail(add, first), rows, bits=bits)
        same_ends(t, small, first)
        assert torch.equal(mx.dequantize(t, LONG)[first * 16:], mx.dequantize(small, rows))


@pytest.mark.parametrize("bits", [4, 8])
def test_many_values(bits):
    """Where a workgroup takes a whole group: the values that the same tiles have in small calls."""
    gen = torch.Generator(device=DEV).manual_seed(bits)
    m, k = 5003, 1552
    t = mx.quantize(layout.lane_tiles(torch.randn((m, k), generator=gen, device=DEV) * 3), m, bits=bits)
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((m + 1, k + 48), 7.0, dtype=dtype, device=DEV)
        mx.dequantize(t, m, dtype=dtype, out=out[:, :k])
        assert (out[m:] == 7).all() and (out[:, k:] == 7).all()
        for first in range(0, t.tiles, 40):
            part = rows_alone(t, first, 40)
            rows = min(part.rows, m - 16 * first)
            assert torch.equal(out[16 * first:16 * first + rows, :k], mx.dequantize(part, rows, dtype=dtype))
