"""Calls of stride_amd.mx at the borders of what they were given: rows beyond the page table or the rope
table, results beside and on their operands."""
import numpy as np
import pytest
import torch

import test_gpu_mx as plain
from stride_amd import harness, layout, mx
from stride_amd._lib import StrideTcError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("m", [5, 200, 1500])
def test_qkv_rows_beyond_the_tables(m):
    """The cache is whole pages, so that its last one can hold positions which a rope table of the
    context's length has no row for; and a slot can lie behind the page table. Such rows are left
    out. (Both tables are the first rows of longer ones here, whose other rows would be taken.)"""
    print("beyond", m, flush=True)
    rng = np.random.default_rng(m + 1)
    ws, _, x, kv, slot, pos, rope = plain.qkv_case(rng, m, 8, 2, 64, 512, slots=11)
    slot %= 8
    at = rng.permutation(8 * 200)[:m]  # places of their own
    slot, pos = (at // 200).astype(np.int32), (at % 200).astype(np.int32)
    bad = rng.permutation(m)[: m // 2]
    kv = harness.PagedKv(kv.arena, kv.table[:8], kv.ref, kv.page_tokens, kv.max_blocks)
    long_rope = plain.dev(np.concatenate([rope, np.full((100, 32, 2), 3.0, np.float32)]))
    q = torch.full((m, 512), 99.0, device=DEV)
    mx.qkv(*ws, x, m, 64, long_rope[:200], plain.dev(slot), plain.dev(pos), kv, layer=1, q_out=q)
    want_q, want = q.clone(), kv.arena.clone()
    for j in bad:  # what the whole call kept of them, taken away
        base = int(kv.table[slot[j], pos[j] // 16]) * kv.ref.block_elems + kv.ref.layer_elems + int(pos[j] % 16) * 64
        for which in (0, 1):
            for h in (0, 1):
                first = base + which * kv.ref.which_elems + h * kv.ref.group_elems
                want[first:first + 64] = 0
    want_q[plain.dev(bad)] = 99
    for i, j in enumerate(bad):
        if i % 3 == 0:
            pos[j] = 200 + i % 8
        elif i % 3 == 1:
            slot[j] = 8 + i % 3
        else:
            slot[j], pos[j] = 8 + i % 3, 207
    kv.arena.zero_()
    q.fill_(99.0)
    mx.qkv(*ws, x, m, 64, long_rope[:200], plain.dev(slot), plain.dev(pos), kv, layer=1, q_out=q)
    assert torch.equal(q, want_q) and torch.equal(kv.arena, want)
    # with the whole of both tables they have their places again
    whole = harness.PagedKv.over(kv.arena, kv.table._base if kv.table._base is not None else kv.table, 2, 64, 2, 16)
    mx.qkv(*ws, x, m, 64, long_rope, plain.dev(slot), plain.dev(pos), whole, layer=1, q_out=q)
    assert whole.slots == 11 and not (q == 99).all(1).any()


def carved(buf, at, rows, cols, bits):
    """Tiles in a buffer of bytes from `at` on, codes then scales; and where they end."""
    like = mx.Tiles.create(rows, cols, bits, "cpu")
    c, s = like.codes.numel(), like.scales.numel()
    return mx.Tiles(buf[at:at + c].view(like.codes.shape), buf[at + c:at + c + s].view(like.scales.shape), cols, bits), at + c + s


@pytest.mark.parametrize("m,n,k", [(5, 96, 528), (300, 1040, 528)])
def test_results_beside_their_operands(m, n, k):
    """Operands and results end to end in one buffer, as a workspace is dealt out, have the bits that
    they have in buffers of their own; a byte less and they are refused."""
    print("beside", m, n, k, flush=True)
    rng = np.random.default_rng(m)
    w, w3, x = plain.held(plain.weights_of(rng, n, k), 4), plain.held(plain.weights_of(rng, n, k), 4), plain.held(plain.acts_of(rng, m, k), 8)
    want_y, want_z = mx.gemm(w, x, m), mx.mlp13(w, w3, x, m)
    T = (m + 15) // 16
    buf = torch.zeros(64 << 20, dtype=torch.uint8, device=DEV)
    bx, at = carved(buf, 0, m, k, 8)
    bz, at = carved(buf, at, m, n, 8)
    bw, at = carved(buf, at, n, k, 4)
    y = buf[at:at + T * 16 * n * 2].view(torch.int16).view(T, n // 16, 16, 16)
    at += T * 16 * n * 2
    bw3, at = carved(buf, at, n, k, 4)
    for t, of in ((bx, x), (bw, w), (bw3, w3)):
        t.codes.copy_(of.codes)
        t.scales.copy_(of.scales)
    mx.gemm(bw, bx, m, out=y)
    mx.mlp13(bw, bw3, bx, m, out=bz)
    live = lambda a: layout.untile_lanes(a.cpu(), m)
    assert torch.equal(live(y), live(want_y))
    for a, b in ((bz, want_z),):
        got, want = plain.mx_plain.unpack(a.codes.cpu().numpy(), a.scales.cpu().numpy(), 8), plain.mx_plain.unpack(b.codes.cpu().numpy(), b.scales.cpu().numpy(), 8)
        assert all(np.array_equal(p[:m], q[:m]) for p, q in zip(got, want))
    back = mx.dequantize(bx, m, out=buf[at:at + m * k * 2].view(torch.bfloat16).view(m, k))
    assert torch.equal(back, mx.dequantize(x, m))
    last, _ = carved(buf, x.nbytes - 16, m, n, 8)
    with pytest.raises(StrideTcError, match="overlap"):
        mx.mlp13(bw, bw3, bx, m, out=last)
    with pytest.raises(StrideTcError, match="overlap"):
        mx.gemm(bw, bx, m, out=buf[x.nbytes - 16:x.nbytes - 16 + y.numel() * 2].view(torch.int16).view(y.shape))


@pytest.mark.parametrize("m,dim", [(5, 528), (300, 2064), (600, 8208), (5, 33296)])
def test_norm_in_the_place_of_its_addition(m, dim):
    """bf16 x tiles written over `add`: the bits of a result of its own."""
    print("in place", m, dim, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(dim)
    T = (m + 15) // 16
    h = torch.randn((T, dim // 16, 16, 16), generator=gen, device=DEV)
    add = torch.randn(h.shape, generator=gen, device=DEV).to(torch.bfloat16)
    gain = torch.rand(dim, generator=gen, device=DEV)
    h2 = h.clone()
    want = mx.norm(h, m, gain, 1e-5, add=add, bits=16)
    got = mx.norm(h2, m, gain, 1e-5, add=add, out=add, bits=16).view(torch.int16)
    assert torch.equal(h, h2) and torch.equal(layout.untile_lanes(got.cpu(), m), layout.untile_lanes(want.cpu(), m))
    with pytest.raises(StrideTcError, match="overlap"):
        mx.norm(h, m, gain, 1e-5, out=h.view(torch.int16).view(-1)[:add.numel()].view(add.shape), bits=16)


def test_arguments_of_another_kind_are_refused_by_a_message():
    """As without a GPU, for the arguments that are looked at after the device; and rows that an operand
    does not have are refused before a result of their size is made."""
    x, w, y = mx.Tiles.create(20, 512, 8, DEV), mx.Tiles.create(64, 512, 4, DEV), torch.zeros((2, 4, 16, 16), dtype=torch.int16, device=DEV)
    h, gain, z = torch.zeros((2, 32, 16, 16), device=DEV), torch.ones(512, device=DEV), mx.Tiles.create(20, 64, 8, DEV)
    kv = harness.PagedKv.create(1, 32, 1, 32, 1, 16, DEV)
    narrow = mx.Tiles.create(32, 512, 4, DEV)
    rope, at = torch.zeros((32, 16, 2), device=DEV), torch.zeros(20, dtype=torch.int32, device=DEV)
    good = dict(wq=w, wk=narrow, wv=narrow, x=x, rows=20, head_dim=32, rope=rope, row_slot=at, row_pos=at, kv=kv)
    mx.qkv(**good)
    for bad, why in ((lambda: mx.gemm(h, x, 20), "w must"), (lambda: mx.gemm(w, x, 20, out=z), "out must"), (lambda: mx.gemm(w, x, 20, out=[y]), "out must"),
                     (lambda: mx.mlp13(h, w, x, 20), "w1 must"), (lambda: mx.mlp13(w, None, x, 20), "w3 must"), (lambda: mx.mlp13(w, w, x, 20, out=y), "out must"),
                     (lambda: mx.quantize(h, out=h), "out must"), (lambda: mx.dequantize(x, out=x), "out must"), (lambda: mx.norm(h, 20, x, 1e-5), "weight must"),
                     (lambda: mx.norm(h, 20, gain, 1e-5, add=x), "add must"), (lambda: mx.norm(h, 20, gain, 1e-5, bits=16, out=x), "out must"),
                     (lambda: mx.norm(h, 20, gain, 1e-5, out=y), "out must"), (lambda: mx.qkv(**{**good, "wq": h}), "wq must"),
                     (lambda: mx.qkv(**{**good, "rope": x}), "rope must"), (lambda: mx.qkv(**{**good, "row_pos": [0] * 20}), "row_pos must"),
                     (lambda: mx.qkv(**{**good, "kv": kv.ref}), "kv must"), (lambda: mx.qkv(**{**good, "q_out": x}), "q_out must"),
                     *((call, "must be") for rows in (-1, -100, 33, 10 ** 12) for call in (
                         lambda rows=rows: mx.gemm(w, x, rows), lambda rows=rows: mx.mlp13(w, w, x, rows), lambda rows=rows: mx.quantize(h, rows, bits=8),
                         lambda rows=rows: mx.dequantize(x, rows), lambda rows=rows: mx.norm(h, rows, gain, 1e-5),
                         lambda rows=rows: mx.norm(h, rows, gain, 1e-5, bits=16), lambda rows=rows: mx.qkv(**{**good, "rows": rows})))):
        with pytest.raises(ValueError, match=why):
            bad()


@pytest.mark.parametrize("m,n", [(3, 48), (260, 1040), (520, 1040), (1100, 2064)])
def test_the_longest_rows(m, n):
    """K = 2^20 in each kind of product: small whole numbers, whose sums fp32 holds exactly (2^20 products of
    at most 18, of either sign: far below 2^24), so that y is the exact sum rounded once; and their blocks
    there and back."""
    print("longest", m, n, flush=True)
    k = 1 << 20
    gen = torch.Generator(device=DEV).manual_seed(m)
    ints = lambda rows, most: torch.randint(-most, most + 1, (rows, k), generator=gen, device=DEV, dtype=torch.int8)
    a, b = ints(n, 3), ints(m, 6)  # e2m1 has all of these, e4m3 too
    tiles = lambda v: layout.lane_tiles(v.to(torch.bfloat16))
    w, x = mx.quantize(tiles(a)), mx.quantize(tiles(b), m, bits=8)
    y = layout.untile_lanes(mx.gemm(w, x, m), m).view(torch.bfloat16)
    want = torch.zeros((m, n), dtype=torch.float64, device=DEV)
    for at in range(0, k, 1 << 15):  # float32 holds each part exactly
        want += (b[:, at:at + (1 << 15)].float() @ a[:, at:at + (1 << 15)].float().t()).double()
    assert want.abs().max() < 2 ** 24 and torch.equal(y, want.float().to(torch.bfloat16))
    for t, v in ((w, a), (x, b)):
        rows = min(64, len(v))
        assert torch.equal(mx.dequantize(t, rows), v[:rows].to(torch.bfloat16))
