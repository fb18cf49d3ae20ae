"""Calls of stride_amd.mx at the borders of what they were given: rows beyond the page table or the rope
table."""
import numpy as np
import pytest
import torch

import test_gpu_mx as plain
from stride_amd import harness, mx

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
