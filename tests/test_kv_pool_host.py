"""The page pool's Python side (stride_amd.kv_pool) on host tensors: what it offers and refuses
before anything is launched. No GPU."""
import pytest
import torch

from stride_amd import harness
from stride_amd.kv_pool import KvPool


def test_an_fp32_pool_is_no_bf16_cache():
    """window_attention, attention and qkv read two bytes an element: they would take an fp32
    arena for one of twice as many bf16 and answer from its halves."""
    pool = KvPool.create(2, 64, 8, 2, 32, 1, 16, "cpu")
    assert isinstance(pool.kv, harness.PagedKv) and pool.kv.ref is pool.ref and pool.kv.capacity == 64
    wide = KvPool.create(2, 64, 8, 2, 32, 1, 16, "cpu", fp32=True)
    assert wide.ref.block_elems == pool.ref.block_elems and wide.ref.arena == wide.arena.data_ptr()
    with pytest.raises(ValueError, match="fp32"):
        wide.kv
