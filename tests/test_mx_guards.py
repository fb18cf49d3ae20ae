"""Calls of the microscaled operators that have to be refused, or that have to leave rows alone, without
a GPU: what the C ABI refuses before a launch."""
import pytest

from stride_amd import _lib, mx

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
