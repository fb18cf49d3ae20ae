"""Operators for models in microscaled 4-bit weights (include/stride_mx.h): blocks of 32 neighbours
along K that share a scale, a power of two; weights in 4 bits (e2m1), activations in 8 (e4m3).

    w = quantize(tiles, bits=4)                    packed weight tiles (layout.pack_tiles) -> Tiles
    x = norm(h, rows, gains, eps, add=y)           h += y, RMSNorm(h) * gains in 8 bits
    q = qkv(wq, wk, wv, x, rows, head_dim, rope, row_slot, row_pos, kv, layer)
    a = quantize(attn, rows, bits=8)               attention's x tiles -> Tiles
    y = gemm(wo, a, rows)                          W x in bf16 tiles, which the next norm adds to h
    z = mlp13(w1, w3, x, rows)                     silu(W1 x) * (W3 x) in 8 bits

A row's result depends on the row and the weights only, whatever the batch. Results go to `out`
(default: allocated here, on torch's current stream, so that with another one set by
set_kernel_stream it is passed), where rows behind `rows` are left as they were. Everything is
read when the launch runs, so it can be captured in a HIP graph.
"""
from __future__ import annotations

from struct import Struct

import torch

from . import _lib, tc
from .harness import PagedKv, other_stream

_TILES = Struct("<2Q2i").pack
_QUANTIZE = Struct("<4iQ24s2i").pack
_DEQUANTIZE = Struct("<4i24sQq2i").pack
_NORM = Struct("<4i3Q24sQif").pack
_GEMM = Struct("<4i24s24sQ").pack
_MLP13 = Struct("<4i24s24s24s24s").pack
_QKV = Struct("<4i24s24s24s24sQq56s3Q2i").pack
_NONE = _TILES(0, 0, 0, 0)

BLOCK, CHUNK, GROUP = 32, 128, 512  # columns of a scale, of a matrix instruction, of a lane's word of scales
_BF16 = (torch.int16, torch.bfloat16)  # or its bits
_device, _stream_of = (getattr(torch._C, name, None) for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"))
_PARTS = {4: (4, 16, 16), 8: (2, 4, 16, 16)}  # a chunk's codes


class Tiles:
    """Rows of `cols` columns in blocks of 4 or 8 bits, by tiles of 16 rows: codes and scales as
    include/stride_mx.h lays them out, uint8 [tiles][4 groups][4][16][16] (8 bits: [2][4][16][16])
    and [tiles][groups][4][16][4] with groups = ceil(cols / 512)."""

    def __init__(self, codes, scales, cols: int, bits: int):
        if bits not in (4, 8) or cols <= 0 or cols % 16 or cols > 1 << 20:
            raise ValueError("blocks have 4 or 8 bits, and cols is a positive multiple of 16, at most 2^20")
        tiles, groups = int(codes.shape[0]), (cols + GROUP - 1) // GROUP
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.device != scales.device \
                or not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("codes and scales must be contiguous uint8 on one device")
        if tuple(codes.shape) != (tiles, 4 * groups, *_PARTS[bits]) or tuple(scales.shape) != (tiles, groups, 4, 16, 4):
            raise ValueError(f"codes must be [tiles][{4 * groups}]{list(_PARTS[bits])} and scales [tiles][{groups}][4][16][4]")
        self._codes, self._scales, self._cols, self._bits = codes, scales, int(cols), bits
        self.tiles, self.rows = tiles, tiles * 16
        self._ref, self._device = _TILES(codes.data_ptr(), scales.data_ptr(), tiles, int(cols)), codes.get_device()

    # what _ref stands for is not exchanged afterwards
    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    cols = property(lambda self: self._cols)
    bits = property(lambda self: self._bits)

    def __reduce__(self):  # a copy has addresses of its own
        return Tiles, (self._codes, self._scales, self._cols, self._bits)

    @staticmethod
    def create(rows: int, cols: int, bits: int, device) -> "Tiles":
        """For `rows` rows, all zeros."""
        if bits not in _PARTS or rows < 0 or cols <= 0:
            raise ValueError("blocks have 4 or 8 bits; rows and cols are counts")
        tiles, groups = (rows + 15) // 16, (cols + GROUP - 1) // GROUP
        return Tiles(torch.zeros((tiles, 4 * groups, *_PARTS[bits]), dtype=torch.uint8, device=device),
                     torch.zeros((tiles, groups, 4, 16, 4), dtype=torch.uint8, device=device), cols, bits)

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def _here(dev: int) -> int:
    """The stream of a launch for tensors of device `dev`, which has to be the current one."""
    if dev != _device() or dev < 0:
        raise ValueError(f"tensors are on device {dev}, the current one is {_device()}")
    return _stream_of(dev) if tc._stream is None else tc.kernel_stream()


def _kind(error: AttributeError, tiles=(), tensors=(), given=()) -> Exception:
    """Why a check has met an argument without the attribute that it reads: the first that is no Tiles or
    no tensor (`given`: None is none either), by name."""
    for args, kind, what in ((tiles, Tiles, "Tiles"), (tensors, torch.Tensor, "a tensor"), (given, torch.Tensor, "a tensor")):
        for name, t in args:
            if not isinstance(t, kind) and not (args is given and t is None):
                return ValueError(f"{name} must be {what}")
    return error


def _operand(t, bits: int, rows: int, dev: int, cols: int, name: str) -> bytes:
    """A Tiles argument's block, looked over (cols 0: any)."""
    if type(t) is not Tiles or t._bits != bits or t._device != dev or not 0 <= rows <= t.rows or (cols and t._cols != cols):
        raise ValueError(f"{name} must be Tiles in {bits} bits with the rows and columns of the call, on its device")
    return t._ref


def _result(out, rows: int, cols: int, like) -> Tiles:
    if out is None:
        _allocates()
        return Tiles.create(rows, cols, 8, getattr(like, "codes", like).device)
    return out


def _allocates() -> None:
    if other_stream():
        raise ValueError("with another stream set by set_kernel_stream, pass out")


def _tile_cols(t, rows: int, name: str) -> int:
    """Columns of tiles [ceil(rows / 16)][cols / 16][16][16]."""
    shape = t.shape
    if len(shape) == 4 and t.is_contiguous():
        tiles, col_tiles, a, b = shape
        if a == 16 and b == 16 and 0 <= rows <= tiles * 16 and col_tiles:
            return col_tiles * 16
    raise ValueError(f"{name} must be contiguous tiles [ceil(rows / 16)][cols / 16][16][16]")


def _y_tiles(out, rows: int, cols: int, like, dev: int):
    """bf16 x tiles that are written (on the device of `like`, a tensor or Tiles)."""
    if out is None:
        _allocates()
        return torch.zeros(((rows + 15) // 16, cols // 16, 16, 16), dtype=torch.int16, device=getattr(like, "codes", like).device)
    if out.dtype not in _BF16 or out.get_device() != dev or _tile_cols(out, rows, "out") != cols:
        raise ValueError(f"out must be 16-bit tiles of {cols} columns on the call's device")
    return out


def quantize(tiles, rows: int | None = None, bits: int = 4, out: Tiles | None = None) -> Tiles:
    """Tiles [t][ct][16][16] of 16-bit (bf16, or its bits in int16) or fp32 values to blocks of 4
    or 8 bits, for the first `rows` rows (default: all)."""
    try:
        if tiles.dtype in _BF16:
            size = 2
        elif tiles.dtype == torch.float32:
            size = 4
        else:
            raise ValueError("tiles must hold bf16 or fp32")
        if bits not in (4, 8):
            raise ValueError("blocks have 4 or 8 bits")
        dev = tiles.get_device()
        stream = _here(dev)
        rows = len(tiles) * 16 if rows is None and tiles.dim() else rows
        cols = _tile_cols(tiles, rows, "tiles")
        if out is None:
            _allocates()
            out = Tiles.create(rows, cols, bits, tiles.device)
        p = _QUANTIZE(rows, (rows + 15) // 16, 0, 0, tiles.data_ptr(), _operand(out, bits, rows, dev, cols, "out"), bits, size)
    except AttributeError as e:
        raise _kind(e, tensors=(("tiles", tiles),))
    rc = _lib.packed().stride_mx_quantize(p, stream)
    if rc:
        _lib.check(rc)
    return out


def microscaled(tiles) -> Tiles:
    """quantize(tiles) of bf16 weights on torch's current stream, whatever set_kernel_stream says: there a
    model's weights are packed and its buffers made."""
    if tiles.dtype not in _BF16:
        raise ValueError("weights are bf16")
    dev = tiles.get_device()
    _here(dev)
    out = Tiles.create(len(tiles) * 16, _tile_cols(tiles, 0, "tiles"), 4, tiles.device)
    p = _QUANTIZE(out.rows, out.tiles, 0, 0, tiles.data_ptr(), out._ref, 4, 2)
    rc = _lib.packed().stride_mx_quantize(p, _stream_of(dev))
    if rc:
        _lib.check(rc)
    return out


def dequantize(t: Tiles, rows: int | None = None, dtype=torch.bfloat16, out=None):
    """The values of the first `rows` rows, row-major [rows][cols] in bf16 or fp32."""
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("values come in bf16 or fp32")
    try:
        stream = _here(t._device)
        rows = t.rows if rows is None else rows
        ref = _operand(t, t._bits, rows, t._device, 0, "t")
        if out is None:
            _allocates()
            out = torch.empty((rows, t.cols), dtype=dtype, device=t.codes.device)
        elif out.dtype != dtype or out.dim() != 2 or out.shape[0] < rows or out.shape[1] != t.cols or out.stride(1) != 1 or out.get_device() != t._device:
            raise ValueError("out must be [rows][cols] of that type on the same device, its rows contiguous")
    except AttributeError as e:
        raise _kind(e, tiles=(("t", t),), given=(("out", out),))
    p = _DEQUANTIZE(rows, (rows + 15) // 16, 0, 0, ref, out.data_ptr(), out.stride(0) if rows > 1 else t.cols, t.bits, 2 if dtype == torch.bfloat16 else 4)
    rc = _lib.packed().stride_mx_dequantize(p, stream)
    if rc:
        _lib.check(rc)
    return out


def norm(h, rows: int, weight, eps: float, add=None, out=None, bits: int = 8):
    """h += add (bf16 tiles, where given), then RMSNorm(h) * weight: in 8 bits (Tiles), or with
    bits=16 in bf16 x tiles. h: fp32 tiles [lt][ct][16][16]."""
    try:
        dev = h.get_device()
        stream = _here(dev)
        if h.dtype != torch.float32:
            raise ValueError("h must be fp32 tiles")
        cols = _tile_cols(h, rows, "h")
        if weight.dtype != torch.float32 or weight.numel() != cols or not weight.is_contiguous() or weight.get_device() != dev:
            raise ValueError("weight must be contiguous fp32 of h's columns, on its device")
        a = 0
        if add is not None:
            if add.dtype not in _BF16 or add.get_device() != dev or _tile_cols(add, rows, "add") != cols:
                raise ValueError("add must be bf16 tiles of h's columns on its device")
            a = add.data_ptr()
        if bits == 8:
            out = _result(out, rows, cols, h)
            ref, x = _operand(out, 8, rows, dev, cols, "out"), 0
        elif bits == 16:
            out = _y_tiles(out, rows, cols, h, dev)
            ref, x = _NONE, out.data_ptr()
        else:
            raise ValueError("a norm's result has 8 or 16 bits")
    except AttributeError as e:
        raise _kind(e, tensors=(("h", h), ("weight", weight)), given=(("add", add), ("out", out)))
    p = _NORM(rows, (rows + 15) // 16, 0, 0, h.data_ptr(), a, weight.data_ptr(), ref, x, cols, eps)
    rc = _lib.packed().stride_mx_norm(p, stream)
    if rc:
        _lib.check(rc)
    return out


def gemm(w: Tiles, x: Tiles, rows: int, out=None):
    """y = W x for the first `rows` rows of x, in bf16 x tiles."""
    try:
        dev = x._device
        stream = _here(dev)
        xr, wr = _operand(x, 8, rows, dev, 0, "x"), _operand(w, 4, 1, dev, x._cols, "w")
        out = _y_tiles(out, rows, w.rows, x, dev)
    except AttributeError as e:
        raise _kind(e, tiles=(("x", x), ("w", w)), given=(("out", out),))
    p = _GEMM(rows, (rows + 15) // 16, 0, 0, xr, wr, out.data_ptr())
    rc = _lib.packed().stride_mx_gemm(p, stream)
    if rc:
        _lib.check(rc)
    return out


def mlp13(w1: Tiles, w3: Tiles, x: Tiles, rows: int, out: Tiles | None = None) -> Tiles:
    """z = silu(W1 x) * (W3 x) in 8 bits."""
    try:
        dev = x._device
        stream = _here(dev)
        xr, r1 = _operand(x, 8, rows, dev, 0, "x"), _operand(w1, 4, 1, dev, x._cols, "w1")
        r3 = _operand(w3, 4, w1.rows, dev, x._cols, "w3")
        out = _result(out, rows, w1.rows, x)
        p = _MLP13(rows, (rows + 15) // 16, 0, 0, xr, r1, r3, _operand(out, 8, rows, dev, w1.rows, "out"))
    except AttributeError as e:
        raise _kind(e, tiles=(("x", x),))
    rc = _lib.packed().stride_mx_mlp13(p, stream)
    if rc:
        _lib.check(rc)
    return out


def qkv(wq: Tiles, wk: Tiles, wv: Tiles, x: Tiles, rows: int, head_dim: int, rope, row_slot, row_pos, kv: PagedKv, layer: int = 0,
        q_out=None):
    """harness.qkv on these weights (rows in layout.rope_rows' order): q with RoPE in fp32 rows, K
    and V appended to the paged bf16 cache. A row is left out, its q as it was, where its slot is no row
    of kv.table or its position lies behind the cache's last page or behind rope."""
    try:
        dev = x._device
        stream = _here(dev)
        xr = _operand(x, 8, rows, dev, 0, "x")
        ws = [_operand(w, 4, 1, dev, x._cols, name) for w, name in ((wq, "wq"), (wk, "wk"), (wv, "wv"))]
        nq = wq.rows
        if not isinstance(kv, PagedKv):
            raise ValueError("kv must be a PagedKv")
        if row_slot.dtype != torch.int32 or row_pos.dtype != torch.int32 or row_slot.numel() < rows or row_pos.numel() < rows \
                or not (row_slot.is_contiguous() and row_pos.is_contiguous()):
            raise ValueError("row_slot and row_pos must be contiguous int32, one for each row")
        if rope.dtype != torch.float32 or not rope.is_contiguous() or rope.dim() != 3 or rope.shape[1] * 2 != head_dim or rope.shape[2] != 2:
            raise ValueError("rope must be contiguous fp32 [positions][head_dim / 2][2]")
        if not row_slot.get_device() == row_pos.get_device() == rope.get_device() == kv.table.get_device() == kv.arena.get_device() == dev:
            raise ValueError("the arguments are on different devices")
        if not 0 <= layer < kv.ref.block_elems // kv.ref.layer_elems or kv.ref.which_elems * head_dim != wk.rows * kv.ref.group_elems:
            raise ValueError("layer or the number of KV heads is not the cache's")
        if q_out is None:
            _allocates()
            q_out = torch.zeros((max(rows, 1), nq), dtype=torch.float32, device=x.codes.device)
        elif q_out.dtype != torch.float32 or q_out.dim() != 2 or q_out.shape[0] < rows or q_out.shape[1] != nq or q_out.stride(1) != 1 \
                or q_out.get_device() != dev:
            raise ValueError("q_out must be fp32 [rows][q columns], its rows contiguous")
    except AttributeError as e:
        raise _kind(e, tiles=(("x", x),), tensors=(("rope", rope), ("row_slot", row_slot), ("row_pos", row_pos)), given=(("q_out", q_out),))
    p = _QKV(rows, (rows + 15) // 16, 0, 0, xr, *ws, q_out.data_ptr(), q_out.stride(0) if rows > 1 else nq,
             bytes(kv.ref), rope.data_ptr(), row_slot.data_ptr(), row_pos.data_ptr(), layer, head_dim)
    rc = _lib.packed().stride_mx_qkv_within(p, kv.table.shape[0], rope.shape[0], stream)
    if rc:
        _lib.check(rc)
    return q_out
