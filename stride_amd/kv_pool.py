"""A pool of KV pages that sequences share (include/stride_serve.h).

    pool = KvPool.create(slots, max_ctx, pages, kv_heads, head_dim, layers, page_tokens, dev)
    pool.reserve(slot, first, end)          pages for table entries that have none
    pool.release(slot, first, end)          gives entries up; a page without holders is free
    pool.fork(src, dst, length)             dst goes on from the first `length` tokens of src
    pool.compact(slot, first, count, keep)  kept positions move together, the rest is given up
    pool.copy(src, dst, tokens, into)       page contents, within a pool or into another
    pool.check()                            raises what earlier calls reported

``pool.kv`` is the harness.PagedKv that tc_qkv, attention and window_attention take (of a bf16
pool; the exact path takes ``pool.ref``). Slots,
ranges and lengths are int32 device tensors, one entry an item, so a call needs nothing from
the host and can be captured in a HIP graph. Free pages are taken lowest number first, by
ascending item and table index: the outcome is fixed. A call whose items break a rule, or that
wants more pages than are free, changes nothing (but see compact) and is reported by check(), which
waits for the device; a serving loop that counts its pages itself (pages_of) needs it only as a guard.

Calls on one pool are ordered by the caller (one stream, or events), captured ones among them.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib, tc
from .harness import PagedKv, here

BAD_ITEM, TWICE, NO_PAGES, MISSING, BAD_KEEP, BAD_REFS = 1, 2, 4, 8, 16, 32
MESSAGES = {
    BAD_ITEM: "a slot, range, length or page was outside its bounds",
    TWICE: "a slot or page to be changed came up twice, or was a source too",
    NO_PAGES: "fewer pages are free than a call wanted",
    MISSING: "a position to be moved has no page",
    BAD_KEEP: "kept positions did not ascend from `first`",
    BAD_REFS: "a held page's reference count was not positive",
}


class KvPool:
    """Table, reference counts and free pages over a KV arena [page][layer][K|V][group][token]
    [dim] (int16 bits of bf16, or fp32)."""

    def __init__(self, arena, table, refs, kv_heads: int, head_dim: int, layers: int, page_tokens: int):
        """Over tensors that exist: the arena, table [slots][max_blocks] int32 (-1: no page) and
        refs [pages] int32, the number of table entries that hold each page."""
        elem = arena.element_size()
        if arena.dtype not in (torch.int16, torch.float32):
            raise ValueError("the arena holds int16 bits of bf16, or fp32")
        if table.dtype != torch.int32 or table.dim() != 2 or refs.dtype != torch.int32:
            raise ValueError("table must be int32 [slots][max_blocks], refs int32 [pages]")
        if not (arena.is_contiguous() and table.is_contiguous() and refs.is_contiguous()):
            raise ValueError("arena, table and refs must be contiguous")
        if not arena.device == table.device == refs.device:
            raise ValueError("arena, table and refs must be on one device")
        pages = refs.numel()
        block = layers * 2 * kv_heads * page_tokens * head_dim
        if pages < 1 or block < 1 or arena.numel() != pages * block:
            raise ValueError("the arena does not hold refs.numel() pages of this shape")
        self.arena, self.table, self.refs = arena, table, refs
        self.kv_heads, self.head_dim, self.layers, self.page_tokens = kv_heads, head_dim, layers, page_tokens
        slots, max_blocks = (int(x) for x in table.shape)
        dev = arena.device
        words = (pages + 31) // 32
        free = torch.zeros(words * 32, dtype=torch.int64, device=dev)
        free[:pages] = refs == 0
        bits = (free.reshape(words, 32) << torch.arange(32, device=dev)).sum(1)
        self.free_bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
        self.errors = torch.zeros(1, dtype=torch.int32, device=dev)
        ints = _lib.load().stride_kv_work_ints(slots, max_blocks, pages)
        self.work = torch.empty(ints, dtype=torch.int32, device=dev)
        group = page_tokens * head_dim
        ref = _lib.KvRef(tc.ptr(arena), tc.ptr(table), block, 2 * kv_heads * group, kv_heads * group, group, max_blocks, head_dim)
        #: The cache as the C calls take it.
        self.ref = ref
        self._kv = PagedKv(arena.reshape(-1), table, ref, page_tokens, max_blocks) if elem == 2 else None
        self._params = _lib.KvPoolParams(ref, tc.ptr(refs), tc.ptr(self.free_bits), tc.ptr(self.errors), tc.ptr(self.work),
                                         ints, pages, slots, layers, kv_heads, elem)
        self._at = C.addressof(self._params)
        self._device = table.get_device()

    @staticmethod
    def create(slots: int, max_ctx: int, pages: int, kv_heads: int, head_dim: int, layers: int, page_tokens: int, device,
               fp32: bool = False) -> "KvPool":
        """A pool of `pages` free pages for `slots` sequences of up to max_ctx tokens."""
        max_blocks = (max_ctx + page_tokens - 1) // page_tokens
        arena = torch.zeros(pages * layers * 2 * kv_heads * page_tokens * head_dim,
                            dtype=torch.float32 if fp32 else torch.int16, device=device)
        table = torch.full((slots, max_blocks), -1, dtype=torch.int32, device=device)
        return KvPool(arena, table, torch.zeros(pages, dtype=torch.int32, device=device), kv_heads, head_dim, layers, page_tokens)

    @property
    def kv(self) -> PagedKv:
        """What the attention and QKV runners of the tensor-core path take, which read bf16: an
        fp32 pool has none (`ref` is what the exact path's parameter blocks take)."""
        if self._kv is None:
            raise ValueError("the runners that take kv read bf16, and this pool holds fp32")
        return self._kv

    @property
    def pages(self) -> int:
        return self.refs.numel()

    @property
    def slots(self) -> int:
        return int(self.table.shape[0])

    def pages_of(self, length: int) -> int:
        """Table entries of a sequence of `length` tokens."""
        return (length + self.page_tokens - 1) // self.page_tokens

    def free_pages(self) -> int:
        """How many pages are free (waits for the device)."""
        self._wait()
        return int((self.refs == 0).sum())

    def _wait(self) -> None:
        """For every stream: the pool's calls may be on another than torch's current one."""
        if self._device >= 0:
            torch.cuda.synchronize(self._device)

    def _items(self, *items) -> int:
        n, dev = items[0].numel(), self._device
        for t in items:
            if t.dtype != torch.int32 or t.get_device() != dev or t.numel() != n or not t.is_contiguous():
                raise ValueError("items are contiguous int32 tensors of one length on the pool's device")
        here(items[0])
        return n

    def reserve(self, slot, first, end) -> None:
        """Pages for the entries [first[i], end[i]) of table row slot[i] that have none."""
        n = self._items(slot, first, end)
        _run(_lib.load().stride_kv_reserve(self._at, slot.data_ptr(), first.data_ptr(), end.data_ptr(), n, tc.kernel_stream()))

    def release(self, slot, first, end) -> None:
        """Gives the entries [first[i], end[i]) of table row slot[i] up (-1 afterwards)."""
        n = self._items(slot, first, end)
        _run(_lib.load().stride_kv_release(self._at, slot.data_ptr(), first.data_ptr(), end.data_ptr(), n, tc.kernel_stream()))

    def fork(self, src, dst, length) -> None:
        """dst[i] becomes the first length[i] tokens of src[i]: whole pages are shared, a part
        page is copied; what dst[i] held is given up."""
        n = self._items(src, dst, length)
        _run(_lib.load().stride_kv_fork(self._at, src.data_ptr(), dst.data_ptr(), length.data_ptr(), n, tc.kernel_stream()))

    def compact(self, slot, first, count, keep) -> None:
        """Position first[i] + k of slot[i] becomes what position keep[i][k] was, for k <
        count[i]; what lies behind is given up. keep: int32 [n][width], count[i] <= width, each
        row strictly ascending from first[i] or above. (With count[i] 0 nothing is written, and
        the page that first[i] lies in may still be shared.) A row that only does not ascend is
        seen while its positions move: they then hold some of that slot's old entries."""
        n = self._items(slot, first, count)
        if keep.dtype != torch.int32 or keep.dim() != 2 or keep.shape[0] != n or (keep.shape[1] > 1 and keep.stride(1) != 1):
            raise ValueError("keep must be int32 [n][width], its rows contiguous")
        if keep.get_device() != self._device:
            raise ValueError("items must be on the pool's device")
        _run(_lib.load().stride_kv_compact(self._at, slot.data_ptr(), first.data_ptr(), count.data_ptr(), keep.data_ptr(),
                                           keep.stride(0) if n > 1 else keep.shape[1], keep.shape[1], n, tc.kernel_stream()))

    def copy(self, src, dst, tokens=None, into: "KvPool | None" = None) -> None:
        """The first tokens[i] (None: all) tokens of page src[i] to page dst[i] of `into` (None:
        this pool). Tables and counts stay as they are."""
        n = self._items(src, dst) if tokens is None else self._items(src, dst, tokens)
        if into is not None and into._device != self._device:
            raise ValueError("the pools must be on one device")
        _run(_lib.load().stride_kv_copy(self._at, None if into is None else into._at, src.data_ptr(), dst.data_ptr(),
                                        0 if tokens is None else tokens.data_ptr(), n, tc.kernel_stream()))

    def check(self) -> None:
        """Raises StrideTcError for what calls reported since the last check (waits for the
        device)."""
        self._wait()
        bits = int(self.errors.item())
        if bits:
            self.errors.zero_()
            self._wait()
            raise _lib.StrideTcError("kv pool: " + "; ".join(m for b, m in MESSAGES.items() if bits & b))


def _run(rc: int) -> None:
    if rc:
        _lib.check(rc)
