"""Logit processing on lm_full's tiles (include/stride_serve.h): penalties for tokens that a
sequence has, biases, a grammar's mask, and the greedy choice.

    counts = TokenCounts.create(slots, vocab, dev)
    counts.record(slot, prompt_tokens, prompt=True)
    best = process(tiles, rows, vocab, counts, row_slot, penalties, bias, mask, mask_row)
    counts.record(row_slot, best[:, 1])

For row j of sequence row_slot[j], token t generated n times so far:
    l1 = (l > 0 ? l / repetition : l * repetition) for a token of the prompt or generated
    l2 = l1 - frequency * n, and - presence where n > 0
    l3 = l2 + bias;  l4 = allowed ? l3 : -inf
The choice is the largest l4, of equal ones the lowest token; (-inf, -1) where a row has
nothing allowed. Everything is read when the launch runs, so it can be captured in a HIP graph.
"""
from __future__ import annotations

import ctypes as C
from struct import Struct

import numpy as np
import torch

from . import _lib, tc
from .harness import here, other_stream

_LOGITS = Struct("<4i13Q3i4x").pack
UNIT = 17 * 32  # scratch of a lane tile, int64
IN_PROMPT = -(1 << 31)  # TokenCounts.counts: the token is in the prompt


def words(vocab: int) -> int:
    return (vocab + 31) // 32


class TokenCounts:
    """Which tokens each sequence has: counts [slots][vocab] int32 (the sign bit: in the prompt;
    below it: times generated) and seen [slots][ceil(vocab / 32)] int32, a bit for every count
    that is not 0."""

    def __init__(self, counts, seen):
        if counts.dtype != torch.int32 or seen.dtype != torch.int32 or counts.dim() != 2 or seen.dim() != 2:
            raise ValueError("counts and seen must be int32 [slots][...]")
        if not (counts.is_contiguous() and seen.is_contiguous()) or counts.device != seen.device:
            raise ValueError("counts and seen must be contiguous and on one device")
        if seen.shape[0] != counts.shape[0] or seen.shape[1] != words(counts.shape[1]):
            raise ValueError("seen must be [slots][ceil(vocab / 32)]")
        self.counts, self.seen = counts, seen
        self.slots, self.vocab = (int(x) for x in counts.shape)
        self._params = _lib.TokenCountsParams(tc.ptr(counts), tc.ptr(seen), self.slots, self.vocab)
        self._at = C.addressof(self._params)
        self._counts_at, self._seen_at, self._device = tc.ptr(counts), tc.ptr(seen), counts.get_device()
        self._scratch = {}

    @staticmethod
    def create(slots: int, vocab: int, device) -> "TokenCounts":
        return TokenCounts(torch.zeros((slots, vocab), dtype=torch.int32, device=device),
                           torch.zeros((slots, words(vocab)), dtype=torch.int32, device=device))

    def record(self, slot, tokens, prompt: bool = False) -> None:
        """Counts tokens[i] for slot[i] (int32 vectors; tokens may be strided, as the indices of
        a BestEntry buffer are); those out of range, -1 among them, are ignored."""
        n = slot.numel()
        if slot.dtype != torch.int32 or tokens.dtype != torch.int32 or tokens.dim() != 1 or tokens.numel() != n \
                or slot.get_device() != self._device or tokens.get_device() != self._device or not slot.is_contiguous():
            raise ValueError("slot (contiguous) and tokens are int32 vectors of one length on the counts' device")
        here(slot)
        rc = _lib.load().stride_logits_record(self._at, slot.data_ptr(), tokens.data_ptr(), tokens.stride(0) if n > 1 else 1, n,
                                              1 if prompt else 0, tc.kernel_stream())
        if rc:
            _lib.check(rc)

    def reset(self, slot, src=None) -> None:
        """slot[i] forgets its tokens, or takes over those of src[i]. A slot to be changed comes
        up once and is no source."""
        n = slot.numel()
        for t in (slot,) if src is None else (slot, src):
            if t.dtype != torch.int32 or t.numel() != n or t.get_device() != self._device or not t.is_contiguous():
                raise ValueError("slot and src are contiguous int32 vectors of one length on the counts' device")
        here(slot)
        rc = _lib.load().stride_logits_reset(self._at, slot.data_ptr(), 0 if src is None else src.data_ptr(), n, tc.kernel_stream())
        if rc:
            _lib.check(rc)


def scratch(rows: int, device):
    """What process() keeps between its workgroups: zeros, and zeros again after each call."""
    return torch.zeros(_lib.load().stride_logits_scratch(rows), dtype=torch.int64, device=device)


def bias_lists(rows, device):
    """(offsets, tokens, values) for process() from a dict {token: bias} (or None) a row."""
    offsets, tokens, values = [0], [], []
    for d in rows:
        for t in sorted(d or {}):
            tokens.append(t)
            values.append(d[t])
        offsets.append(len(tokens))
    pad = [0] if not tokens else []  # an empty tensor has no address
    return (torch.tensor(offsets, dtype=torch.int32, device=device), torch.tensor(tokens + pad, dtype=torch.int32, device=device),
            torch.tensor(values + [float(x) for x in pad], dtype=torch.float32, device=device))


def pack_mask(allowed, device):
    """[masks][vocab] truth values (NumPy or a list of token collections with a vocabulary: see
    mask_of) -> int32 bit words [masks][ceil(vocab / 32)]."""
    a = np.asarray(allowed, dtype=bool)
    m, v = a.shape
    wide = np.zeros((m, words(v) * 32), dtype=bool)
    wide[:, :v] = a
    bits = np.packbits(wide, axis=1, bitorder="little").view("<u4")
    return torch.from_numpy(bits.view(np.int32).copy()).to(device)


def mask_of(lists, vocab: int, device):
    """Masks that allow exactly the tokens of each list."""
    a = np.zeros((len(lists), vocab), dtype=bool)
    for i, tokens in enumerate(lists):
        a[i, np.asarray(list(tokens), dtype=np.int64)] = True
    return pack_mask(a, device)


def process(logits, rows: int, vocab: int, counts: TokenCounts | None = None, row_slot=None, penalties=None, bias=None,
            mask=None, mask_row=None, out=None, best=None, work=None):
    """Processes lm_full's tiles [rt][lt][16][16] for `rows` rows and returns the BestEntry
    buffer (int32 [rows][2]: value bits, token). penalties: fp32 [rows][3] (repetition, presence,
    frequency), with counts; bias: (offsets, tokens, values), see bias_lists; mask: bit words
    [masks][words], with mask_row int32 [rows] (below 0: no mask). out: receives the processed
    tiles (may be `logits`). work: scratch(rows) (default: one that `counts` keeps for this
    stream, or a new one). With another stream set by set_kernel_stream, best and work are
    passed."""
    i32, f32 = torch.int32, torch.float32
    here(logits)
    T = (rows + 15) // 16
    shape = logits.shape
    if logits.dtype != f32 or len(shape) != 4 or shape[1] != T or shape[0] * 16 < vocab or shape[2] != 16 or shape[3] != 16 \
            or not logits.is_contiguous():
        raise ValueError("logits must be contiguous fp32 tiles [ceil(vocab / 16)][ceil(rows / 16)][16][16]")
    dev, o_at = logits.get_device(), 0
    if out is not None:
        if out.get_device() != dev or out.dtype != f32 or out.shape != shape or not out.is_contiguous():
            raise ValueError("out must be tiles like logits")
        o_at = out.data_ptr()
    if best is None:
        if other_stream():
            raise ValueError("with another stream set by set_kernel_stream, pass best and work")
        best = torch.empty((rows, 2), dtype=i32, device=logits.device)
    elif best.get_device() != dev or best.dtype != i32 or best.numel() < 2 * rows or not best.is_contiguous():
        raise ValueError("best must be contiguous int32 [rows][2]")
    c = s = sl = pen = slots = 0
    if counts is not None:
        if counts.vocab != vocab or counts._device != dev:
            raise ValueError("the counts are of another vocabulary or device")
        if row_slot is None or penalties is None:
            raise ValueError("counts need row_slot and penalties")
        if row_slot.get_device() != dev or row_slot.dtype != i32 or row_slot.numel() < rows or not row_slot.is_contiguous():
            raise ValueError("row_slot must be contiguous int32 [rows]")
        if penalties.get_device() != dev or penalties.dtype != f32 or penalties.numel() < 3 * rows or not penalties.is_contiguous():
            raise ValueError("penalties must be contiguous fp32 [rows][3]")
        c, s, sl, pen, slots = counts._counts_at, counts._seen_at, row_slot.data_ptr(), penalties.data_ptr(), counts.slots
    bo = bt = bv = 0
    if bias is not None:
        o, t, v = bias
        n = t.numel()
        if not o.get_device() == t.get_device() == v.get_device() == dev or o.dtype != i32 or t.dtype != i32 or v.dtype != f32 or o.numel() < rows + 1 or v.numel() != n \
                or not (o.is_contiguous() and t.is_contiguous() and v.is_contiguous()):
            raise ValueError("bias is (offsets int32 [rows + 1], tokens int32, values fp32), contiguous")
        if n:  # without entries there is nothing to add
            bo, bt, bv = o.data_ptr(), t.data_ptr(), v.data_ptr()
    mk = mr = masks = 0
    if mask is not None:
        if mask.get_device() != dev or mask.dtype != i32 or mask.dim() != 2 or mask.size(1) != (vocab + 31) // 32 or not mask.is_contiguous():
            raise ValueError("mask must be contiguous int32 [masks][ceil(vocab / 32)]")
        if mask_row is None or mask_row.get_device() != dev or mask_row.dtype != i32 or mask_row.numel() < rows or not mask_row.is_contiguous():
            raise ValueError("a mask needs mask_row, contiguous int32 [rows]")
        mk, mr, masks = mask.data_ptr(), mask_row.data_ptr(), mask.size(0)
    stream = tc.kernel_stream()
    if work is None:
        work = _work_of(counts, T, rows, stream, logits.device)
    elif work.get_device() != dev or work.dtype != torch.int64 or work.numel() < T * UNIT or not work.is_contiguous():
        raise ValueError("work must be scratch(rows)")
    p = _LOGITS(rows, T, 0, 0, logits.data_ptr(), o_at, sl, c, s, pen, bo, bt, bv, mk, mr, best.data_ptr(), work.data_ptr(),
                vocab, slots, masks)
    rc = _lib.packed().stride_logits_process(p, stream)
    if rc:
        _lib.check(rc)
    return best


def _work_of(counts, T: int, rows: int, stream: int, device):
    """A scratch of its own for each stream that uses the counts, kept with them. A captured
    graph must not find it in eager use on another stream: it gets one that is its own."""
    if tc._stream is not None:
        raise ValueError("with a stream set by set_kernel_stream, pass work (scratch(rows))")
    if counts is None or torch.cuda.is_current_stream_capturing():
        return scratch(rows, device)
    kept = counts._scratch.get(stream)
    if kept is None or kept.numel() < T * UNIT:
        kept = counts._scratch[stream] = scratch(rows, device)
    return kept
