"""A K/V cache held in 4 or 8 bits: written, read back, attended to.

No counterpart in the reference, whose cache is bf16.  ``QuantKVCache`` holds
the K/V rows of ``num_seqs`` sequences and ``num_layers`` layers: head_dim is
cut into groups of 32 values, each held as signed codes (4 bits: -7 .. 7, 8
bits: -127 .. 127) times one bf16 scale, the group's largest magnitude / 7 or
/ 127 (``include/qwen_megakernel.h`` has the format).  A position costs
``kv_heads * (head_dim * bits / 4 + head_dim / 8)`` bytes a layer for K and V:
0.28 (4 bits) or 0.53 (8 bits) of the bf16 cache.

Which rows a call is about is a ``KVRows``: segment b holds some consecutive
rows of the call's tensors at consecutive positions of one sequence.  One row
a segment is a decode step, many rows a prompt or a chunk of one.

    cache = QuantKVCache(num_seqs=2, max_seq_len=4096, bits=4)
    rows = KVRows([0, 100], [7, 1])   # 7 rows of sequence 0, 1 row of sequence 1
    cache.write(k, v, rows)           # k, v [8, kv_heads, head_dim]
    out = cache.attend(q, rows)       # q [8, q_heads, head_dim]
    k8, v8 = cache.read(rows)

All calls are stream-ordered, allocate through torch's caching allocator only
and can be captured in a CUDA graph; ``BatchDecoder(kv_bits=4)`` decodes with
such a cache.  These are inference operators: no gradient passes through.
"""

from __future__ import annotations

import math

import torch

from . import _native
from .weights import HEAD_DIM, NUM_KV_HEADS

GROUP = 32  # QMK_KV_GROUP
CAPACITY_STEP = 128  # QMK_KV_CAPACITY_STEP
MAX_RATIO = 16  # QMK_KV_MAX_RATIO
BAD_ROW = 1  # QMK_KV_BAD_ROW
NONFINITE = 2  # QMK_KV_NONFINITE
TIMEOUT = 4  # QMK_KV_TIMEOUT
COPIES_PENDING = 8  # QMK_KV_COPIES_PENDING


class KVCacheError(RuntimeError):
    """A device-side finding reported by a quantized cache's status word."""


def _index(values, what: str) -> list[int]:
    out = [int(v) for v in values]
    if any(v < 0 or v >= 2**31 for v in out):
        raise ValueError(f"{what} must be in [0, 2^31)")
    return out


class KVRows:
    """The rows of a call, in segments of consecutive positions.

    Segment b holds ``counts[b]`` rows (default 1), the next ones of the
    call's tensors, at positions ``starts[b]``, ``starts[b] + 1``, ... of
    sequence ``seq_ids[b]`` (default b)."""

    def __init__(self, starts, counts=None, seq_ids=None, device="cuda"):
        starts = _index(starts, "starts")
        if not starts:
            raise ValueError("KVRows needs at least one segment")
        seqs = list(range(len(starts))) if seq_ids is None else _index(seq_ids, "seq_ids")
        counts_ = [1] * len(starts) if counts is None else _index(counts, "counts")
        if len(seqs) != len(starts) or len(counts_) != len(starts):
            raise ValueError("starts, counts and seq_ids must have equal length")
        offsets = [0]
        for c in counts_:
            offsets.append(offsets[-1] + c)
        if offsets[-1] >= 2**31 - 1:
            raise ValueError("too many rows")
        self.rows = offsets[-1]
        self.max_rows = max(counts_)
        self._covers = True  # every row lies in a segment
        # host-known limits: checked against the cache at every call
        self._num_seqs = max(seqs) + 1
        self._end = max(s + c for s, c in zip(starts, counts_))
        spans = sorted((q, s, s + c) for q, s, c in zip(seqs, starts, counts_) if c)
        self._overlap = any(a[0] == b[0] and b[1] < a[2] for a, b in zip(spans, spans[1:]))
        self.start = self._to(starts, device)
        self.row_offsets = None if counts is None else self._to(offsets, device)
        self.seq = None if seq_ids is None else self._to(seqs, device)

    @staticmethod
    def _to(values, device):
        t = torch.tensor(values, dtype=torch.int32)
        return t.to(device) if torch.device(device).type != "cuda" else t.pin_memory().to(device, non_blocking=True)

    @classmethod
    def from_tensors(cls, start, row_offsets=None, seq=None, rows=None, max_rows=None) -> "KVRows":
        """Rows described by device tensors (int32), which a program may change
        between calls, a captured graph's included: ``start`` [segments],
        ``row_offsets`` [segments + 1] or None (one row a segment), ``seq``
        [segments] or None (segment b is sequence b).  With ``row_offsets``,
        ``rows`` is the number of rows of the call's tensors and ``max_rows``
        the most that a segment may hold.  Nothing of the tensors is known on
        the host: a row out of range is reported by ``check_status``; a write
        must not hold a position twice (what stays is then not defined)."""
        self = cls.__new__(cls)
        if row_offsets is None:
            if rows not in (None, start.numel()) or max_rows not in (None, 1):
                raise ValueError("without row_offsets every segment has one row")
            rows, max_rows = start.numel(), 1
        elif rows is None or max_rows is None:
            raise ValueError("row_offsets needs rows and max_rows")
        self._covers = row_offsets is None
        self.rows, self.max_rows = int(rows), int(max_rows)
        if self.rows < 0 or self.max_rows < 0:
            raise ValueError("rows and max_rows must be >= 0")
        self._num_seqs, self._end, self._overlap = 0, 0, False
        self.start, self.row_offsets, self.seq = start, row_offsets, seq
        return self


class QuantKVCache:
    """K/V rows of ``num_seqs`` sequences and ``num_layers`` layers in
    ``bits`` (4 or 8) bits a value."""

    def __init__(self, num_seqs: int, max_seq_len: int, num_layers: int = 1, num_kv_heads: int = NUM_KV_HEADS,
                 head_dim: int = HEAD_DIM, bits: int = 4, device="cuda"):
        if bits not in (4, 8):
            raise ValueError("bits must be 4 or 8")
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if min(num_seqs, max_seq_len, num_layers, num_kv_heads) < 1:
            raise ValueError("num_seqs, max_seq_len, num_layers and num_kv_heads must be >= 1")
        ops = _native.ops()
        # (the overloads themselves: looking them up costs a call about a microsecond)
        self._write, self._read, self._attend = ops.kv_write.default, ops.kv_read.default, ops.kv_attend.default
        self.num_seqs, self.num_layers, self.num_kv_heads = int(num_seqs), int(num_layers), int(num_kv_heads)
        self.max_seq_len, self.head_dim, self.bits = int(max_seq_len), int(head_dim), int(bits)
        self.capacity = -(-self.max_seq_len // CAPACITY_STEP) * CAPACITY_STEP
        shape = (self.num_seqs, self.num_layers, self.num_kv_heads, self.capacity)
        codes, scales = shape + (self.head_dim * self.bits // 8,), shape + (self.head_dim // GROUP,)
        self.k_codes = torch.zeros(codes, dtype=torch.uint8, device=device)
        self.v_codes = torch.zeros_like(self.k_codes)
        self.k_scales = torch.zeros(scales, dtype=torch.bfloat16, device=device)
        self.v_scales = torch.zeros_like(self.k_scales)
        self.device = self.k_codes.device
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.v_codes, self.k_scales, self.v_scales))

    def reset(self) -> None:
        """Every position reads as zeros again."""
        for t in (self.k_codes, self.v_codes, self.k_scales, self.v_scales):
            t.zero_()

    def check_rows(self, rows: KVRows) -> None:
        """Refuse what the host knows to be outside the cache."""
        if rows._num_seqs > self.num_seqs:
            raise ValueError(f"rows name sequence {rows._num_seqs - 1}; the cache has {self.num_seqs}")
        if rows._end > self.max_seq_len:
            raise ValueError(f"rows end at position {rows._end - 1}; max_seq_len is {self.max_seq_len}")
        if rows.max_rows > self.max_seq_len:
            raise ValueError(f"max_rows {rows.max_rows} exceeds max_seq_len {self.max_seq_len}")

    def _check(self, rows: KVRows, layer: int, name: str, t: torch.Tensor) -> None:
        if not 0 <= layer < self.num_layers:
            raise ValueError(f"layer {layer} outside [0, {self.num_layers})")
        self.check_rows(rows)
        shape = t.shape
        if len(shape) != 3 or shape[0] != rows.rows or shape[2] != self.head_dim:
            raise ValueError(f"{name} must be [rows={rows.rows}, heads, head_dim={self.head_dim}], got {list(shape)}")

    def write(self, k: torch.Tensor, v: torch.Tensor, rows: KVRows, layer: int = 0) -> None:
        """Quantize ``k`` and ``v`` [rows, kv_heads, head_dim] (bf16, fp16 or
        fp32; any strides with head_dim contiguous) into the rows' positions.
        A NaN is held as 0 and an infinity as the group's end of range; either
        is reported by ``check_status``."""
        self._check(rows, layer, "k", k)  # (v must match k: the operator checks it)
        if rows._overlap:
            raise ValueError("rows hold a position of a sequence twice")
        self._write(self.k_codes, self.v_codes, self.k_scales, self.v_scales, self.bits, self.max_seq_len, layer, k, v,
                    rows.start, rows.row_offsets, rows.seq, rows.max_rows, self.status)

    def read(self, rows: KVRows, layer: int = 0, dtype: torch.dtype = torch.bfloat16,
             out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values that the rows' positions hold, (k, v) [rows, kv_heads,
        head_dim], rounded to ``dtype``; into ``out`` (and its type) if given."""
        k, v = (None, None) if out is None else out
        if out is not None:
            self._check(rows, layer, "out[0]", k)
        elif not 0 <= layer < self.num_layers:
            raise ValueError(f"layer {layer} outside [0, {self.num_layers})")
        else:
            self.check_rows(rows)
        new = self._read(self.k_codes, self.v_codes, self.k_scales, self.v_scales, self.bits, self.max_seq_len, layer,
                         k, v, rows.start, rows.row_offsets, rows.seq, rows.max_rows, rows.rows, dtype,
                         not rows._covers, self.status)
        return new if out is None else out

    def attend(self, q: torch.Tensor, rows: KVRows, layer: int = 0, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of ``q`` [rows, q_heads, head_dim] over the cache:
        the row at position p attends to positions 0 .. p of its sequence, q
        head j to K/V head ``j // (q_heads / kv_heads)``.  ``scale`` defaults to
        1 / sqrt(head_dim).  Returns ``out`` (q's type and shape); rows that no
        segment holds are left as they are in a given ``out`` and 0 else."""
        self._check(rows, layer, "q", q)
        heads = q.shape[1]
        if heads < 1 or heads % self.num_kv_heads or heads // self.num_kv_heads > MAX_RATIO:
            raise ValueError(f"q has {heads} heads: not 1 .. {MAX_RATIO} times the cache's {self.num_kv_heads}")
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype):
            raise ValueError("out must have q's shape and type")
        new = self._attend(self.k_codes, self.v_codes, self.k_scales, self.v_scales, self.bits, self.max_seq_len,
                           layer, q, out, rows.start, rows.row_offsets, rows.seq, rows.max_rows,
                           self._scale if scale is None else float(scale), not rows._covers, self.status)
        return new if out is None else out

    def check_status(self) -> None:
        """Raise KVCacheError if a call since the last check reported
        something (waits for the device)."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            what = []
            if code & BAD_ROW:
                what.append("row with a sequence or position out of range (not written, read as zeros)")
            if code & NONFINITE:
                what.append("NaN or infinity written (held as 0 or as the end of the group's range)")
            if code & TIMEOUT:
                what.append("attention did not complete a copy within 1 s (outputs invalid)")
            if code & COPIES_PENDING:
                what.append("copies still in flight after the drain limit (context suspect: recreate it)")
            raise KVCacheError("quantized K/V cache: " + "; ".join(what))
