"""An 8-bit key/value cache and attention over it: what a decoder block's
CIM layers need between their projections.

The cache is paged: int8 codes [pages, kv_heads, 2, block, head_dim] (0 = key,
1 = value) with one f32 scale for each (page, head, side), so that a code q
stands for q * scale. A page table [batch, width] (int32) names each
sequence's pages; token p of sequence b lies in page table[b, p // block].

Every call takes the sequences alike: ``lengths[b]`` counts the tokens that
sequence b holds with this call's tokens, which are its last ones, and their
rows are packed; sequence b's rows are ``starts[b]`` to ``starts[b + 1] - 1``
(``starts`` None: one row for every sequence, a decoding step). The same
tensors therefore serve the write of a step's keys and values and the
attention of its queries. Lengths, starts and table live on the device, so a
step can be captured into a CUDA graph and replayed with new contents.
``most`` bounds a sequence's rows in the call and ``longest`` its length; both
are host numbers that size the launch (a graph's ``most`` has to cover every
replay; any ``longest`` gives the right results). By default they are all rows and
what the table can hold, which starts many idle blocks for a batch of prompts. Under capture, and to avoid a
synchronization in every call, pass ``status``: without it each call makes a
status word of its own and reads it back. A ``workspace`` belongs to calls that
run one after another, graphs among them.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import abi
from .cim_ops import FLOAT_TYPES, StatusWord, Workspace, launch
from .native import CudaError, lib

BLOCKS = (16, 32, 64, 128)

# abi.KvSequences and abi.KvAttention: packing them takes half the time of
# filling the ctypes structures.
_SEQUENCES = struct.Struct("@iqqiqqqi4x")
_ATTENTION = struct.Struct("@iiqqqqqfiiq")
assert _SEQUENCES.size == ctypes.sizeof(abi.KvSequences)
assert _ATTENTION.size == ctypes.sizeof(abi.KvAttention)


class Int8KVCache:
    """Keys and values of one layer in 8 bits, with a scale for each block of
    tokens and head. ``codes`` and ``scales`` are its tensors, to copy pages from
    and into; the names cannot be bound to others. A deep or unpickled copy is
    a cache over tensors of its own, a shallow one over the same."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, block: int = 64, *,
                 device: int | torch.device = 0) -> None:
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        self._shape_check(pages, kv_heads, head_dim, block)
        if dev.type != "cuda":
            raise TypeError("the cache must lie on a CUDA device")
        self._init(torch.zeros(pages, kv_heads, 2, block, head_dim, dtype=torch.int8, device=dev),
                   torch.zeros(pages, kv_heads, 2, dtype=torch.float32, device=dev))

    @classmethod
    def over(cls, codes: torch.Tensor, scales: torch.Tensor) -> "Int8KVCache":
        """A cache over existing tensors: int8 codes [pages, kv_heads, 2, block,
        head_dim] and f32 scales [pages, kv_heads, 2] (never negative), both
        contiguous."""
        if codes.dim() != 5 or codes.shape[2] != 2:
            raise ValueError("codes must be [pages, kv_heads, 2, block, head_dim]")
        cls._shape_check(codes.shape[0], codes.shape[1], codes.shape[4], codes.shape[3])
        if not codes.is_cuda or codes.dtype != torch.int8 or not codes.is_contiguous() \
                or codes.data_ptr() % 16:
            raise TypeError("codes must be a contiguous CUDA torch.int8 tensor on a 16-byte "
                            "boundary")
        if scales.device != codes.device or scales.dtype != torch.float32 \
                or scales.shape != codes.shape[:3] or not scales.is_contiguous() \
                or scales.data_ptr() % 8:
            raise TypeError("scales must be a contiguous CUDA torch.float32 tensor [pages, "
                            "kv_heads, 2] on an 8-byte boundary, on the codes' device")
        self = cls.__new__(cls)
        self._init(codes, scales)
        return self

    @staticmethod
    def _shape_check(pages: int, kv_heads: int, head_dim: int, block: int) -> None:
        if block not in BLOCKS:
            raise ValueError("block must be 16, 32, 64 or 128 tokens")
        if not 16 <= head_dim <= 128 or head_dim % 16:
            raise ValueError("head_dim must be a multiple of 16 up to 128")
        if not 1 <= kv_heads <= 32767 or not 0 <= pages <= 0x7fffffff:
            raise ValueError("pages or kv_heads out of range")

    def _init(self, codes: torch.Tensor, scales: torch.Tensor) -> None:
        # The calls take addresses. These aliases, which nobody else sees, keep
        # the memory there whatever is done to the tensors that are handed out.
        self._memory = codes.detach(), scales.detach()
        self._codes, self._scales = codes, scales
        self.pages, self.kv_heads, _, self.block, self.head_dim = codes.shape
        self.device, self._index = codes.device, codes.get_device()
        self._view = bytes(abi.KvCache(codes=codes.data_ptr(), scales=scales.data_ptr(),
                                       pages=self.pages, kv_heads=self.kv_heads,
                                       block=self.block, head_dim=self.head_dim))

    @property
    def codes(self) -> torch.Tensor:
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        return self._scales

    def __reduce__(self):  # no addresses: they are taken of the copied tensors
        return type(self).over, (self._codes, self._scales)

    # ------------------------------------------------------------- descriptions

    def _int32(self, t: torch.Tensor, count: int, name: str) -> None:
        if t.dtype != torch.int32 or t.get_device() != self._index or t.dim() != 1 \
                or t.numel() != count or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous int32 tensor [{count}] on the cache's "
                            "device")

    def _sequences(self, table: torch.Tensor, lengths: torch.Tensor,
                   starts: torch.Tensor | None, rows: int, most: int | None) -> tuple:
        """abi.KvSequences' fields."""
        if table.get_device() != self._index or table.dtype != torch.int32 or table.dim() != 2:
            raise TypeError("table must be an int32 tensor [batch, pages a sequence] on the "
                            "cache's device")
        batch, width = table.shape
        stride = width
        if not table.is_contiguous():
            stride = table.stride(0)
            if width > 1 and table.stride(1) != 1 or batch > 1 and stride < width:
                raise TypeError("table rows must be contiguous and must not overlap")
        self._int32(lengths, batch, "lengths")
        if batch > 65535:
            raise ValueError("at most 65535 sequences a call")
        if starts is None:
            if rows != batch:
                raise ValueError("without starts there must be one row for every sequence")
            most = 1
        else:
            self._int32(starts, batch + 1, "starts")
            most = rows if most is None else most
            if not 0 <= most <= 0x7fffffff:
                raise ValueError("most out of range")
        return (batch, table.data_ptr(), stride, width, lengths.data_ptr(),
                0 if starts is None else starts.data_ptr(), rows, most)

    def _rows(self, t: torch.Tensor, heads: int, name: str) -> tuple[int, int]:
        """Checks packed rows; returns their and their heads' strides."""
        if t.dtype not in FLOAT_TYPES or t.get_device() != self._index or t.dim() != 3:
            raise TypeError(f"{name} must be an f32, bf16 or f16 tensor [rows, heads, head_dim] "
                            "on the cache's device")
        _, has, dim = t.shape
        if has != heads or dim != self.head_dim:
            raise ValueError(f"{name} must have {heads} heads of {self.head_dim}")
        if t.is_contiguous():
            return has * dim, dim
        rows, of_heads, last = t.stride()
        if last != 1:
            raise TypeError(f"{name}'s last axis must be contiguous")
        return rows, of_heads

    def _status_word(self, status: StatusWord | None) -> StatusWord:
        if status is None:
            return StatusWord(self.device)
        if status.tensor.get_device() != self._index:
            raise ValueError("status must be on the cache's device")
        return status

    # -------------------------------------------------------------------- calls

    def write(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
              lengths: torch.Tensor, starts: torch.Tensor | None = None, *,
              most: int | None = None, status: StatusWord | None = None) -> None:
        """Quantise packed rows [rows, kv_heads, head_dim] (views of a fused
        projection are fine) into the sequences' last positions.

        A touched block's scale becomes max(its old one, max(amax, 2^-80) / 127)
        with amax over the block's new values; the old one counts only when the
        block holds earlier tokens, whose codes are rounded again where the
        scale grew. Two sequences of one call must not write the same page.
        NaN and infinities are stored as 0 and +-127 and reported through the
        status."""
        k_rows, k_heads = self._rows(k, self.kv_heads, "k")
        v_rows, v_heads = self._rows(v, self.kv_heads, "v")
        rows = k.shape[0]
        if v.shape[0] != rows or k.dtype != v.dtype:
            raise ValueError("k and v must have one shape and type")
        seqs = _SEQUENCES.pack(*self._sequences(table, lengths, starts, rows, most))
        own_status = status is None
        status = self._status_word(status)
        launch("cim22_cuda_kv_write", self._index, lib().cim22_cuda_kv_write, self._view, seqs,
               FLOAT_TYPES[k.dtype], k.data_ptr(), k_rows, k_heads, v.data_ptr(), v_rows, v_heads,
               status.tensor.data_ptr())
        if own_status:
            status.raise_if_set()

    def read(self, table: torch.Tensor, lengths: torch.Tensor,
             starts: torch.Tensor | None = None, *, tokens: int | None = None,
             most: int | None = None, dtype: torch.dtype = torch.float32,
             out: tuple[torch.Tensor, torch.Tensor] | None = None,
             status: StatusWord | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values of each sequence's last starts[b + 1] - starts[b] tokens,
        packed: (k, v), contiguous [tokens, kv_heads, head_dim]; zeros for rows
        that a sequence has no tokens for (an empty slot's). tokens is the number
        of packed rows (starts' last entry; the batch without starts); rows behind
        the last sequence's are left as they are."""
        if out is None:
            if dtype not in FLOAT_TYPES:
                raise TypeError("dtype must be f32, bf16 or f16")
            if tokens is None:
                if starts is not None:
                    raise ValueError("tokens (the number of packed rows) is needed with starts")
                tokens = lengths.shape[0]
            k = torch.empty(tokens, self.kv_heads, self.head_dim, dtype=dtype, device=self.device)
            out = k, torch.empty_like(k)
        k, v = out
        for t, name in ((k, "k"), (v, "v")):
            self._rows(t, self.kv_heads, name)
            if not t.is_contiguous():
                raise TypeError(f"{name} must be contiguous")
        rows = k.shape[0]
        if v.shape[0] != rows or k.dtype != v.dtype:
            raise ValueError("k and v must have one shape and type")
        seqs = _SEQUENCES.pack(*self._sequences(table, lengths, starts, rows, most))
        own_status = status is None
        status = self._status_word(status)
        launch("cim22_cuda_kv_read", self._index, lib().cim22_cuda_kv_read, self._view, seqs,
               FLOAT_TYPES[k.dtype], k.data_ptr(), v.data_ptr(), status.tensor.data_ptr())
        if own_status:
            status.raise_if_set()
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
               starts: torch.Tensor | None = None, *, scale: float | None = None,
               causal: bool = True, window: int = 0, return_lse: bool = False,
               most: int | None = None, longest: int | None = None,
               workspace: Workspace | None = None, out: torch.Tensor | None = None,
               status: StatusWord | None = None):
        """softmax(scale * q k^T) v over the cache, for packed queries [rows,
        q_heads, head_dim] (kv head h serves q heads h * group ...). Query i of
        a sequence's n sits at position lengths[b] - n + i. causal: it sees
        positions up to its own; window > 0: only the last window of them. A
        query that sees nothing gives zeros. scale defaults to
        head_dim ** -0.5; out must not overlap q. Returns out [rows, q_heads,
        head_dim] of q's type, or (out, lse) with the f32 logarithm of each row's
        sum of exponentials. A query row that holds NaN or an infinity gives NaN
        wherever it sees a key. longest: the longest of lengths (default: what the
        table can hold)."""
        if q.dim() != 3:
            raise TypeError("q must be [rows, q_heads, head_dim]")
        rows, heads, _ = q.shape
        row_stride, head_stride = self._rows(q, heads, "q")
        if heads < 1 or heads % self.kv_heads:
            raise ValueError("q_heads must be a multiple of kv_heads")
        seqs = self._sequences(table, lengths, starts, rows, most)
        scale = self.head_dim ** -0.5 if scale is None else float(scale)
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
        if not 0 <= window <= 0x7fffffff:
            raise ValueError("window out of range")
        if longest is None:
            longest = table.shape[1] * self.block
        elif not 0 <= longest <= 0x7fffffffffffffff:
            raise ValueError("longest out of range")
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else \
                torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != self.device \
                or not out.is_contiguous():
            raise TypeError("out must be contiguous, of q's shape and type")
        elif out.data_ptr() == q.data_ptr() and q.numel():
            raise ValueError("out must not be q")
        lse = torch.empty(rows, heads, dtype=torch.float32, device=self.device) \
            if return_lse else None
        call = _ATTENTION.pack(FLOAT_TYPES[q.dtype], heads, q.data_ptr(), row_stride, head_stride,
                               out.data_ptr(), 0 if lse is None else lse.data_ptr(), scale,
                               bool(causal), window, longest)
        seqs = _SEQUENCES.pack(*seqs)
        own_status = status is None
        status = self._status_word(status)
        buffer = None if workspace is None else workspace.buffer
        if buffer is not None and buffer.get_device() != self._index:
            raise ValueError("workspace must be on the cache's device")

        def attend(at: int, nbytes: int) -> None:
            launch("cim22_cuda_kv_attend", self._index, lib().cim22_cuda_kv_attend, self._view,
                   seqs, call, at, nbytes, status.tensor.data_ptr())

        have = 0 if buffer is None else buffer.numel()
        try:
            attend(buffer.data_ptr() if have else 0, have)
        except CudaError: # nothing was launched; most calls need no more than is there
            need = lib().cim22_cuda_kv_attend_workspace(self._view, seqs, call)
            if need <= have:
                raise
            buffer = (workspace or Workspace(self.device)).get(need)
            attend(buffer.data_ptr(), buffer.numel())
        if own_status:
            status.raise_if_set()
        return (out, lse) if return_lse else out
