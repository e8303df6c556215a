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
replay; any ``longest`` gives the right results). Under capture, and to avoid a
synchronization in every call, pass ``status``: without it each call makes a
status word of its own and reads it back. A ``workspace`` belongs to calls that
run one after another, graphs among them.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import abi
from .cim_ops import FLOAT_TYPES, StatusWord, Workspace, launch
from .native import lib

BLOCKS = (16, 32, 64, 128)


class Int8KVCache:
    """Keys and values of one layer in 8 bits, with a scale for each block of
    tokens and head."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, block: int = 64, *,
                 device: int | torch.device = 0) -> None:
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        self._shape_check(pages, kv_heads, head_dim, block)
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
        self.codes, self.scales = codes, scales
        self.pages, self.kv_heads, _, self.block, self.head_dim = codes.shape
        self.device, self._index = codes.device, codes.get_device()
        self._view = abi.KvCache(codes=codes.data_ptr(), scales=scales.data_ptr(),
                                 pages=self.pages, kv_heads=self.kv_heads, block=self.block,
                                 head_dim=self.head_dim)

    # ------------------------------------------------------------- descriptions

    def _int32(self, t: torch.Tensor, count: int, name: str) -> None:
        if t.get_device() != self._index or t.dtype != torch.int32 or t.dim() != 1 \
                or t.shape[0] != count or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous int32 tensor [{count}] on the cache's "
                            "device")

    def _sequences(self, table: torch.Tensor, lengths: torch.Tensor,
                   starts: torch.Tensor | None, rows: int, most: int | None) -> abi.KvSequences:
        if table.get_device() != self._index or table.dtype != torch.int32 or table.dim() != 2:
            raise TypeError("table must be an int32 tensor [batch, pages a sequence] on the "
                            "cache's device")
        batch, width = table.shape
        if not table.is_contiguous() and (width > 1 and table.stride(1) != 1
                                          or batch > 1 and table.stride(0) < width):
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
        return abi.KvSequences(batch, table.data_ptr(), table.stride(0), width,
                               lengths.data_ptr(), None if starts is None else starts.data_ptr(),
                               rows, most)

    def _rows(self, t: torch.Tensor, heads: int, name: str) -> None:
        if t.get_device() != self._index or t.dtype not in FLOAT_TYPES or t.dim() != 3:
            raise TypeError(f"{name} must be an f32, bf16 or f16 tensor [rows, heads, head_dim] "
                            "on the cache's device")
        _, has, dim = t.shape
        if has != heads or dim != self.head_dim:
            raise ValueError(f"{name} must have {heads} heads of {self.head_dim}")
        if t.stride(2) != 1:
            raise TypeError(f"{name}'s last axis must be contiguous")

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
        self._rows(k, self.kv_heads, "k")
        self._rows(v, self.kv_heads, "v")
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must have one shape and type")
        seqs = self._sequences(table, lengths, starts, k.shape[0], most)
        own_status = status is None
        status = status or StatusWord(self.device)
        launch("cim22_cuda_kv_write", self._index, lib().cim22_cuda_kv_write,
               ctypes.byref(self._view), ctypes.byref(seqs), FLOAT_TYPES[k.dtype], k.data_ptr(),
               k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
               status.tensor.data_ptr())
        if own_status:
            status.raise_if_set()

    def read(self, table: torch.Tensor, lengths: torch.Tensor,
             starts: torch.Tensor | None = None, *, tokens: int | None = None,
             most: int | None = None, dtype: torch.dtype = torch.float32,
             out: tuple[torch.Tensor, torch.Tensor] | None = None,
             status: StatusWord | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values of each sequence's last starts[b + 1] - starts[b] tokens,
        packed: (k, v), contiguous [tokens, kv_heads, head_dim]. tokens is the
        number of packed rows (starts' last entry; the batch without starts)."""
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
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must have one shape and type")
        seqs = self._sequences(table, lengths, starts, k.shape[0], most)
        own_status = status is None
        status = status or StatusWord(self.device)
        launch("cim22_cuda_kv_read", self._index, lib().cim22_cuda_kv_read,
               ctypes.byref(self._view), ctypes.byref(seqs), FLOAT_TYPES[k.dtype], k.data_ptr(),
               v.data_ptr(), status.tensor.data_ptr())
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
        head_dim ** -0.5; out must not overlap q. Returns out [rows, q_heads, head_dim] of q's type, or
        (out, lse) with the f32 logarithm of each row's sum of exponentials.
        longest: the longest of lengths (default: what the table can hold)."""
        if q.dim() != 3:
            raise TypeError("q must be [rows, q_heads, head_dim]")
        heads = q.shape[1]
        self._rows(q, heads, "q")
        if heads < 1 or heads % self.kv_heads:
            raise ValueError("q_heads must be a multiple of kv_heads")
        seqs = self._sequences(table, lengths, starts, q.shape[0], most)
        scale = self.head_dim ** -0.5 if scale is None else float(scale)
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
        if not 0 <= window <= 0x7fffffff:
            raise ValueError("window out of range")
        held = seqs.table_width * self.block
        longest = held if longest is None else longest
        if longest < 0:
            raise ValueError("longest must not be negative")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != self.device \
                or not out.is_contiguous():
            raise TypeError("out must be contiguous, of q's shape and type")
        elif out.data_ptr() == q.data_ptr() and q.numel():
            raise ValueError("out must not be q")
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=self.device) \
            if return_lse else None
        call = abi.KvAttention(FLOAT_TYPES[q.dtype], heads, q.data_ptr(), q.stride(0),
                               q.stride(1), out.data_ptr(),
                               None if lse is None else lse.data_ptr(), scale, int(causal),
                               window, longest)
        own_status = status is None
        status = status or StatusWord(self.device)
        cache, seqs, call = ctypes.byref(self._view), ctypes.byref(seqs), ctypes.byref(call)
        ws = None
        nbytes = lib().cim22_cuda_kv_attend_workspace(cache, seqs, call)
        if nbytes:
            ws = (workspace or Workspace(self.device)).get(nbytes)
        launch("cim22_cuda_kv_attend", self._index, lib().cim22_cuda_kv_attend, cache, seqs, call,
               None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(),
               status.tensor.data_ptr())
        if own_status:
            status.raise_if_set()
        return (out, lse) if return_lse else out
