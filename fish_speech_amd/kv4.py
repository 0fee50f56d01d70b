"""The 4-bit paged K/V cache as a Python object: append, attend, read.

The reference's cache holds K and V in the model's own type (KVCache, fish_speech/models/text2semantic/llama.py:196-214);
:class:`KV4Cache` holds one layer of it at 4.25 bits per value (include/fishmi.h has the number format and the pool's
layout).  ``MiDualAR.setup_caches(..., kv_bits=4)`` makes the slow transformer keep its cache this way; this class offers
the same operators to other attention code.  Everything runs on torch's current stream of the cache's device and may be
captured into a HIP graph; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import FishmiError, Kv4CacheC, Kv4QueryC, Kv4RowsC, check

PAGE = 64   # tokens per page


def page_bytes(n_kv_head: int, head_dim: int) -> int:
    """Bytes one page of 64 tokens takes in the pool of one layer."""
    n = _lib.load().fmi_kv4_page_bytes(int(n_kv_head), int(head_dim))
    if n < 0:
        check(int(n))
    return int(n)


class KV4Cache:
    """One layer's pool of ``n_pages`` pages.  Which pages a sequence owns is the caller's business: every call takes a
    block table, int32 (n_seqs, max_pages), whose entry [s, i] names the page of tokens [64 i, 64 i + 64) of sequence s;
    an id outside [0, n_pages) (-1, say) means "no page"."""

    def __init__(self, n_pages: int, n_kv_head: int, head_dim: int, device="cuda:0", pool: Optional[torch.Tensor] = None):
        self.lib = _lib.load()
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise FishmiError("KV4Cache needs a GPU device (no CPU fallback)")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.n_pages, self.n_kv_head, self.head_dim = int(n_pages), int(n_kv_head), int(head_dim)
        shape = (self.n_pages, self.n_kv_head, 2, page_bytes(n_kv_head, head_dim) // (2 * self.n_kv_head))
        if self.n_pages < 1:
            raise ValueError(f"n_pages {n_pages} must be positive")
        if pool is None:
            pool = torch.zeros(shape, dtype=torch.uint8, device=self.device)
        elif pool.dtype != torch.uint8 or tuple(pool.shape) != shape or pool.device != self.device or not pool.is_contiguous():
            raise ValueError(f"pool must be a contiguous uint8 tensor of shape {shape} on {self.device}")
        self.pool = pool

    # ---- argument checks
    def _index(self, name: str, t: torch.Tensor, n: Optional[int] = None) -> torch.Tensor:
        if t.dtype != torch.int32 or t.device != self.device or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous 1-d int32 tensor on {self.device}")
        if n is not None and t.numel() != n:
            raise ValueError(f"{name} has {t.numel()} entries, expected {n}")
        return t

    def _rows(self, name: str, t: torch.Tensor, rows: Optional[int] = None, heads: Optional[int] = None) -> torch.Tensor:
        if t.dtype != torch.bfloat16 or t.device != self.device or t.dim() != 3 or t.shape[2] != self.head_dim:
            raise ValueError(f"{name} must be a bfloat16 tensor (rows, heads, {self.head_dim}) on {self.device}")
        if (rows is not None and t.shape[0] != rows) or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({rows}, {heads}, {self.head_dim})")
        if t.numel() and (t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != self.head_dim)):
            raise ValueError(f"{name}: the heads of a row must be contiguous (strides {t.stride()})")
        return t

    @staticmethod
    def _stride(t: torch.Tensor) -> int:
        return int(t.stride(0)) if t.shape[0] > 1 else int(t.shape[1] * t.shape[2])

    def _c(self, block_table: torch.Tensor) -> Kv4CacheC:
        if (block_table.dtype != torch.int32 or block_table.device != self.device or block_table.dim() != 2
                or not block_table.is_contiguous()):
            raise ValueError(f"block_table must be a contiguous int32 tensor (n_seqs, max_pages) on {self.device}")
        return Kv4CacheC(self.pool.data_ptr(), block_table.data_ptr(), self.n_pages, self.n_kv_head, self.head_dim,
                         block_table.shape[0], block_table.shape[1])

    def _stream(self):
        return C.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)

    # ---- operators
    def append(self, k: torch.Tensor, v: torch.Tensor, row_seq: torch.Tensor, row_pos: torch.Tensor,
               block_table: torch.Tensor, *, q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
               rope: Optional[torch.Tensor] = None, rope_layout: str = "interleaved",
               q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
               eps: float = 1e-6) -> Optional[torch.Tensor]:
        """Store new tokens: k, v bf16 (rows, n_kv_head, head_dim), row r = position ``row_pos[r]`` of sequence
        ``row_seq[r]``.  On the way, in this order: head RMSNorm of q and k (``q_norm`` / ``k_norm``, bf16 (head_dim,),
        llama.py:862-864), rotation of their first dims by ``rope`` (bf16 (positions, dims / 2, 2), as
        llama.py:1004-1038 builds it; pairs (2 i, 2 i + 1) or, ``rope_layout="half"``, (i, i + dims / 2)).  Returns the
        normed and rotated q (rows, n_head, head_dim) if q was given.

        Rows whose sequence or position lies outside the block table (or the rotation table) are padding: nothing is
        written for them, in the cache or in ``q_out``.  A (sequence, position) pair may appear once per call."""
        rows = int(k.shape[0])
        self._rows("k", k, rows, self.n_kv_head)
        self._rows("v", v, rows, self.n_kv_head)
        self._index("row_seq", row_seq, rows)
        self._index("row_pos", row_pos, rows)
        a = Kv4RowsC(k_dev=k.data_ptr(), v_dev=v.data_ptr(), k_stride=self._stride(k), v_stride=self._stride(v),
                     norm_eps=float(eps), row_seq_dev=row_seq.data_ptr(), row_pos_dev=row_pos.data_ptr(), rows=rows)
        if rope_layout not in ("interleaved", "half"):
            raise ValueError(f"rope_layout {rope_layout!r}: 'interleaved' or 'half'")
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None and (w.dtype != torch.bfloat16 or w.device != self.device or tuple(w.shape) != (self.head_dim,)
                                  or not w.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous bfloat16 tensor ({self.head_dim},) on {self.device}")
        if q is None and (q_norm is not None or q_out is not None):
            raise ValueError("q_norm and q_out go with q")
        if rope is not None:
            if rope.dtype != torch.bfloat16 or rope.device != self.device or rope.dim() != 3 or rope.shape[2] != 2 \
                    or not rope.is_contiguous():
                raise ValueError(f"rope must be a contiguous bfloat16 tensor (positions, dims / 2, 2) on {self.device}")
            a.rope_dev, a.rope_len, a.rope_dim = rope.data_ptr(), rope.shape[0], 2 * rope.shape[1]
            a.rope_half = int(rope_layout == "half")
        a.q_norm_dev = q_norm.data_ptr() if q_norm is not None else None
        a.k_norm_dev = k_norm.data_ptr() if k_norm is not None else None
        if q is not None:
            self._rows("q", q, rows)
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            self._rows("q_out", q_out, rows, int(q.shape[1]))
            if rope is not None and a.rope_half and q_out.data_ptr() == q.data_ptr() and rows:
                raise ValueError("the half-split rotation cannot write q_out over q")
            a.q_dev, a.q_stride, a.n_head = q.data_ptr(), self._stride(q), int(q.shape[1])
            a.q_out_dev, a.q_out_stride = q_out.data_ptr(), self._stride(q_out)
        with torch.cuda.device(self.device):
            check(self.lib.fmi_op_kv4_append(C.byref(self._c(block_table)), C.byref(a), self._stream()))
        return q_out

    def attend(self, q: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, block_table: torch.Tensor, *,
               max_q: int, max_kv: int, out: Optional[torch.Tensor] = None, scale: Optional[float] = None,
               splits: int = 0) -> torch.Tensor:
        """Causal attention over the cache (llama.py:928-934): q bf16 (rows, n_head, head_dim); sequence s has rows
        ``q_start[s] .. q_start[s + 1] - 1`` as its last positions and ``kv_len[s]`` cached keys, its own included;
        both int32 on the device, so a captured graph replays with new lengths.  ``max_q`` / ``max_kv``: upper bounds of
        one sequence's rows and keys (rows beyond ``max_q`` are not computed; ``max_kv`` only tunes the launch).  Rows
        that see no key give 0.  Rows behind the last sequence are left as they were in ``out`` (undefined without one).
        ``splits``: key ranges per query tile, 0 = chosen from the sizes; with a fixed number a row's bits do not depend
        on the other sequences of the call."""
        self._rows("q", q)
        n_seqs = int(block_table.shape[0])
        self._index("q_start", q_start, n_seqs + 1)
        self._index("kv_len", kv_len, n_seqs)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        self._rows("out", out, int(q.shape[0]), int(q.shape[1]))
        c = self._c(block_table)
        a = Kv4QueryC(q_dev=q.data_ptr(), q_stride=self._stride(q), n_head=int(q.shape[1]), q_start_dev=q_start.data_ptr(),
                      kv_len_dev=kv_len.data_ptr(), n_seqs=n_seqs, total_q=int(q.shape[0]), max_q=int(max_q),
                      max_kv=int(max_kv), scale=1.0 / math.sqrt(self.head_dim) if scale is None else float(scale),
                      splits=int(splits))
        need = self.lib.fmi_kv4_attention_ws_bytes(C.byref(c), C.byref(a))
        if need < 0:
            check(int(need))
        # from torch's allocator: ordered with the stream, private to a graph that is being captured
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        with torch.cuda.device(self.device):
            check(self.lib.fmi_op_kv4_attention(C.byref(c), C.byref(a), C.c_void_p(out.data_ptr()), self._stride(out),
                                                C.c_void_p(ws.data_ptr() if ws is not None else None), need,
                                                self._stream()))
        return out

    def read(self, row_seq: torch.Tensor, row_pos: torch.Tensor, block_table: torch.Tensor
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """The stored values of (sequence, position) pairs: k, v bf16 (rows, n_kv_head, head_dim), exact.  Pairs outside
        the sequences, the block table or the pool read as 0."""
        rows = int(row_seq.numel())
        self._index("row_seq", row_seq)
        self._index("row_pos", row_pos, rows)
        k, v = (torch.empty(rows, self.n_kv_head, self.head_dim, dtype=torch.bfloat16, device=self.device) for _ in range(2))
        with torch.cuda.device(self.device):
            check(self.lib.fmi_op_kv4_read(C.byref(self._c(block_table)), C.c_void_p(row_seq.data_ptr()),
                                           C.c_void_p(row_pos.data_ptr()), rows, C.c_void_p(k.data_ptr()),
                                           C.c_void_p(v.data_ptr()), self._stream()))
        return k, v
