"""The 4-bit paged K/V cache as a Python object: append, attend, step (both in one launch), read.

The reference's cache holds K and V in the model's own type (KVCache, fish_speech/models/text2semantic/llama.py:196-214);
:class:`KV4Cache` holds one layer of it at 4.25 bits per value (include/fishmi.h has the number format and the pool's
layout).  ``MiDualAR.setup_caches(..., kv_bits=4)`` makes the slow transformer keep its cache this way; this class offers
the same operators to other attention code.  Everything runs on torch's current stream of the cache's device and may be
captured into a HIP graph; there is no CPU fallback.
"""
from __future__ import annotations

import functools
import math
import operator
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import FishmiError, check

PAGE = 64   # tokens per page

# The argument structs of include/fishmi.h as packed bytes.  A generation loop makes one append and one attend per layer and
# token, each a few microseconds of GPU work: building a ctypes.Structure field by field took longer than the launch.
_CACHE = struct.Struct("@PPiiiii")              # fmi_kv4_cache
_ROWS = struct.Struct("@PPPqqqPqiPPdPiiiPPi")   # fmi_kv4_rows
_QUERY = struct.Struct("@PqiPPiiiifi")          # fmi_kv4_query
_BF16, _I32 = torch.bfloat16, torch.int32
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def page_bytes(n_kv_head: int, head_dim: int) -> int:
    """Bytes one page of 64 tokens takes in the pool of one layer."""
    n = _lib.load().fmi_kv4_page_bytes(int(n_kv_head), int(head_dim))
    if n < 0:
        check(int(n))
    return int(n)


@functools.lru_cache(maxsize=1024)
def _attention_ws_bytes(n_kv_head: int, head_dim: int, n_head: int, n_seqs: int, rows: int, max_q: int, max_kv: int,
                        splits: int) -> int:
    """fmi_kv4_attention_ws_bytes: a function of these sizes alone (which are checked where they are new)"""
    for name, v in (("max_q", max_q), ("max_kv", max_kv), ("splits", splits)):
        if not -1 << 31 <= v < 1 << 31:
            raise ValueError(f"{name} must be a number of 32 bits, not {v}")
    c = _CACHE.pack(0, 0, 1, n_kv_head, head_dim, n_seqs, 1)
    q = _QUERY.pack(0, 0, n_head, 0, 0, n_seqs, rows, max_q, max_kv, 1.0, splits)
    n = _lib.load().fmi_kv4_attention_ws_bytes(c, q)
    if n < 0:
        check(int(n))
    return int(n)


def _whole(name: str, v) -> int:
    """v, or what it stands for now (a one-element tensor), as an int"""
    try:
        return operator.index(v)
    except TypeError:
        raise ValueError(f"{name} must be a whole number, not {v!r}") from None


def _real(name: str, v) -> float:
    """v as a float that fits an fp32 field (inf and NaN pass: the library refuses them where they mean nothing)"""
    try:
        f = float(v)
    except (TypeError, ValueError):
        raise ValueError(f"{name} must be a number, not {v!r}") from None
    if math.isfinite(f) and abs(f) > 3.4028234663852886e38:
        raise ValueError(f"{name} {f} is out of the range of fp32")
    return f


class KV4Cache:
    """One layer's pool of ``n_pages`` pages.  Which pages a sequence owns is the caller's business: every call takes a
    block table, int32 (n_seqs, max_pages), whose entry [s, i] names the page of tokens [64 i, 64 i + 64) of sequence s;
    an id outside [0, n_pages) (-1, say) means "no page"."""

    def __init__(self, n_pages: int, n_kv_head: int, head_dim: int, device="cuda:0", pool: Optional[torch.Tensor] = None):
        device = torch.device(device)
        if device.type != "cuda":
            raise FishmiError("KV4Cache needs a GPU device (no CPU fallback)")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        block = page_bytes(n_kv_head, head_dim) // (2 * int(n_kv_head))
        if n_pages < 1:
            raise ValueError(f"n_pages {n_pages} must be positive")
        shape = (int(n_pages), int(n_kv_head), 2, block)
        if pool is None:
            pool = torch.zeros(shape, dtype=torch.uint8, device=device)
        elif pool.dtype != torch.uint8 or tuple(pool.shape) != shape or pool.device != device or not pool.is_contiguous():
            raise ValueError(f"pool must be a contiguous uint8 tensor of shape {shape} on {device}")
        self._setup(pool, int(head_dim))

    def _setup(self, pool: torch.Tensor, head_dim: int):
        self.lib = _lib.load()
        self.pool, self.device, self.head_dim = pool, pool.device, head_dim
        self.n_pages, self.n_kv_head = int(pool.shape[0]), int(pool.shape[1])
        self._dev = pool.get_device()

    # ---- argument checks (ordered for the calls that pass: a handful of attribute reads each)
    def _index(self, name: str, t: torch.Tensor, n: int) -> int:
        """-> the address of a contiguous int32 vector of n entries"""
        if t.dtype is not _I32 or t.get_device() != self._dev or not t.is_contiguous() or t.shape != (n,):
            raise ValueError(f"{name} must be a contiguous int32 tensor ({n},) on {self.device}, not {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        return t.data_ptr()

    def _rows(self, name: str, t: torch.Tensor, rows: int, heads: int) -> int:
        """-> the row stride of a bf16 tensor (rows, heads, head_dim) whose rows are contiguous"""
        D = self.head_dim
        if t.dtype is not _BF16 or t.get_device() != self._dev or t.shape != (rows, heads, D):
            raise ValueError(f"{name} must be a bfloat16 tensor {(rows, heads, D)} on {self.device}, not {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        s0, s1, s2 = t.stride()
        if rows and (s2 != 1 or (s1 != D and heads != 1)):
            raise ValueError(f"{name}: the heads of a row must be contiguous (strides {(s0, s1, s2)})")
        return s0 if rows > 1 else heads * D

    def _cache(self, block_table: torch.Tensor) -> bytes:
        if (block_table.dtype is not _I32 or block_table.get_device() != self._dev or block_table.dim() != 2
                or not block_table.is_contiguous()):
            raise ValueError(f"block_table must be a contiguous int32 tensor (n_seqs, max_pages) on {self.device}")
        n, w = block_table.shape
        return _CACHE.pack(self.pool.data_ptr(), block_table.data_ptr(), self.n_pages, self.n_kv_head, self.head_dim, n, w)

    def _new(self, rows: int, heads: int) -> torch.Tensor:
        D = self.head_dim      # (torch.empty without strides takes a third longer)
        return torch.empty_strided((rows, heads, D), (heads * D, D, 1), dtype=_BF16, device=self.device)

    def _call(self, fn, *args):
        """fn(*args, stream) with the cache's device current"""
        dev = self._dev
        if _current_device() == dev:
            rc = fn(*args, _raw_stream(dev))
        else:
            with torch.cuda.device(dev):
                rc = fn(*args, _raw_stream(dev))
        if rc:
            check(rc)

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
        normed and rotated q (rows, n_head, head_dim) if q was given (into ``q_out``, which may be q itself unless the
        rotation is half-split).

        Rows whose sequence or position lies outside the block table (or the rotation table) are padding: nothing is
        written for them, in the cache or in ``q_out``.  A (sequence, position) pair may appear once per call."""
        qp = qs = op = os = heads = 0
        rows = k.shape[0]
        if q is not None:
            heads = q.shape[1] if q.dim() == 3 else 0
            qs, qp = self._rows("q", q, rows, heads), q.data_ptr()
            if q_out is None:
                q_out, os = self._new(rows, heads), heads * self.head_dim
            else:
                os = self._rows("q_out", q_out, rows, heads)
            op = q_out.data_ptr()
        elif q_norm is not None or q_out is not None:
            raise ValueError("q_norm and q_out go with q")
        if qp and op == qp and rope is not None and rope_layout == "half":
            raise ValueError("the half-split rotation cannot write q_out over q")
        a = self._new_rows(qp, qs, op, os, heads, k, v, row_seq, row_pos, rope, rope_layout, q_norm, k_norm, eps)
        self._call(self.lib.fmi_op_kv4_append, self._cache(block_table), a)
        return q_out

    def _new_rows(self, qp, qs, op, os, heads, k, v, row_seq, row_pos, rope, rope_layout, q_norm, k_norm, eps) -> bytes:
        """-> fmi_kv4_rows of checked arguments"""
        rows, KVH = k.shape[0], self.n_kv_head
        ks, vs = self._rows("k", k, rows, KVH), self._rows("v", v, rows, KVH)
        ps, pp = self._index("row_seq", row_seq, rows), self._index("row_pos", row_pos, rows)
        if rope_layout not in ("interleaved", "half"):
            raise ValueError(f"rope_layout {rope_layout!r}: 'interleaved' or 'half'")
        qn = kn = rp = rl = rd = 0
        if rope is not None:
            if (rope.dtype is not _BF16 or rope.get_device() != self._dev or rope.dim() != 3 or rope.shape[2] != 2
                    or not rope.is_contiguous()):
                raise ValueError(f"rope must be a contiguous bfloat16 tensor (positions, dims / 2, 2) on {self.device}")
            rp, rl, rd = rope.data_ptr(), rope.shape[0], 2 * rope.shape[1]
        if q_norm is not None:
            qn = self._weight("q_norm", q_norm)
        if k_norm is not None:
            kn = self._weight("k_norm", k_norm)
        if type(eps) is not float:
            eps = _real("eps", eps)
        return _ROWS.pack(qp, k.data_ptr(), v.data_ptr(), qs, ks, vs, op, os, heads, qn, kn, eps, rp, rl, rd,
                          rope_layout == "half", ps, pp, rows)

    def _weight(self, name: str, w: torch.Tensor) -> int:
        if w.dtype is not _BF16 or w.get_device() != self._dev or w.shape != (self.head_dim,) or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous bfloat16 tensor ({self.head_dim},) on {self.device}")
        return w.data_ptr()

    def attend(self, q: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, block_table: torch.Tensor, *,
               max_q: int, max_kv: int, out: Optional[torch.Tensor] = None, scale: Optional[float] = None,
               splits: int = 0) -> torch.Tensor:
        """Causal attention over the cache (llama.py:928-934): q bf16 (rows, n_head, head_dim); sequence s has rows
        ``q_start[s] .. q_start[s + 1] - 1`` as its last positions and ``kv_len[s]`` cached keys, its own included;
        both int32 on the device, so a captured graph replays with new lengths.  ``max_q`` / ``max_kv``: upper bounds of
        one sequence's rows and keys (rows beyond ``max_q`` are not computed; ``max_kv`` only tunes the launch).  Rows
        that see no key give 0, rows whose q holds an infinity or a NaN give NaN.  Rows behind the last sequence are left as they were in ``out`` (undefined without one;
        it may be q itself).
        ``splits``: key ranges per query tile, 0 = chosen from the sizes; with a fixed number (and ``max_q``) a row's bits
        do not depend on the other sequences of the call."""
        n, heads = q.shape[0], q.shape[1] if q.dim() == 3 else 0
        qs = self._rows("q", q, n, heads)
        c = self._cache(block_table)
        n_seqs = block_table.shape[0]
        sp, lp = self._index("q_start", q_start, n_seqs + 1), self._index("kv_len", kv_len, n_seqs)
        if out is None:
            out, os = self._new(n, heads), heads * self.head_dim
        else:
            os = self._rows("out", out, n, heads)
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else _real("scale", scale)
        if type(max_q) is not int:
            max_q = _whole("max_q", max_q)
        if type(max_kv) is not int:
            max_kv = _whole("max_kv", max_kv)
        if type(splits) is not int:
            splits = _whole("splits", splits)
        need = _attention_ws_bytes(self.n_kv_head, self.head_dim, heads, n_seqs, n, max_q, max_kv, splits)
        a = _QUERY.pack(q.data_ptr(), qs, heads, sp, lp, n_seqs, n, max_q, max_kv, scale, splits)
        if need:           # from torch's allocator: ordered with the stream, private to a graph that is being captured
            ws = torch.empty(need, dtype=torch.uint8, device=self.device)
            self._call(self.lib.fmi_op_kv4_attention, c, a, out.data_ptr(), os, ws.data_ptr(), need)
        else:
            self._call(self.lib.fmi_op_kv4_attention, c, a, out.data_ptr(), os, 0, 0)
        return out

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, row_seq: torch.Tensor, row_pos: torch.Tensor,
             block_table: torch.Tensor, *, max_kv: int, rope: Optional[torch.Tensor] = None, rope_layout: str = "interleaved",
             q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
             out: Optional[torch.Tensor] = None, scale: Optional[float] = None, splits: int = 0) -> torch.Tensor:
        """A generation step, one new token per sequence, in one launch: ``append`` of the rows, then the attention of each
        row's q over the keys up to its own position -- the same stored bytes and the same output as ``append`` and ``attend``
        (with the same ``splits``).  A sequence may have one row per call; padding rows are left as they were in ``out``
        (undefined without one).  The other arguments are theirs."""
        rows, heads = k.shape[0], q.shape[1] if q.dim() == 3 else 0
        qs = self._rows("q", q, rows, heads)
        a = self._new_rows(q.data_ptr(), qs, 0, 0, heads, k, v, row_seq, row_pos, rope, rope_layout, q_norm, k_norm, eps)
        if out is None:
            out, os = self._new(rows, heads), heads * self.head_dim
        else:
            os = self._rows("out", out, rows, heads)
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else _real("scale", scale)
        if type(max_kv) is not int:
            max_kv = _whole("max_kv", max_kv)
        if type(splits) is not int:
            splits = _whole("splits", splits)
        need = _attention_ws_bytes(self.n_kv_head, self.head_dim, max(heads, 1), rows, rows, 1, max_kv, splits)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None    # (as in attend)
        self._call(self.lib.fmi_op_kv4_step, self._cache(block_table), a, scale, max_kv, splits, out.data_ptr(), os,
                   ws.data_ptr() if need else 0, need)
        return out

    def read(self, row_seq: torch.Tensor, row_pos: torch.Tensor, block_table: torch.Tensor
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """The stored values of (sequence, position) pairs: k, v bf16 (rows, n_kv_head, head_dim), exact.  Pairs outside
        the sequences, the block table or the pool read as 0."""
        rows = row_seq.numel()
        sp, pp = self._index("row_seq", row_seq, rows), self._index("row_pos", row_pos, rows)
        k, v = self._new(rows, self.n_kv_head), self._new(rows, self.n_kv_head)
        self._call(self.lib.fmi_op_kv4_read, self._cache(block_table), sp, pp, rows, k.data_ptr(), v.data_ptr())
        return k, v
