"""Many sequences in one paged cache held in 4 bits (include/cllm_cuda.h,
"Serving many sequences"; cllm_cuda_kv4_*).

The reference serves one sequence from a contiguous fp32 cache
(src/core/engine.cpp:119-146); here any number of sequences share a pool of
pages that takes 1.25 bytes per key/value pair of numbers instead of 8:

    cache = KV4Cache.empty(n_layers, n_pages, 64, n_head_kv, head_dim, n_seqs, max_pages)
    cache = cache.fork(source, new_len)      # start, fork, grow, free sequences
    q = cache.append(layer, k, v, seq, pos, q=q, rope=table)
    o = cache.attention(layer, q)            # one new row per sequence
    cache, live = cache.compact()

Everything runs on torch's current stream, reads nothing back to the host and
can be captured into a CUDA graph.  fork and compact move pages in place and
return a cache with a new table; the old one must not be used after them.
There is no fallback: without the CUDA library the calls fail.
"""
from __future__ import annotations

import torch

from . import _lib

TILE = 16  # positions of a tile; a page is a whole number of tiles


def page_bytes(page_len: int, n_head_kv: int, head_dim: int) -> int:
    """Bytes of one page of one layer."""
    n = _lib.load().cllm_cuda_kv4_page_bytes(page_len, n_head_kv, head_dim)
    if n == 0:
        raise _lib.CudaError(_lib.ERR_INVALID_ARG,
                             f"kv4: page_len {page_len}, {n_head_kv} KV heads, head_dim {head_dim} is not supported")
    return n


def _ready(t: torch.Tensor, dtype, what: str) -> None:
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise _lib.CudaError(_lib.ERR_INVALID_ARG, f"kv4: {what} must be a contiguous CUDA tensor of {dtype}")


def _rows(t: torch.Tensor, what: str) -> tuple[int, int]:
    """(address, row stride) of a 2-D fp32 tensor whose rows are contiguous."""
    if not t.is_cuda or t.dtype != torch.float32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise _lib.CudaError(_lib.ERR_INVALID_ARG, f"kv4: {what} must be a 2-D fp32 CUDA tensor with dense rows")
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class KV4Cache:
    """A pool of pages, the sequences in it and their lengths.

    pages: uint8 [layer][page][kv head][page_len / 16][20 * head_dim]
    table: int32 [sequence][slot], page ids; lens: int32 [sequence]
    """

    def __init__(self, pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor):
        _ready(pages, torch.uint8, "pages")
        _ready(table, torch.int32, "table")
        _ready(lens, torch.int32, "lens")
        if pages.dim() != 5 or table.dim() != 2 or lens.shape[0] != table.shape[0] or pages.shape[4] not in (1280, 2560):
            raise _lib.CudaError(_lib.ERR_INVALID_ARG, "kv4: pages [layer][page][kv head][page_len/16][20 head_dim], "
                                                       "table [sequence][slot], lens [sequence]")
        self.lib = _lib.load()
        self.pages, self.table, self.lens = pages, table, lens
        self.n_layers, self.n_pages, self.n_head_kv = pages.shape[:3]
        self.page_len, self.head_dim = pages.shape[3] * TILE, pages.shape[4] // 20
        self.n_seqs, self.max_pages = table.shape
        self.page_bytes = pages.shape[2] * pages.shape[3] * pages.shape[4]

    @classmethod
    def empty(cls, n_layers: int, n_pages: int, page_len: int, n_head_kv: int, head_dim: int, n_seqs: int,
              max_pages: int, device="cuda") -> "KV4Cache":
        """A pool with n_seqs sequences of no positions."""
        page_bytes(page_len, n_head_kv, head_dim)
        pages = torch.zeros((n_layers, n_pages, n_head_kv, page_len // TILE, 20 * head_dim), dtype=torch.uint8,
                            device=device)
        return cls(pages, torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(n_seqs, dtype=torch.int32, device=device))

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.n_layers:
            raise _lib.CudaError(_lib.ERR_INVALID_ARG, f"kv4: layer {layer} of {self.n_layers}")
        return self.pages.data_ptr() + layer * self.n_pages * self.page_bytes

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, seq: torch.Tensor, pos: torch.Tensor,
               q: torch.Tensor | None = None, rope: torch.Tensor | None = None, values: bool = False):
        """Write the rows of k and v (rotated by `rope`, the table of cllm_cuda_rope_table, where given) as the
        positions `pos` of the sequences `seq`.  Returns the rotated q (None without q); with `values` also the
        keys and values that the cache now holds: (q, k, v)."""
        _ready(seq, torch.int32, "seq")
        _ready(pos, torch.int32, "pos")
        n, kv_dim = k.shape[0], self.n_head_kv * self.head_dim
        kp, ldkv = _rows(k, "k")
        vp, ldv = _rows(v, "v")
        if k.shape[1] != kv_dim or v.shape != k.shape or ldv != ldkv or seq.numel() != n or pos.numel() != n:
            raise _lib.CudaError(_lib.ERR_INVALID_ARG, f"kv4: k and v are rows of {kv_dim} values with one stride, "
                                                       "seq and pos one entry a row")
        qp, ldq, heads, q_out = 0, 0, 0, None
        if q is not None:
            qp, ldq = _rows(q, "q")
            heads = q.shape[1] // self.head_dim
            if q.shape[0] != n or q.shape[1] % self.head_dim:
                raise _lib.CudaError(_lib.ERR_INVALID_ARG, f"kv4: q has a row per token, of heads of {self.head_dim}")
            q_out = torch.empty((n, q.shape[1]), dtype=torch.float32, device=q.device)
        if rope is not None:
            _ready(rope, torch.float32, "rope")
            if rope.numel() % self.head_dim:
                raise _lib.CudaError(_lib.ERR_INVALID_ARG, "kv4: rope is [position][head_dim / 2][2]")
        k_out = v_out = None
        if values:
            k_out = torch.empty((n, kv_dim), dtype=torch.float32, device=k.device)
            v_out = torch.empty((n, kv_dim), dtype=torch.float32, device=k.device)
        _lib.check(self.lib.cllm_cuda_kv4_append(
            qp, ldq, q_out.data_ptr() if heads else 0, kp, vp, ldkv, n, heads,
            0 if rope is None else rope.data_ptr(), 0 if rope is None else rope.numel() // self.head_dim,
            seq.data_ptr(), pos.data_ptr(), self._layer(layer), self.n_pages, self.page_len, self.n_head_kv,
            self.head_dim, self.table.data_ptr(), self.n_seqs, self.max_pages, k_out.data_ptr() if values else 0,
            v_out.data_ptr() if values else 0, _stream(k.device)))
        return (q_out, k_out, v_out) if values else q_out

    def attention(self, layer: int, q: torch.Tensor, begin: torch.Tensor | None = None, scale: float = 0.0,
                  lse: bool = False):
        """Attention of the newest rows of every sequence: sequence s brings the rows begin[s] .. begin[s+1] of q
        (one each without `begin`), the last of which sees all its positions.  Returns [rows][heads * head_dim];
        with `lse` also [rows][heads], the log of the softmax's sum."""
        qp, ldq = _rows(q, "q")
        n, heads = q.shape[0], q.shape[1] // self.head_dim
        if q.shape[1] % self.head_dim:
            raise _lib.CudaError(_lib.ERR_INVALID_ARG, f"kv4: q has rows of heads of {self.head_dim}")
        if begin is not None:
            _ready(begin, torch.int32, "begin")
            if begin.numel() != self.n_seqs + 1:
                raise _lib.CudaError(_lib.ERR_INVALID_ARG, "kv4: begin has an entry more than there are sequences")
        out = torch.empty((n, q.shape[1]), dtype=torch.float32, device=q.device)
        logs = torch.empty((n, heads), dtype=torch.float32, device=q.device) if lse else None
        _lib.check(self.lib.cllm_cuda_kv4_attention(
            qp, ldq, 0 if begin is None else begin.data_ptr(), n, heads, self._layer(layer), self.n_pages,
            self.page_len, self.n_head_kv, self.head_dim, self.table.data_ptr(), self.lens.data_ptr(), self.n_seqs,
            self.max_pages, scale, out.data_ptr(), logs.data_ptr() if lse else 0, _stream(q.device)))
        return (out, logs) if lse else out

    def fork(self, source: torch.Tensor, new_len: torch.Tensor) -> "KV4Cache":
        """New sequence s continues old sequence source[s] (-1: none) and has room for new_len[s] positions; old
        sequences that none continues are freed.  A sequence that finds no room has length -1 afterwards."""
        _ready(source, torch.int32, "source")
        _ready(new_len, torch.int32, "new_len")
        n = source.numel()
        if new_len.numel() != n:
            raise _lib.CudaError(_lib.ERR_INVALID_ARG, "kv4: source and new_len have one entry per new sequence")
        table = torch.empty((n, self.max_pages), dtype=torch.int32, device=self.table.device)
        lens = torch.empty(n, dtype=torch.int32, device=self.table.device)
        _lib.check(self.lib.cllm_cuda_kv4_fork(
            self.pages.data_ptr(), self.n_layers, self.n_pages, self.page_bytes, self.page_len,
            self.table.data_ptr(), self.lens.data_ptr(), self.n_seqs, source.data_ptr(), new_len.data_ptr(), n,
            self.max_pages, table.data_ptr(), lens.data_ptr(), _stream(table.device)))
        return KV4Cache(self.pages, table, lens)

    def compact(self) -> tuple["KV4Cache", torch.Tensor]:
        """Move the pages in use to the lowest ids; returns the cache and their number (int32 [1])."""
        table = torch.empty_like(self.table)
        live = torch.empty(1, dtype=torch.int32, device=self.table.device)
        _lib.check(self.lib.cllm_cuda_kv4_compact(
            self.pages.data_ptr(), self.n_layers, self.n_pages, self.page_bytes, self.page_len,
            self.table.data_ptr(), self.lens.data_ptr(), self.n_seqs, self.max_pages, table.data_ptr(),
            live.data_ptr(), _stream(table.device)))
        return KV4Cache(self.pages, table, self.lens), live
