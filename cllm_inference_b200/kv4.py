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

Everything runs on torch's current stream of the cache's device, whichever device
is current, with tensors of that device, and reads nothing back to the host.  It
can be captured into a CUDA graph, after a call of that size outside of it.  The
library has one workspace for a device: attention, fork and compact on several
streams, or in graphs, must not overlap on the GPU (order them with events).
fork and compact move pages in place and return a cache with a new table; the old
one must not be used after them (but see fork, where the pool is too small).
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


_I32, _F32, _U8 = torch.int32, torch.float32, torch.uint8
_raw_stream = torch._C._cuda_getCurrentRawStream  # torch's current stream of a device, as an integer
_current_device = torch._C._cuda_getDevice


def _refuse(what: str):
    raise _lib.CudaError(_lib.ERR_INVALID_ARG, "kv4: " + what)


def _ready(t: torch.Tensor, dtype, what: str, device: int) -> None:
    if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous():
        _refuse(f"{what} must be a contiguous tensor of {dtype} on cuda:{device}")


def _rows(t: torch.Tensor, what: str, device: int) -> tuple[int, int, int]:
    """(rows, values in a row, row stride) of a 2-D fp32 tensor whose rows are dense."""
    steps = t.stride()
    if len(steps) != 2 or t.dtype is not _F32 or t.get_device() != device:
        _refuse(f"{what} must be a 2-D fp32 tensor with dense rows on cuda:{device}")
    n, width = t.shape
    ld, step = steps
    if step != 1 and width > 1:
        _refuse(f"{what} must be a 2-D fp32 tensor with dense rows on cuda:{device}")
    return n, width, ld if n > 1 else width


def _dense_like(t: torch.Tensor) -> torch.Tensor:
    out = torch.empty_like(t)
    return out if out.is_contiguous() else t.new_empty(t.shape)


class KV4Cache:
    """A pool of pages, the sequences in it and their lengths.

    pages: uint8 [layer][page][kv head][page_len / 16][20 * head_dim]
    table: int32 [sequence][slot], page ids; lens: int32 [sequence]
    """

    __slots__ = ("lib", "pages", "table", "lens", "n_layers", "n_pages", "n_head_kv", "page_len", "head_dim",
                 "n_seqs", "max_pages", "page_bytes", "device")

    def __init__(self, pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor):
        self.device = device = pages.get_device()
        if device < 0:
            _refuse("pages must be a CUDA tensor")
        _ready(pages, _U8, "pages", device)
        _ready(table, _I32, "table", device)
        _ready(lens, _I32, "lens", device)
        shape, slots = pages.shape, table.shape
        if len(shape) != 5 or len(slots) != 2 or lens.shape != slots[:1] or shape[4] not in (1280, 2560):
            _refuse("pages [layer][page][kv head][page_len/16][20 head_dim], table [sequence][slot], lens [sequence]")
        self.lib = _lib.load()
        self.pages, self.table, self.lens = pages, table, lens
        self.n_layers, self.n_pages, self.n_head_kv, tiles, tile_bytes = shape
        self.page_len, self.head_dim = tiles * TILE, tile_bytes // 20
        self.n_seqs, self.max_pages = slots
        self.page_bytes = self.n_head_kv * tiles * tile_bytes

    @classmethod
    def empty(cls, n_layers: int, n_pages: int, page_len: int, n_head_kv: int, head_dim: int, n_seqs: int,
              max_pages: int, device="cuda") -> "KV4Cache":
        """A pool with n_seqs sequences of no positions."""
        page_bytes(page_len, n_head_kv, head_dim)
        pages = torch.zeros((n_layers, n_pages, n_head_kv, page_len // TILE, 20 * head_dim), dtype=_U8, device=device)
        return cls(pages, torch.full((n_seqs, max_pages), -1, dtype=_I32, device=device),
                   torch.zeros(n_seqs, dtype=_I32, device=device))

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.n_layers:
            _refuse(f"layer {layer} of {self.n_layers}")
        return self.pages.data_ptr() + layer * self.n_pages * self.page_bytes

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, seq: torch.Tensor, pos: torch.Tensor,
               q: torch.Tensor | None = None, rope: torch.Tensor | None = None, values: bool = False):
        """Write the rows of k and v (rotated by `rope`, the table of cllm_cuda_rope_table, where given) as the
        positions `pos` of the sequences `seq`.  Returns the rotated q (None without q); with `values` also the
        keys and values that the cache now holds: (q, k, v)."""
        device = self.device
        if _current_device() != device:  # the C calls launch on the current device
            with torch.cuda.device(device):
                return self.append(layer, k, v, seq, pos, q, rope, values)
        _ready(seq, _I32, "seq", device)
        _ready(pos, _I32, "pos", device)
        n, kv_dim, ldkv = _rows(k, "k", device)
        if (n, kv_dim, ldkv) != _rows(v, "v", device) or kv_dim != self.n_head_kv * self.head_dim or seq.numel() != n or \
                pos.numel() != n:
            _refuse(f"k and v are rows of {self.n_head_kv * self.head_dim} values with one stride, seq and pos one "
                    "entry a row")
        qp = ldq = heads = qo = 0
        q_out = None
        if q is not None:
            nq, width, ldq = _rows(q, "q", device)
            heads = width // self.head_dim
            if nq != n or width % self.head_dim:
                _refuse(f"q has a row per token, of heads of {self.head_dim}")
            q_out = _dense_like(q)
            qp, qo = q.data_ptr(), q_out.data_ptr()
        table = n_pos = 0
        if rope is not None:
            _ready(rope, _F32, "rope", device)
            n_pos, rest = divmod(rope.numel(), self.head_dim)
            if rest:
                _refuse("rope is [position][head_dim / 2][2]")
            table = rope.data_ptr()
        k_out = v_out = None
        ko = vo = 0
        if values:
            k_out, v_out = _dense_like(k), _dense_like(v)
            ko, vo = k_out.data_ptr(), v_out.data_ptr()
        rc = self.lib.cllm_cuda_kv4_append(
            qp, ldq, qo, k.data_ptr(), v.data_ptr(), ldkv, n, heads, table, n_pos, seq.data_ptr(), pos.data_ptr(),
            self._layer(layer), self.n_pages, self.page_len, self.n_head_kv, self.head_dim, self.table.data_ptr(),
            self.n_seqs, self.max_pages, ko, vo, _raw_stream(device))
        if rc:
            _lib.check(rc)
        return (q_out, k_out, v_out) if values else q_out

    def attention(self, layer: int, q: torch.Tensor, begin: torch.Tensor | None = None, scale: float = 0.0,
                  lse: bool = False):
        """Attention of the newest rows of every sequence: sequence s brings the rows begin[s] .. begin[s+1] of q
        (one each without `begin`), the last of which sees all its positions.  Returns [rows][heads * head_dim];
        with `lse` also [rows][heads], the log of the softmax's sum."""
        device = self.device
        if _current_device() != device:
            with torch.cuda.device(device):
                return self.attention(layer, q, begin, scale, lse)
        n, width, ldq = _rows(q, "q", device)
        heads = width // self.head_dim
        if width % self.head_dim:
            _refuse(f"q has rows of heads of {self.head_dim}")
        first = 0
        if begin is not None:
            _ready(begin, _I32, "begin", device)
            if begin.numel() != self.n_seqs + 1:
                _refuse("begin has an entry more than there are sequences")
            first = begin.data_ptr()
        out = _dense_like(q)
        logs = q.new_empty((n, heads)) if lse else None
        rc = self.lib.cllm_cuda_kv4_attention(
            q.data_ptr(), ldq, first, n, heads, self._layer(layer), self.n_pages, self.page_len, self.n_head_kv,
            self.head_dim, self.table.data_ptr(), self.lens.data_ptr(), self.n_seqs, self.max_pages, scale,
            out.data_ptr(), logs.data_ptr() if lse else 0, _raw_stream(device))
        if rc:
            _lib.check(rc)
        return (out, logs) if lse else out

    def _with(self, table: torch.Tensor, lens: torch.Tensor, n_seqs: int) -> "KV4Cache":
        """This pool with other sequences."""
        new = KV4Cache.__new__(KV4Cache)
        new.lib, new.pages, new.table, new.lens = self.lib, self.pages, table, lens
        new.n_layers, new.n_pages, new.n_head_kv = self.n_layers, self.n_pages, self.n_head_kv
        new.page_len, new.head_dim, new.page_bytes = self.page_len, self.head_dim, self.page_bytes
        new.n_seqs, new.max_pages, new.device = n_seqs, self.max_pages, self.device
        return new

    def fork(self, source: torch.Tensor, new_len: torch.Tensor) -> "KV4Cache":
        """New sequence s continues old sequence source[s] (-1: none) and has room for new_len[s] positions; old
        sequences that none continues are freed.  The first sequence that finds no room and all after it have length -1
        afterwards.  Then this cache can be forked again, before anything is appended, with fewer or smaller requests
        that continue no more of a sequence; the first result is void."""
        device = self.device
        if _current_device() != device:
            with torch.cuda.device(device):
                return self.fork(source, new_len)
        _ready(source, _I32, "source", device)
        _ready(new_len, _I32, "new_len", device)
        n = source.numel()
        if new_len.numel() != n:
            _refuse("source and new_len have one entry per new sequence")
        if self.n_seqs == 0 and n > 0:  # the C call wants an old sequence: an empty one that no source names
            one = self._with(self.table.new_zeros((1, self.max_pages)), self.lens.new_zeros(1), 1)
            return one.fork(torch.where(source < 0, source, 1), new_len)
        table = torch.empty_like(self.table) if n == self.n_seqs else self.table.new_empty((n, self.max_pages))
        lens = torch.empty_like(new_len)
        rc = self.lib.cllm_cuda_kv4_fork(
            self.pages.data_ptr(), self.n_layers, self.n_pages, self.page_bytes, self.page_len,
            self.table.data_ptr(), self.lens.data_ptr(), self.n_seqs, source.data_ptr(), new_len.data_ptr(), n,
            self.max_pages, table.data_ptr(), lens.data_ptr(), _raw_stream(device))
        if rc:
            _lib.check(rc)
        return self._with(table, lens, n)

    def compact(self) -> tuple["KV4Cache", torch.Tensor]:
        """Move the pages in use to the lowest ids; returns the cache and their number (int32 [1])."""
        device = self.device
        if _current_device() != device:
            with torch.cuda.device(device):
                return self.compact()
        if self.n_seqs == 0:
            return self, self.lens.new_zeros(1)
        table = torch.empty_like(self.table)
        live = self.lens.new_empty(1)
        rc = self.lib.cllm_cuda_kv4_compact(
            self.pages.data_ptr(), self.n_layers, self.n_pages, self.page_bytes, self.page_len,
            self.table.data_ptr(), self.lens.data_ptr(), self.n_seqs, self.max_pages, table.data_ptr(),
            live.data_ptr(), _raw_stream(device))
        if rc:
            _lib.check(rc)
        return self._with(table, self.lens, self.n_seqs), live
