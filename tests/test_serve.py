"""CPU tests of the serving operators: geometry and refusals, which answer
before any CUDA call, and the plain restatement's own consistency."""
import ctypes

import numpy as np
import pytest

from cllm_inference_b200 import _lib
from tests import serve_oracle as O

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(264)


def _err(lib, rc, text, code=_lib.ERR_INVALID_ARG):
    assert rc == code
    assert text in _lib.last_error()


def test_page_bytes(lib):
    assert lib.cllm_cuda_kv4_page_bytes(64, 8, 128) == 64 * 8 * 160
    assert lib.cllm_cuda_kv4_page_bytes(16, 1, 64) == 16 * 80
    for geometry in ((0, 8, 128), (20, 8, 128), (64, 0, 128), (64, 8, 96), (-16, 8, 64), (8192, 1, 64)):
        assert lib.cllm_cuda_kv4_page_bytes(*geometry) == 0


def test_append_refusals(lib):
    def call(q=P, ldq=256, q_out=P, k=P, v=P, ldkv=256, n=1, heads=2, rope=None, n_pos=0, seq=P, pos=P, pages=P,
             n_pages=4, page_len=16, kv=2, hd=128, table=P, n_seqs=1, slots=1):
        return lib.cllm_cuda_kv4_append(q, ldq, q_out, k, v, ldkv, n, heads, rope, n_pos, seq, pos, pages, n_pages,
                                        page_len, kv, hd, table, n_seqs, slots, None, None, None)

    _err(lib, call(hd=80), "head_dim 80")
    _err(lib, call(page_len=24), "page_len 24")
    _err(lib, call(page_len=8192), "page_len 8192")
    _err(lib, call(kv=0), "0 KV heads")
    _err(lib, call(n_pages=0), "0 pages")
    for size in (dict(n=-1), dict(heads=-1), dict(n_seqs=0), dict(slots=0), dict(rope=P, n_pos=0)):
        _err(lib, call(**size), "bad sizes")
    for null in ("k", "v", "seq", "pos", "pages", "table", "q", "q_out"):
        _err(lib, call(**{null: None}), "null argument")
    _err(lib, call(pages=ODD), "16-byte aligned")
    _err(lib, call(ldkv=255), "shorter")
    _err(lib, call(ldq=255), "shorter")
    _err(lib, call(ldq=260), "in place")
    assert call(n=0, k=None) == 0


def test_attention_refusals(lib):
    def call(q=P, ldq=512, begin=P, n=3, heads=4, pages=P, n_pages=4, page_len=16, kv=2, hd=128, table=P, lens=P,
             n_seqs=2, slots=2, scale=0.0, out=P):
        return lib.cllm_cuda_kv4_attention(q, ldq, begin, n, heads, pages, n_pages, page_len, kv, hd, table, lens,
                                           n_seqs, slots, scale, out, None, None)

    _err(lib, call(hd=256), "head_dim 256")
    for size in (dict(n=-1), dict(heads=0), dict(heads=5), dict(n_seqs=0), dict(slots=0), dict(slots=2 ** 30),
                 dict(scale=float("inf")), dict(scale=float("nan"))):
        _err(lib, call(**size), "bad sizes")
    _err(lib, call(begin=None), "q_begin")
    for null in ("q", "pages", "table", "lens", "out"):
        _err(lib, call(**{null: None}), "null argument")
    _err(lib, call(pages=ODD), "aligned")
    _err(lib, call(ldq=511), "shorter")
    assert call(n=0, q=None) == 0


def test_fork_and_compact_refusals(lib):
    Q, R = ctypes.c_void_p(512), ctypes.c_void_p(1024)

    def fork(pages=P, layers=1, n_pages=4, page_bytes=1280, page_len=16, table=P, lens=P, n_old=1, source=P, new=P,
             n_new=1, slots=1, out=Q, len_out=R):
        return lib.cllm_cuda_kv4_fork(pages, layers, n_pages, page_bytes, page_len, table, lens, n_old, source, new,
                                      n_new, slots, out, len_out, None)

    for size in (dict(n_old=0), dict(n_new=-1), dict(layers=0), dict(n_pages=0), dict(page_bytes=0),
                 dict(page_bytes=1288), dict(page_len=10), dict(slots=0), dict(slots=2 ** 28)):
        _err(lib, fork(**size), "bad sizes")
    for null in ("pages", "table", "lens", "source", "new", "out", "len_out"):
        _err(lib, fork(**{null: None}), "null argument")
    _err(lib, fork(pages=ODD), "aligned")
    _err(lib, fork(out=P), "buffers of their own")
    _err(lib, fork(len_out=P), "buffers of their own")
    assert fork(n_new=0, pages=None) == 0

    def compact(pages=P, n_seqs=1, table=P, lens=P, out=P, live=P, page_bytes=1280):
        return lib.cllm_cuda_kv4_compact(pages, 1, 4, page_bytes, 16, table, lens, n_seqs, 1, out, live, None)

    for size in (dict(n_seqs=0), dict(page_bytes=8)):
        _err(lib, compact(**size), "bad sizes")
    for null in ("pages", "table", "lens", "out", "live"):
        _err(lib, compact(**{null: None}), "null argument")


def test_scores_refusals(lib):
    def call(x=P, ld=100, rows=2, vocab=100, tokens=P, k=4, logprob=P, rank=P, ids=P, lps=P):
        return lib.cllm_cuda_token_scores(x, ld, rows, vocab, tokens, k, logprob, P, rank, ids, lps, None)

    for size in (dict(rows=-1), dict(vocab=0), dict(ld=99)):
        _err(lib, call(**size), "bad sizes")
    for k in (-1, 33):
        _err(lib, call(k=k), "top_k")
    _err(lib, call(vocab=3), "top_k")
    for null in (dict(x=None), dict(ids=None), dict(lps=None), dict(tokens=None), dict(tokens=None, logprob=None)):
        _err(lib, call(**null), "null argument")
    assert call(rows=0, x=None) == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_a_tile_reads_back_what_was_written(hd):
    rng = np.random.default_rng(hd)
    k, v = rng.standard_normal((2, 16, hd)).astype(np.float32)
    tile = rng.integers(0, 256, 20 * hd).astype(np.uint8)
    for p in rng.permutation(16):
        O.write_position(tile, p, k[p], v[p])
    kr, vr = O.read_tiles(tile, hd)
    np.testing.assert_array_equal(kr, O.values(*O.quantise(k), np.float64))
    np.testing.assert_array_equal(vr, O.values(*O.quantise(v), np.float64))
    step = (k.reshape(16, -1, 32).max(-1) - k.reshape(16, -1, 32).min(-1)) / 15
    assert (np.abs(kr - k).reshape(16, -1, 32).max(-1) <= 0.51 * step + 2.0 ** -9 * np.abs(k).max()).all()
