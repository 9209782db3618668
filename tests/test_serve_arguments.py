"""Arguments of the serving operators that the first refusal tests (test_serve.py) leave out; no GPU."""
import ctypes

import pytest

from cllm_inference_b200 import _lib


def _at(i):
    return ctypes.c_void_p(256 * i)


@pytest.mark.parametrize("alias", ["source", "new_len"])
def test_fork_refuses_lengths_written_over_its_request(lib, alias):
    """Every CTA of the one-launch form reads the request while others write the lengths."""
    request = {"source": _at(4), "new_len": _at(5)}
    rc = lib.cllm_cuda_kv4_fork(_at(1), 1, 4, 1280, 16, _at(2), _at(3), 1, request["source"], request["new_len"], 1, 1,
                                _at(6), request[alias], None)
    assert rc == _lib.ERR_INVALID_ARG and "buffers of their own" in _lib.last_error()


def test_scores_take_one_row_for_all(lib):
    """A row stride of 0 (an expanded row) is an argument like any other: it gets past the sizes."""
    def call(ld, logits=_at(1)):
        return lib.cllm_cuda_token_scores(logits, ld, 2, 100, None, 0, None, _at(2), None, None, None, None)

    assert call(0, None) == _lib.ERR_INVALID_ARG and "null argument" in _lib.last_error()
    for ld in (-100, -1, 1, 99):
        assert call(ld) == _lib.ERR_INVALID_ARG and "bad sizes" in _lib.last_error()


def test_nothing_to_do_for_no_sequences(lib):
    """A batch whose sequences have all left has no rows: no error, as for no rows of some sequences."""
    P = _at(1)

    def append(n, seqs):
        return lib.cllm_cuda_kv4_append(P, 256, P, P, P, 256, n, 2, None, 0, P, P, P, 4, 16, 2, 128, P, seqs, 1, None,
                                        None, None)

    def attention(n, seqs):
        return lib.cllm_cuda_kv4_attention(P, 512, P, n, 4, P, 4, 16, 2, 128, P, P, seqs, 2, 0.0, P, None, None)

    for call in (append, attention):
        assert call(0, 0) == 0 and call(0, 1) == 0
        for n, seqs in ((1, 0), (0, -1), (-1, 0)):
            assert call(n, seqs) == _lib.ERR_INVALID_ARG and "bad sizes" in _lib.last_error()
