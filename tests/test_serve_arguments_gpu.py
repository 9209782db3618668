"""Arguments of the serving operators' front ends at their borders."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_scores_of_an_expanded_row(cuda, lib):
    from cllm_inference_b200.scoring import token_scores

    x = torch.randn(1, 5000, device="cuda") * 3
    tokens = torch.tensor([4, 0, 4999, 17, 4], dtype=torch.int32, device="cuda")
    got, want = token_scores(x.expand(5, -1), tokens, 7), token_scores(x.expand(5, -1).contiguous(), tokens, 7)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_cache_without_sequences_starts_anew(cuda, lib):
    """After the last sequence has left, the pool is free for others."""
    from cllm_inference_b200 import _lib
    from cllm_inference_b200.kv4 import KV4Cache

    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = KV4Cache.empty(1, 6, 16, 1, 64, 2, 3).fork(ints(-1, -1), ints(40, 33))
    none = cache.fork(ints(), ints())
    assert none.n_seqs == 0
    assert none.append(0, torch.zeros(0, 64, device="cuda"), torch.zeros(0, 64, device="cuda"), ints(), ints()) is None
    assert none.attention(0, torch.zeros(0, 64, device="cuda")).shape == (0, 64)
    assert none.fork(ints(), ints()).n_seqs == 0
    packed, live = none.compact()
    assert int(live[0]) == 0 and packed.n_seqs == 0
    new = packed.fork(ints(-1, 0, -1), ints(40, 5, 16))  # there is no sequence 0 to continue
    assert new.lens.tolist() == [40, -1, 16]
    assert new.table.tolist() == [[0, 1, 2], [-1, -1, -1], [3, -1, -1]]
    _lib.check(lib.cllm_cuda_check_device_status())
