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
