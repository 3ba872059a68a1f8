"""Batches without a row, in every shape the targets may have."""
import pytest
import torch

from maester_amd import linear_token_logprobs, token_logprobs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead", [(0,), (0, 5), (5, 0), (2, 0, 3)])
@pytest.mark.parametrize("k", [0, 4])
@pytest.mark.parametrize("grad", [False, True])
def test_no_rows(gpu, lead, k, grad):
    x = torch.zeros(*lead, 16, device=gpu, requires_grad=grad)
    t = torch.zeros(lead, dtype=torch.long, device=gpu)
    out = token_logprobs(x, t, top_k=k)
    assert out.logp.shape == out.entropy.shape == lead
    assert (out.top_ids is None and out.top_logp is None) if k == 0 else out.top_ids.shape == out.top_logp.shape == (*lead, k)
    c = torch.ones(8, 16, device=gpu, requires_grad=grad)
    logp, entropy = linear_token_logprobs(x, c, t)
    assert logp.shape == entropy.shape == lead
    if grad:
        (out.logp.sum() + logp.sum() + entropy.sum()).backward()
        assert x.grad.shape == x.shape and bool((c.grad == 0).all())
