"""Forward-mode derivatives: no entry point of the per-token objectives or of the optimizer step drops a tangent silently."""
import pytest
import torch
from torch.autograd import forward_ad

from maester_amd import adamw_step, global_grad_norm, linear_token_logprobs, token_logprobs

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(device, grad):
    x, c = torch.randn(6, 16, device=device), torch.randn(16, 16, device=device)
    t = torch.zeros(6, dtype=torch.long, device=device)
    step = torch.zeros((), dtype=torch.int64, device=device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.clone().requires_grad_(grad), torch.ones_like(x))
        weight = forward_ad.make_dual(c, torch.ones_like(c))
        for call in (lambda: token_logprobs(dual, t), lambda: token_logprobs(dual.view(2, 3, 16), t.view(2, 3), top_k=2),
                     lambda: linear_token_logprobs(dual, c, t), lambda: linear_token_logprobs(x, weight, t),
                     lambda: global_grad_norm([x, dual]),
                     lambda: adamw_step([x], [dual], [torch.zeros_like(x)], [torch.zeros_like(x)], step)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            token_logprobs(dual, t)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda v: token_logprobs(v, t).logp, (x,), (torch.ones_like(x),))


@pytest.mark.gpu
def test_plain_tensors_inside_a_level(gpu):
    x, t = torch.randn(6, 16, device=gpu), torch.zeros(6, dtype=torch.long, device=gpu)
    want = token_logprobs(x, t).logp
    with forward_ad.dual_level():
        assert torch.equal(token_logprobs(x, t).logp, want)
        assert torch.equal(linear_token_logprobs(x, x, t)[0], linear_token_logprobs(x, x, t)[0])
