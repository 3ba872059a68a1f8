"""Rows of logits that share memory: a broadcast row, overlapping windows."""
import numpy as np
import pytest
import torch

from maester_amd import token_logprobs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(5, 37), (600, 5003)])
def test_a_broadcast_row(gpu, dtype, rows, vocab):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(vocab, generator=g).to(gpu, dtype)
    t = torch.randint(0, vocab, (rows,), generator=g).to(gpu)
    t[2] = -100
    w = torch.randn(rows, generator=g).to(gpu)
    out = []
    for make in (lambda l: l.expand(rows, vocab), lambda l: l.repeat(rows, 1)):
        leaf = x.clone().requires_grad_()
        got = token_logprobs(make(leaf), t, top_k=3)
        grad, = torch.autograd.grad((got.logp, got.entropy), leaf, (w, w))
        with torch.no_grad():
            assert torch.equal(token_logprobs(make(leaf), t).logp, got.logp)
        out.append((*got, grad))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_overlapping_windows(gpu):
    flat = torch.randn(40, device=gpu)
    windows = flat.unfold(0, 16, 3)
    t = torch.arange(len(windows), device=gpu)
    got, want = token_logprobs(windows, t, top_k=2), token_logprobs(windows.clone(memory_format=torch.contiguous_format), t, top_k=2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert np.allclose(got.logp.cpu().numpy(), torch.log_softmax(windows.double(), 1).gather(1, t[:, None])[:, 0].cpu().numpy(), atol=1e-5)
