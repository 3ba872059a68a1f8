"""The outputs of both forms of the log-probabilities are tensors of their own: editing one in place reaches neither the
other nor what the backward needs."""
import pytest
import torch

from maester_amd import linear_logprobs, linear_token_logprobs, token_logprobs

pytestmark = pytest.mark.gpu
ROWS, WIDTH, VOCAB = 300, 64, 515


def _logits_form(lead, ignored, dev):
    x = torch.randn(*lead, VOCAB, device=dev).requires_grad_()
    t = torch.randint(0, VOCAB, lead, device=dev)
    if ignored:
        t.view(-1)[::3] = -100
    return (x,), lambda: token_logprobs(x, t, softcap=9.0)[:2]


def _linear_form(lead, ignored, dev):
    e, c = torch.randn(*lead, WIDTH, device=dev).requires_grad_(), torch.randn(VOCAB, WIDTH, device=dev).requires_grad_()
    t = torch.randint(0, VOCAB, lead, device=dev)
    if ignored:
        t.view(-1)[::3] = -100
    return (e, c), lambda: linear_token_logprobs(e, c, t)


EDITS = {"mul": lambda t: t.mul_(0.5), "fill": lambda t: t.masked_fill_(torch.arange(t.numel(), device=t.device).view(t.shape) % 2 == 0, 0.0)}
PLAIN = {"mul": lambda t: t * 0.5, "fill": lambda t: t.masked_fill(torch.arange(t.numel(), device=t.device).view(t.shape) % 2 == 0, 0.0)}


@pytest.mark.parametrize("form", [_logits_form, _linear_form])
@pytest.mark.parametrize("lead", [(ROWS,), (10, ROWS // 10), (5, 6)])
@pytest.mark.parametrize("ignored", [False, True])
def test_outputs_edited_in_place(gpu, form, lead, ignored, monkeypatch):
    monkeypatch.setitem(linear_logprobs._FILTER_WORK, torch.float32, 0)      # ignored rows are dropped from 257 rows on
    leaves, call = form(lead, ignored, gpu)
    for which in (0, 1):
        for name, edit in EDITS.items():
            out = list(call())
            out[which] = PLAIN[name](out[which])
            want = torch.autograd.grad(out[0].sum() + 0.3 * out[1].sum(), leaves)
            out = call()
            other = out[1 - which].detach().clone()
            edit(out[which])
            assert torch.equal(out[1 - which], other)
            got = torch.autograd.grad(out[0].sum() + 0.3 * out[1].sum(), leaves)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (which, name)


@pytest.mark.parametrize("form", [_logits_form, _linear_form])
@pytest.mark.parametrize("lead", [(ROWS,), (5, 6)])
def test_detached_outputs_edited(gpu, form, lead):
    leaves, call = form(lead, True, gpu)
    out = call()
    want = torch.autograd.grad(out[0].sum() + out[1].sum(), leaves)
    for which in (0, 1):
        out = call()
        out[which].detach().clamp_(max=-1.0)
        got = torch.autograd.grad(out[0].sum() + out[1].sum(), leaves)       # (the sums' gradients are ones)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), which


def test_no_memory_is_shared(gpu):
    for form in (_logits_form, _linear_form):
        _, call = form((7,), False, gpu)
        with torch.no_grad():
            a, b = call()
        assert a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr() and a._base is None and b._base is None
