"""Rows that do not count give the classifier no gradient whatever their hidden states hold: padding may be NaN."""
import pytest
import torch

from maester_amd import linear_token_logprobs

pytestmark = pytest.mark.gpu


# few bf16 rows (two parts of the logits' gradient), one block, several blocks, an odd last block; rows in place and strided
@pytest.mark.parametrize("n,chunk", [(1, None), (5, None), (40, None), (64, None), (65, None), (300, None), (300, 128), (130, 33)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("strided", [False, True])
def test_padding_rows(gpu, n, chunk, dtype, bad, strided):
    k, vocab = 72, 1003
    g = torch.Generator().manual_seed(n)
    e = torch.randn(n, k, generator=g).to(dtype)
    c = (torch.randn(vocab, k, generator=g) / 4).to(dtype).to(gpu)
    t = torch.randint(0, vocab, (n,), generator=g)
    t[::3], t[1::7] = -100, vocab                                     # ignored, and outside the vocabulary
    dead = (t < 0) | (t >= vocab)
    w = torch.randn(n, generator=g).to(gpu)
    out = []
    for value in (0.0, bad):
        x = e.clone()
        x[dead] = value
        x = x.to(gpu)
        if strided:
            x = torch.full((n, k + 24), bad, dtype=dtype, device=gpu)[:, 8:8 + k].copy_(x)
        x.requires_grad_()
        leaf = c.clone().requires_grad_()
        logp, entropy = linear_token_logprobs(x, leaf, t.to(gpu), chunk_rows=chunk, filter_ignored=False)
        out.append((logp, entropy, *torch.autograd.grad((logp, entropy), (x, leaf), (w, w))))
    for a, b in zip(*out):
        assert bool(torch.isfinite(b).all()) and torch.equal(a, b)
    assert bool((out[1][2][dead.to(gpu)] == 0).all())


def test_nothing_counts(gpu):
    e = torch.full((70, 64), float("nan"), device=gpu, dtype=torch.bfloat16, requires_grad=True)
    c = torch.randn(300, 64, device=gpu).bfloat16().requires_grad_()
    logp, entropy = linear_token_logprobs(e, c, torch.full((70,), -100, device=gpu))
    (logp.sum() + entropy.sum()).backward()
    assert bool((e.grad == 0).all()) and bool((c.grad == 0).all())


def test_in_a_graph(gpu):
    n, k, vocab = 100, 64, 515
    e, c = torch.randn(n, k, device=gpu).requires_grad_(), torch.randn(vocab, k, device=gpu).requires_grad_()
    t = torch.randint(0, vocab, (n,), device=gpu)

    def step():
        out = linear_token_logprobs(e, c, t)
        return torch.autograd.grad(out[0].sum() + out[1].sum(), (e, c))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            e.copy_(torch.randn(n, k, device=gpu))
            e[i::4] = float("nan")
        t.random_(0, vocab)
        t[i::4] = -100
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(got, want)), i
