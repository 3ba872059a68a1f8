"""Calls on several streams at once and two captured graphs that share their memory: as one after the other, bit for bit."""
import pytest
import torch

from maester_amd import AdamW, linear_token_logprobs, token_logprobs

pytestmark = pytest.mark.gpu


def _work(seed, dev):
    """One step of everything on data of its own; (inputs to renew, the step)."""
    g = torch.Generator().manual_seed(seed)
    n, k, vocab = 70 + 30 * seed, 136, 5003
    e = torch.randn(n, k, generator=g).to(dev).bfloat16()
    w = torch.nn.Parameter((torch.randn(vocab, k, generator=g) / 4).to(dev).bfloat16())
    x = torch.randn(n, 20011, generator=g).to(dev).requires_grad_()
    t = torch.randint(0, vocab, (n,), generator=g).to(dev)
    t[::5] = -100
    opt = AdamW([w], lr=1e-2, state_bits=8, master_weights=True, max_grad_norm=1.0, seed=seed)

    def step():
        logp, entropy = linear_token_logprobs(e, w, t, softcap=20.0)
        rows = token_logprobs(x, t, top_k=7)
        dx, = torch.autograd.grad((rows.logp, rows.entropy), x, (logp.detach(), entropy.detach()))
        w.grad, = torch.autograd.grad(logp.sum() + 0.1 * entropy.sum(), w)
        opt.step()
        return [logp.detach(), entropy.detach(), rows.logp.detach(), rows.top_ids, dx, w.grad, w.detach(), opt.grad_norm]

    return e, step


def test_streams(gpu):
    want = []
    for seed in (1, 2, 3):
        _, step = _work(seed, gpu)
        want.append([[r.clone() for r in step()] for _ in range(4)])
    work = [_work(seed, gpu)[1] for seed in (1, 2, 3)]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = [[], [], []]
    for _ in range(4):
        for i, (step, stream) in enumerate(zip(work, streams)):
            with torch.cuda.stream(stream):
                got[i].append([r.clone() for r in step()])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for p, q in zip(a, b) for x, y in zip(p, q))


def test_two_graphs_of_one_pool(gpu):
    pairs = []
    for seed in (1, 2):
        (e, step), (f, eager) = _work(seed, gpu), _work(seed, gpu)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            eager()
        torch.cuda.current_stream().wait_stream(side)
        pairs.append((e, step, f, eager))
    torch.cuda.synchronize()
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for _, step, _, _ in pairs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = step()
        graphs.append((graph, out))
    for i in range(3):
        for (graph, out), (e, _, f, eager) in zip(graphs, pairs):
            e.mul_(0.9)
            f.copy_(e)
            graph.replay()
            torch.cuda.synchronize()
            want = eager()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i
