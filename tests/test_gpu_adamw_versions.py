"""What an AdamW step writes counts as modified in place: a backward through what a graph saved before it raises."""
import pytest
import torch

from maester_amd import AdamW, Blocks8, adamw_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("state_bits", [32, 8])
def test_a_graph_from_before_the_step_raises(gpu, state_bits):
    w = torch.nn.Parameter(torch.randn(64, 32, device=gpu))
    x = torch.randn(8, 32, device=gpu, requires_grad=True)
    opt = AdamW([w], state_bits=state_bits)
    y = x @ w.t()
    (y.square().mean()).backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("eight", [False, True])
def test_versions_of_everything_written(gpu, eight):
    def state(p):
        return Blocks8.zeros_like(p) if eight else torch.zeros_like(p, dtype=torch.float32)

    params = [torch.randn(300, device=gpu).bfloat16(), torch.randn(0, device=gpu).bfloat16(), torch.randn(7, 5, device=gpu)]
    grads = [torch.randn_like(p) for p in params]
    masters = [params[0].float(), None, None]
    m, v = [state(p) for p in params], [state(p) for p in params]
    step = torch.zeros((), dtype=torch.int64, device=gpu)
    written = [*params, masters[0], step, *(t for s in (*m, *v) for t in (s if eight else (s,)))]
    before, read = [t._version for t in written], [g._version for g in grads]
    adamw_step(params, grads, m, v, step, masters=masters, max_grad_norm=1.0)
    assert all(t._version > n for t, n in zip(written, before))
    assert [g._version for g in grads] == read


def test_inference_tensors(gpu):
    # they count no versions, and a step over them needs none
    with torch.inference_mode():
        p, g, m, v = (torch.ones(100, device=gpu) for _ in range(4))
        step = torch.zeros((), dtype=torch.int64, device=gpu)
        adamw_step([p], [g], [m], [v], step)
        assert int(step) == 1 and float(p[0]) < 1
    with torch.inference_mode():
        q = torch.nn.Parameter(torch.ones(100, device=gpu))
        m, v = torch.zeros(100, device=gpu), torch.zeros(100, device=gpu)
    plain = torch.ones(100, device=gpu)
    adamw_step([q.detach(), plain], [g, g], [m, torch.zeros(100, device=gpu)], [v, torch.zeros(100, device=gpu)], step)
    assert plain._version > 0
