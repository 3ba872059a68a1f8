"""Sharded and other wrapped tensors have no memory of their own: they are refused by name, before anything is allocated."""
import pytest
import torch
import torch.distributed as dist

from maester_amd import AdamW, adamw_step, global_grad_norm, linear_token_logprobs, token_logprobs


@pytest.fixture
def sharded():
    from torch.distributed.device_mesh import DeviceMesh
    from torch.distributed.tensor import Shard, distribute_tensor
    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        mesh = DeviceMesh("cpu", [0])
        yield lambda *shape: distribute_tensor(torch.ones(*shape), mesh, [Shard(0)])
    finally:
        dist.destroy_process_group()


def test_optimizer(sharded):
    p, q = torch.nn.Parameter(torch.ones(8)), torch.nn.Parameter(sharded(8))
    for params in ([q], [p, q], [{"params": [p]}, {"params": [q]}]):
        with pytest.raises(TypeError, match="DTensor"):
            AdamW(params)
    opt = AdamW([p])
    with pytest.raises(TypeError, match="DTensor"):
        opt.add_param_group({"params": [q]})
    p.grad = torch.ones(8)
    opt.param_groups[0]["params"][0] = q                     # swapped behind the optimizer's back
    q.grad = sharded(8)
    with pytest.raises(TypeError, match="DTensor"):
        opt.step()
    assert not opt.state


def test_functions(sharded):
    x, d = torch.ones(4, 16), sharded(4, 16)
    t, step = torch.zeros(4, dtype=torch.long), torch.zeros((), dtype=torch.long)
    for call in (lambda: adamw_step([d], [x], [x], [x], step), lambda: adamw_step([x, d], [x, x], [x, x], [x, x], step),
                 lambda: adamw_step([x], [d], [x], [x], step), lambda: adamw_step([x], [x], [x], [d], step),
                 lambda: adamw_step([x.bfloat16()], [x], [x.clone()], [x.clone()], step, masters=[d]), lambda: global_grad_norm([x, d]),
                 lambda: token_logprobs(d, t), lambda: linear_token_logprobs(d, x, t), lambda: linear_token_logprobs(x, d, t)):
        with pytest.raises(TypeError, match="DTensor"):
            call()


def test_what_step_cannot_take_is_refused_before_the_states_are_made():
    p = torch.nn.Parameter(torch.ones(8, 4).t())
    p.grad = torch.ones(4, 8)
    opt = AdamW([p], state_bits=8)
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    half = torch.nn.Parameter(torch.ones(8).half())
    half.grad = torch.ones(8).half()
    with pytest.raises(TypeError, match="float16"):
        AdamW([half]).step()
    cpu = torch.nn.Parameter(torch.ones(8))
    cpu.grad = torch.ones(8)
    third = AdamW([cpu])
    with pytest.raises(RuntimeError, match="MI355X"):
        third.step()
    assert not opt.state and not third.state
