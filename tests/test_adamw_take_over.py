"""States of torch's optimizers taken over by ``AdamW``: what it cannot continue is refused before anything changes."""
import copy
import warnings

import pytest
import torch

from maester_amd import AdamW

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _trained(kind=torch.optim.AdamW, steps=(3, 3), device="cpu", **kw):
    """A state of ``kind`` over two parameters after so many steps of each."""
    params = [torch.nn.Parameter(torch.full((4,), 1.0 + i, device=device)) for i in range(2)]
    opt = kind(params, **kw)
    for n in range(max(steps)):
        for p, last in zip(params, steps):
            p.grad = torch.ones_like(p) if n < last else None
        opt.step()
    return params, opt.state_dict()


def _ours(device="cpu", **kw):
    params = [torch.nn.Parameter(torch.full((4,), 1.0 + i, device=device)) for i in range(2)]
    return params, AdamW(params, **{"lr": 0.125, **kw})


@pytest.mark.parametrize("kind,kw,text", [(torch.optim.AdamW, dict(maximize=True), "maximize"), (torch.optim.AdamW, dict(amsgrad=True), "amsgrad"),
                                          (torch.optim.Adam, dict(weight_decay=0.1), "decoupled"), (torch.optim.SGD, dict(momentum=0.9), "exp_avg"),
                                          (torch.optim.Adamax, {}, "exp_avg_sq"), (torch.optim.RMSprop, {}, "exp_avg"),
                                          (torch.optim.NAdam, {}, "not a state of"), (torch.optim.RAdam, {}, "not a state of")])
def test_refused_before_anything_changes(kind, kw, text):
    _, state = _trained(kind, lr=0.5, **kw)
    params, ours = _ours()
    before = copy.deepcopy(ours.state_dict())
    with pytest.raises(ValueError, match=text):
        ours.load_state_dict(state)
    assert ours.state_dict() == before and not ours.state


def test_taken_over():
    for kind, kw in ((torch.optim.AdamW, {}), (torch.optim.Adam, dict(weight_decay=0.0))):
        params, state = _trained(kind, lr=0.5, **kw)
        _, ours = _ours()
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            ours.load_state_dict(state)
        group = ours.param_groups[0]
        assert int(group["step"]) == 3 and group["lr"] == 0.5 and group["state_bits"] == 32
        for p, i in zip(group["params"], (0, 1)):
            assert torch.equal(ours.state[p]["exp_avg"], state["state"][i]["exp_avg"])


def test_counters_that_differ_are_said():
    _, state = _trained(steps=(5, 2))
    _, ours = _ours()
    with pytest.warns(UserWarning, match="bias correction"):
        ours.load_state_dict(state)
    assert int(ours.param_groups[0]["step"]) == 5


@pytest.mark.parametrize("device", DEVICES)
def test_a_rate_on_the_host_moves_to_the_parameters(device):
    # torch takes a rate as a tensor on the host; map_location="cpu" brings one of ours there too
    for state in (_trained(device=device, lr=torch.tensor(0.25), foreach=False)[1], None):
        params, ours = _ours(device, lr=torch.tensor(0.25, device=device))
        if state is None:
            state = copy.deepcopy(ours.state_dict())
            state["param_groups"][0]["lr"] = torch.tensor(0.25, dtype=torch.float64)
            state["param_groups"][0]["step"] = torch.tensor(3)
        ours.load_state_dict(state)
        group = ours.param_groups[0]
        assert group["lr"].device == params[0].device and group["lr"].dtype == torch.float32 and float(group["lr"]) == 0.25
        assert group["step"].device == params[0].device and group["step"].dtype == torch.int64 and int(group["step"]) == 3
        if device == "cuda":
            for p in params:
                p.grad = torch.ones_like(p)
            ours.step()
            assert int(group["step"]) == 4 and bool((params[0] < 1).all())


@pytest.mark.parametrize("bits", [16, 0, None])
def test_a_state_of_ours_with_unknown_bits(bits):
    _, ours = _ours()
    state = copy.deepcopy(ours.state_dict())
    state["param_groups"][0]["state_bits"] = bits
    with pytest.raises(ValueError, match="state_bits"):
        ours.load_state_dict(state)


def test_a_group_without_parameters():
    p = torch.nn.Parameter(torch.ones(4))
    make = lambda: AdamW([{"params": [p]}, {"params": [], "lr": torch.tensor(0.5)}])  # noqa: E731
    state = copy.deepcopy(make().state_dict())
    ours = make()
    ours.load_state_dict(state)
    assert ours.param_groups[1]["params"] == [] and float(ours.param_groups[1]["lr"]) == 0.5
