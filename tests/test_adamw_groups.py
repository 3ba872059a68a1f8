"""Options of ``AdamW``'s parameter groups are checked when a group is added, whichever way."""
import pytest
import torch

from maester_amd import AdamW

NAN = float("nan")
WRONG = [dict(state_bits=16), dict(state_bits="8"), dict(lr=-1.0), dict(lr=NAN), dict(betas=(1.0, 0.9)), dict(betas=(0.9, NAN)), dict(eps=-1.0),
         dict(weight_decay=NAN), dict(seed=-1), dict(seed=1 << 32)]


@pytest.mark.parametrize("kw", WRONG)
def test_refused(kw):
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(ValueError):
        AdamW([p], **kw)
    with pytest.raises(ValueError):
        AdamW([{"params": [p]}, {"params": [q], **kw}])
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [q], **kw})
    assert len(opt.param_groups) == 1


def test_taken():
    p, q, r = (torch.nn.Parameter(torch.zeros(3)) for _ in range(3))
    opt = AdamW([{"params": [p], "state_bits": 8, "lr": 0.0}, {"params": [q], "betas": (0.0, 0.5)}], lr=torch.tensor(1e-3), seed=(1 << 32) - 1)
    opt.add_param_group({"params": [r], "weight_decay": 0.0})
    assert [g["state_bits"] for g in opt.param_groups] == [8, 32, 32] and opt.param_groups[2]["weight_decay"] == 0.0
