"""What ``MuonCuda.load_state_dict`` takes and refuses (no GPU: no step is made)."""

import copy

import pytest
import torch

from triton_pesq_b200 import AdamWCuda, MuonCuda


def snapshot(opt):
    return copy.deepcopy([{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups]), copy.deepcopy(dict(opt.state))


@pytest.mark.parametrize("other", [torch.optim.SGD, torch.optim.AdamW, AdamWCuda])
def test_other_optimisers_are_refused_before_their_first_step_too(other):
    """Without a state of any parameter, what another optimiser saves differs in its groups alone."""

    params = [torch.nn.Parameter(torch.ones(4, 4))]
    opt = MuonCuda(params, lr=0.5)
    before = snapshot(opt)
    with pytest.raises(ValueError, match="missing"):
        opt.load_state_dict(other(params).state_dict())
    assert snapshot(opt) == before


def test_groups_come_back_with_what_schedulers_add():
    params = [torch.nn.Parameter(torch.ones(4, 4)), torch.nn.Parameter(torch.ones(3, 4))]
    opt = MuonCuda([{"params": params[:1], "lr": 0.5}, {"params": params[1:], "steps": 3}])
    torch.optim.lr_scheduler.LambdaLR(opt, lambda step: 1.0)
    new = MuonCuda([{"params": params[:1]}, {"params": params[1:]}])
    new.load_state_dict(opt.state_dict())
    assert snapshot(new) == snapshot(opt) and new.param_groups[0]["initial_lr"] == 0.5
    with pytest.raises(ValueError):
        new.load_state_dict(MuonCuda(params).state_dict())


def test_a_state_is_taken_as_often_as_it_is_given():
    """By an optimiser that has loaded one before, and by copies of one, whose defaults the base class adds to."""

    params = [torch.nn.Parameter(torch.ones(4, 4))]
    opt, fresh = MuonCuda(params, lr=0.5), MuonCuda(params).state_dict()
    for _ in range(2):
        opt.load_state_dict(fresh)
        twin = copy.deepcopy(opt)
        twin.load_state_dict(fresh)
    assert twin.param_groups[0]["lr"] == opt.param_groups[0]["lr"] == 1e-3
