"""What an AdamWCuda takes as saved state, and its copies."""

import copy
import io

import pytest
import torch

from triton_pesq_b200 import AdamWCuda


def parameters(device="cpu", dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(device, dtype)) for s in ((5, 7), (300,))]


def saved(bits, dtype=torch.float32):
    """A state dict of two parameters as an optimiser of `bits` bits leaves it."""

    kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
    state = {}
    for i, (size, units) in enumerate((((5, 7), 1), ((300,), 2))):
        state[i] = {"step": torch.tensor([3, 0]), "moment1": torch.full((256 * units,), 2.0).to(kind),
                    "moment2": torch.full((256 * units,), 3.0).to(kind)}
        if bits == 8:
            state[i]["scales"] = torch.full((2, units), 1e-3)
        if dtype != torch.float32:
            state[i]["master"] = torch.zeros(size)
    groups = AdamWCuda(parameters(dtype=dtype), state_bits=bits).state_dict()["param_groups"]
    return {"state": state, "param_groups": groups}


@pytest.mark.parametrize("bits", [8, 32])
def test_state_of_the_other_width_is_refused(bits):
    opt = AdamWCuda(parameters(), state_bits=40 - bits, lr=0.5)
    opt.load_state_dict({**saved(40 - bits), "param_groups": opt.state_dict()["param_groups"]})
    before = opt.state_dict()
    with pytest.raises(ValueError, match="bits"):
        opt.load_state_dict(saved(bits))
    after = opt.state_dict()  # as it was
    assert after["param_groups"] == before["param_groups"] and after["state"].keys() == before["state"].keys()
    for i, s in before["state"].items():
        assert all(torch.equal(v.view(torch.uint8), after["state"][i][k].view(torch.uint8)) for k, v in s.items())


def test_state_of_another_kind_is_refused():
    opt = AdamWCuda(parameters())
    theirs = parameters()
    other = torch.optim.AdamW(theirs)
    for p in theirs:
        p.grad = torch.ones_like(p)
    other.step()
    with pytest.raises(ValueError):
        opt.load_state_dict(other.state_dict())
    short = saved(32)
    short["state"][1]["moment1"] = short["state"][1]["moment1"][:256]
    with pytest.raises(ValueError):
        opt.load_state_dict(short)
    for lost in ("step", "moment2"):
        part = saved(32)
        del part["state"][0][lost]
        with pytest.raises(ValueError):
            opt.load_state_dict(part)
    with pytest.raises(ValueError):  # 16-bit parameters' masters
        opt.load_state_dict(saved(32, torch.bfloat16))
    with pytest.raises(ValueError):
        AdamWCuda(parameters(dtype=torch.bfloat16)).load_state_dict(saved(32))
    groups = saved(32)
    groups["param_groups"][0]["params"] = [0]
    with pytest.raises(ValueError):
        opt.load_state_dict(groups)
    assert not opt.state
    opt.load_state_dict(saved(32))
    assert len(opt.state) == 2


def test_copies_keep_their_options():
    opt = AdamWCuda(parameters(), state_bits=8, seed=5, lr=0.25)
    opt.load_state_dict({**saved(8), "param_groups": opt.state_dict()["param_groups"]})
    buffer = io.BytesIO()
    torch.save(opt, buffer)
    buffer.seek(0)
    for other in (copy.deepcopy(opt), torch.load(buffer, weights_only=False)):
        assert other.state_bits == 8 and other.seed == 5 and other.param_groups[0]["lr"] == 0.25
        assert len(other.state) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_copies_step_on_as_the_original(cuda_device, bits, dtype):
    def advance(opt, seed):
        g = torch.Generator(cuda_device).manual_seed(seed)
        for group in opt.param_groups:
            for p in group["params"]:
                p.grad = torch.randn(p.shape, device=cuda_device, generator=g).to(p.dtype)
        opt.step()

    opt = AdamWCuda(parameters(cuda_device, dtype), lr=1e-2, state_bits=bits, seed=3)
    advance(opt, 1)
    buffer = io.BytesIO()
    torch.save(opt, buffer)
    buffer.seek(0)
    others = [copy.deepcopy(opt), torch.load(buffer, weights_only=False)]
    for seed in (2, 3):
        for o in (opt, *others):
            advance(o, seed)
    for o in others:
        for p, q in zip(opt.param_groups[0]["params"], o.param_groups[0]["params"]):
            assert p is not q and torch.equal(p, q)
            for k, t in opt.state[p].items():
                assert torch.equal(t.contiguous().view(torch.uint8), o.state[q][k].contiguous().view(torch.uint8)), k
