"""Resets against values that are not numbers: what lies before a reset, or
behind one for the gradients, does not reach the other side."""

import pytest
import torch

from triton_pesq_b200 import gated_scan

pytestmark = pytest.mark.gpu

# whole rows; rows in one CTA; cut in both directions, by boxes and by lanes
SHAPES = [(600, 20, 64), (2, 200, 64), (2, 200, 33), (2, 3000, 64), (2, 3000, 33)]


def call(dev, dy, dlast, reset, reverse):
    leaves = [t.detach().requires_grad_(True) for t in dev]
    y, last = gated_scan(*leaves, reset=reset, reverse=reverse)
    return (y, last, *torch.autograd.grad((y, last), leaves, (dy, dlast)))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("late", [False, True])
def test_what_a_reset_parts(cuda_device, shape, dtype, reverse, which, late):
    """Two utterances in a row, one of them with a NaN in x or in a gate: outputs and gradients of the other are
    those without it, bit for bit."""

    batch, steps, width = shape
    g = torch.Generator(cuda_device).manual_seed(steps + width)
    dev = [torch.randn(*shape, device=cuda_device, generator=g).to(dtype) for _ in range(3)]
    dev += [torch.linspace(-5, 1, width, device=cuda_device), torch.randn(batch, width, device=cuda_device, generator=g)]
    dy = torch.randn(*shape, device=cuda_device, generator=g).to(dtype)
    dlast = torch.randn(batch, width, device=cuda_device, generator=g)
    cut = steps // 2
    order = list(range(steps - 1, -1, -1)) if reverse else list(range(steps))
    reset = torch.zeros(batch, steps, dtype=torch.bool, device=cuda_device)
    reset[:, order[cut]] = True
    clean = call(dev, dy, dlast, reset, reverse)
    dev[which] = dev[which].clone()
    dev[which][:, order[cut + 2 if late else cut - 2]] = float("nan")
    got = call(dev, dy, dlast, reset, reverse)
    free = order[:cut] if late else order[cut:]
    for a, b in zip((got[0], *got[2:5]), (clean[0], *clean[2:5])):
        assert torch.equal(a[:, free], b[:, free])
    assert torch.equal(got[6], clean[6]) if late else torch.equal(got[1], clean[1])
    assert torch.isnan(got[0][:, order[cut + 2 if late else cut - 2]]).all()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("reverse", [False, True])
def test_a_reset_does_not_look_at_its_decay_gate(cuda_device, shape, reverse):
    """a = 0 there whatever the gate holds: the gate's gradient is zero, and nothing else changes."""

    batch, steps, width = shape
    g = torch.Generator(cuda_device).manual_seed(1)
    dev = [torch.randn(*shape, device=cuda_device, generator=g) for _ in range(3)]
    dev += [torch.linspace(-5, 1, width, device=cuda_device), torch.randn(batch, width, device=cuda_device, generator=g)]
    dy, dlast = torch.randn(*shape, device=cuda_device, generator=g), torch.ones(batch, width, device=cuda_device)
    reset = torch.rand(batch, steps, device=cuda_device, generator=g) < 0.1
    clean = call(dev, dy, dlast, reset, reverse)
    dev[2] = torch.where(reset[:, :, None], float("nan"), dev[2])
    for a, b in zip(call(dev, dy, dlast, reset, reverse), clean):
        assert torch.equal(a, b)
    assert not clean[4][reset].any()
