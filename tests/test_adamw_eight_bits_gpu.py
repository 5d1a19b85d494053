"""The 8-bit moments over long runs."""

import pytest
import torch

import train_reference as R
from triton_pesq_b200 import adamw_step

pytestmark = pytest.mark.gpu

BLOCK = 256


def eight_bit_state(n, device):
    m, v = (torch.zeros(n, device=device, dtype=torch.float8_e4m3fn) for _ in range(2))
    return m, v, torch.zeros(2, n // BLOCK, device=device), torch.zeros(2, dtype=torch.int64, device=device)


@pytest.mark.parametrize("beta1, steps", [(0.9, 20000), (0.95, 6000), (0.99, 6000)])
@pytest.mark.parametrize("share", [1.0, 1e-2, 1e-4])
def test_first_moment_decays_where_the_gradient_stops(cuda_device, beta1, steps, share):
    """64 of 256 values, whose gradients are ``share`` of the others', get none
    after 50 steps.  By the definition they move on by ten learning rates at most and
    stay.  A code is within a step of its value, and near zero a step is as large as the
    value: three times the definition's way is allowed, on average; and nothing is left at
    the end, since after k steps a code has survived with a probability of beta1**k."""

    stop, lr = 50, 1e-3
    g = torch.Generator(cuda_device).manual_seed(0)
    p = [torch.zeros(BLOCK, device=cuda_device)]
    m, v, scales, step = eight_bit_state(BLOCK, cuda_device)
    grads = 1e-2 * torch.randn(steps, BLOCK, device=cuda_device, generator=g)
    grads[:, :64] *= share
    grads[stop:, :64] = 0
    for t in range(steps):
        if t == stop:
            at = p[0][:64].clone()
        adamw_step(p, [grads[t]], m, v, step, scales=scales, lr=lr, betas=(beta1, 0.999), weight_decay=0.0, seed=7)
    wide = [torch.zeros(64, dtype=torch.float64) for _ in range(3)]
    few = grads[:stop + 1500, :64].cpu().double()  # (beta1**1500 < 1e-6)
    for t in range(stop + 1500):
        if t == stop:
            there = wide[0].clone()
        wide = list(R.adamw(wide[0], few[t], wide[1], wide[2], t + 1, lr, (beta1, 0.999), decay=0.0))
    moved, want = (p[0][:64] - at).abs().mean(), (wide[0] - there).abs().mean()
    assert float(moved) <= 3 * float(want)
    assert not m[:64].float().any()
    assert m[64:].float().any() and torch.isfinite(p[0]).all()


def test_a_steady_small_gradient_is_followed(cuda_device):
    """Values whose moment is a few of the smallest steps and whose gradient is a fifth of one: the moment
    goes to the gradient on average.  A code there is 0 or 1 steps, in mean 0.2, of standard deviation
    0.4; 4096 values 100 times (of which each tenth is new) leave 0.002 and ten times that is allowed."""

    n = 16 * BLOCK
    m, v, scales, step = eight_bit_state(n, cuda_device)
    code = torch.full((n,), 5 * 2.0**-9, device=cuda_device)
    code[::BLOCK] = 448.0
    m.copy_(code), v.copy_(torch.full_like(code, 448.0))
    scales.fill_(1.0)
    p, g = [torch.zeros(n, device=cuda_device)], torch.full((n,), 0.2 * 2.0**-9, device=cuda_device)
    g[::BLOCK] = 448.0
    mean = 0.0
    for t in range(300):
        adamw_step(p, [g], m, v, step, scales=scales, seed=3)
        if t >= 200:
            units = m.float().view(-1, BLOCK)[:, 1:] * scales[0][:, None]
            mean += float(units.mean()) * 512 / 100
    assert abs(mean - 0.2) <= 0.02
