"""The 8-bit moments over long runs, and their codes against the definition in 32 bits."""

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


def definition(g, m, v, scales, t, seed, betas=(0.9, 0.999)):
    """The codes and scales after step t in 32 bits, operation by operation (of torch on the GPU, each of which rounds
    once); the first moment to the nearest code."""

    m, v = ((w.float().view(-1, BLOCK) * scales[k][:, None]).view(-1) for k, w in enumerate((m, v)))
    m = betas[0] * m + (1 - betas[0]) * g
    root = (betas[1] * v.square() + (1 - betas[1]) * g * g).sqrt()
    both = torch.stack([m, root]).view(2, -1, BLOCK)
    scales = both.abs().amax(dim=2) * (1 / 448)
    unit = (both * torch.where(scales > 0, 1 / scales, scales)[:, :, None]).view(2, -1)
    word = 0xFFFFFFFF
    h = (torch.arange(g.numel(), device=g.device) + t * 0x9E3779B9 + seed * 0x85EBCA6B) & word
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & word
    h = ((h ^ (h >> 15)) * 0x846CA68B) & word
    bits, u = ((h ^ (h >> 16)) & 0xFFFFF).int(), unit[1]
    normal = ((u.view(torch.int32) + bits) & ~0xFFFFF).view(torch.float32)
    small = torch.floor(u * 512 + bits.float() * 2.0**-20).clamp_min(1) / 512
    code = torch.where(u >= 2.0**-6, normal, torch.where(u > 0, small, u))
    return unit[0].clamp(-448, 448).to(torch.float8_e4m3fn), code.to(torch.float8_e4m3fn), scales


def test_codes_are_the_definitions(cuda_device):
    """Every code of the roots, those below 2**-6 units too (an eighth of the values here), and every code of a first
    moment that moves by half a step or more."""

    n, t, seed = 2**20, 5, 11
    g = torch.Generator().manual_seed(1)
    grad = torch.randn(n, generator=g) * 10.0 ** -(6 * torch.rand(n, generator=g))
    both = torch.stack([torch.randn(n, generator=g), torch.rand(n, generator=g) ** 8]).view(2, -1, BLOCK)
    scales = both.abs().amax(2) / 448
    m, v = (both / scales[:, :, None]).view(2, -1).to(torch.float8_e4m3fn).to(cuda_device)
    grad, s, m0, before = grad.to(cuda_device), scales.to(cuda_device), m.clone(), scales.to(cuda_device)
    want_m, want_v, want_s = definition(grad, m, v, s, t, seed)
    adamw_step([torch.zeros(n, device=cuda_device)], [grad], m, v, torch.tensor([t - 1, 0], device=cuda_device), scales=s,
               seed=seed)
    assert torch.equal(s, want_s)
    assert int((want_v.float() < 2.0**-6).sum()) > n // 16
    assert torch.equal(v.view(torch.uint8), want_v.view(torch.uint8))
    old = (m0.float().view(-1, BLOCK) * before[0][:, None] / want_s[0][:, None]).view(-1)
    new = 0.9 * old + 0.1 * (grad.view(-1, BLOCK) / want_s[0][:, None]).view(-1)
    far = ((new - old).abs() > 2.0**-9) | (new.abs() > 2.0**-5)
    same = m.view(torch.uint8) == want_m.view(torch.uint8)
    assert same[far].all() and int(far.sum()) > n // 2
    assert ((m.float() - want_m.float()).abs()[~far] <= 2.0**-9).all()


def test_codes_of_small_roots_are_the_definitions(cuda_device):
    """10**8 roots below 2**-6 units: a rounding before the random bits come in, not after, shows in one of ten million."""

    n, t, seed = 2**27, 3, 2
    g = torch.Generator(cuda_device).manual_seed(2)
    grad = torch.rand(n, device=cuda_device, generator=g) * (2.0**-6 * 31)
    grad[::BLOCK] = 448.0
    v = torch.full((n,), 2.0**-9, device=cuda_device)
    v[::BLOCK] = 448.0
    v, s = v.to(torch.float8_e4m3fn), torch.ones(2, n // BLOCK, device=cuda_device)
    m = torch.zeros_like(v)
    _, want, want_s = definition(grad, m, v, s, t, seed)
    adamw_step([torch.zeros(n, device=cuda_device)], [grad], m, v, torch.tensor([t - 1, 0], device=cuda_device), scales=s,
               seed=seed)
    assert torch.equal(s, want_s)
    assert float((want.float() <= 2.0**-6).float().mean()) > 0.99
    assert torch.equal(v.view(torch.uint8), want.view(torch.uint8))
