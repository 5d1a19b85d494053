"""What the linear attention gives in 32 bits is as exact as arithmetic of 32 bits, by the norm of the difference from 64 bits.

Bounds.  The states' own roundings, which decay with them, are some ten of random sign: sqrt(10) * 2^-23.  A decay's gradient
beside 16 bits sums products over up to 128 channels, whose instruction cuts off what its accumulator does not hold: at most
24 times (eight steps of three terms, 16 of two) half of 2^-24 of the sum on average.  Of float32 a product leaves out the product of two lower
terms, 2^-22 at most, and its sums are rounded: with the states' roundings 2^-22 more."""

import pytest
import torch

from test_linear_attention_gpu import definition, make, on
from triton_pesq_b200 import linear_attention

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
STATES = 10**0.5 * 2.0**-23


def both(shape, dtype, device, seed, reset=False, decays=0.2):
    """(names, mine, in 64 bits) of all outputs and gradients, with a decay for each step."""

    (q, k, v, decay, state), dy, dlast, kw = make(*shape, dtype, gated=True, reset=reset, seed=seed)
    tensors, kw = [t.to(device) for t in (q, k, v, decays * decay, state)], on(device, kw)
    dy, dlast = dy.to(device), dlast.to(device)
    mine, wide = [t.clone().requires_grad_(True) for t in tensors], [t.double().requires_grad_(True) for t in tensors]
    out, want = linear_attention(*mine, **kw), definition(*wide, **kw)
    got = [*out, *torch.autograd.grad(out, mine, (dy, dlast))]
    ref = [*want, *torch.autograd.grad(want, wide, (dy.double(), dlast.double()))]
    return ("y", "last", "dq", "dk", "dv", "d log_decay", "d state"), [t.detach() for t in got], [t.detach() for t in ref]


def far(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", [(3, 1, 6, 18, 9), (1, 2, 12, 16, 44), (10, 8, 3, 12, 117), (3, 300, 4, 64, 64), (2, 150, 4, 32, 24),
                                   (2, 300, 4, 64, 100), (2, 300, 4, 100, 64), (4, 62, 14, 72, 11), (2, 300, 4, 128, 128),
                                   (8, 500, 12, 64, 64), (1, 888, 13, 115, 110)])
def test_gradients_of_decays_beside_16_bits(cuda_device, dtype, shape):
    names, got, want = both(shape, dtype, cuda_device, 31)
    for name, a, e in zip(names, got, want):
        if name == "d log_decay":
            assert far(a, e) <= STATES + 24 * 2.0**-25, far(a, e)
        elif a.dtype == F32:
            assert far(a, e) <= STATES, (name, far(a, e))


@pytest.mark.parametrize("shape", [(3, 5, 6, 18, 9), (3, 300, 4, 64, 64), (2, 300, 4, 100, 64), (2, 300, 4, 64, 128), (2, 300, 4, 128, 128),
                                   (1, 888, 13, 115, 110), (8, 500, 12, 64, 64)])
@pytest.mark.parametrize("reset", [False, True])
def test_float32(cuda_device, shape, reset):
    for decays in (0.2, 0.02):
        names, got, want = both(shape, F32, cuda_device, 32, reset=reset, decays=decays)
        for name, a, e in zip(names, got, want):
            assert far(a, e) <= STATES + 2.0**-22, (name, far(a, e))


def test_steps_without_a_backward(cuda_device):
    """Single steps are sums of 32 bits throughout."""

    for dtype, shape in ((F32, (3, 7, 4, 128, 128)), (BF16, (3, 7, 4, 100, 64))):
        (q, k, v, decay, state), _, _, kw = make(*shape, dtype, gated=True, seed=33)
        _, last = linear_attention(*(t.to(cuda_device) for t in (q, k, v, decay, state)), **kw)
        _, want = definition(*(t.double() for t in (q, k, v, decay, state)), **kw)
        assert far(last.cpu(), want) <= STATES
