"""More rows in a call than a launch takes along its second dimension: bands of many clips in the batch."""

import pytest
import torch

from triton_pesq_b200 import gated_scan, norm_join

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [65535, 65536, 140001])
@pytest.mark.parametrize("shape", [(1, 8), (20, 8), (3, 5)])
def test_gated_scan(cuda_device, batch, shape):
    """Rows are worked on by themselves: as in two calls of half the rows each, bit for bit; the decay's
    gradient is their sum."""

    steps, width = shape
    g = torch.Generator(cuda_device).manual_seed(batch + steps)
    dev = [torch.randn(batch, steps, width, device=cuda_device, generator=g) for _ in range(3)]
    dev += [torch.randn(width, device=cuda_device, generator=g), torch.randn(batch, width, device=cuda_device, generator=g)]
    dy, dlast = torch.randn_like(dev[0]), torch.randn_like(dev[4])
    reset = torch.rand(batch, steps, device=cuda_device, generator=g) < 0.1
    lengths = torch.randint(0, steps + 1, (batch,), device=cuda_device, generator=g)

    def call(rows):
        leaves = [t.detach()[rows].requires_grad_(True) if k != 3 else t.detach().requires_grad_(True) for k, t in enumerate(dev)]
        y, last = gated_scan(*leaves, reset=reset[rows], lengths=lengths[rows])
        with torch.no_grad():
            plain = gated_scan(*leaves, reset=reset[rows], lengths=lengths[rows])
        assert torch.equal(plain[0], y) and torch.equal(plain[1], last)
        return (y, last, *torch.autograd.grad((y, last), leaves, (dy[rows], dlast[rows])))

    got = call(slice(None))
    parts = [call(rows) for rows in (slice(0, 50000), slice(50000, 100000), slice(100000, None)) if batch > rows.start]
    for k, a in enumerate(got):
        if k != 5:
            assert torch.equal(a, torch.cat([p[k] for p in parts]))
        else:  # (sums of `batch` terms in 32 bits, of about the same size and any sign)
            want = sum(p[k].double() for p in parts)
            assert float((a - want).abs().max()) <= 1e-5 * batch**0.5


def test_norm_join_shared_gate(cuda_device):
    batch, steps, width = 70001, 2, 8
    g = torch.Generator(cuda_device).manual_seed(1)
    x, z = (torch.randn(batch, steps, width, device=cuda_device, generator=g) for _ in range(2))
    gate, v = torch.randn(batch, 1, width, device=cuda_device, generator=g), torch.ones(width, device=cuda_device)

    def call(rows):
        leaf = gate[rows].detach().requires_grad_(True)
        out = norm_join(x[rows], z[rows], v, v, gate=leaf)
        return (*out, *torch.autograd.grad(sum((o * x[rows]).sum() for o in out), leaf))

    got, parts = call(slice(None)), [call(slice(0, 40000)), call(slice(40000, None))]
    for k, a in enumerate(got):
        assert torch.equal(a, torch.cat([p[k] for p in parts]))
