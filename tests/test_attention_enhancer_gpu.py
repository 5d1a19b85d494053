"""The linear attention, the layer norm and Muon together, as the example's enhancer uses them."""

import pytest
import torch

from examples.enhancer import AttentionBlock, Enhancer, train
from triton_pesq_b200 import _lib
from triton_pesq_b200.signals import add_noise, speech_like

pytestmark = pytest.mark.gpu


def plain_block(block, stream, normed, state):
    """The block's definition in elementary operations, in the type of its inputs."""

    inner = normed @ block.inner.weight.to(normed).T + block.inner.bias.to(normed)
    q, k, v, gate = inner.chunk(4, dim=2)
    q, k, v = (t.unflatten(2, (block.heads, block.channels)) for t in (q, k, v))
    a = torch.exp(-torch.nn.functional.softplus(block.attention.decay.to(normed)))
    ys = []
    for t in range(q.shape[1]):
        state = a[:, None, None] * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        ys.append(block.channels**-0.5 * (q[:, t, :, None, :] @ state)[:, :, 0])
    y = torch.stack(ys, dim=1)
    var, mean = torch.var_mean(y, dim=-1, correction=0, keepdim=True)
    y = (y - mean) / torch.sqrt(var + block.norm.eps) * block.norm.weight.to(y) + block.norm.bias.to(y)
    y = y.flatten(2) @ block.outer.weight.to(y).T + block.outer.bias.to(y)

    def rms(x):
        return x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + block.join.eps)

    stream = stream + block.join.scale.to(y) * torch.nn.functional.silu(gate) * rms(y) * block.join.post_weight.to(y)
    return stream, rms(stream) * block.join.pre_weight.to(y), state


def test_a_block_and_its_gradients(cuda_device):
    """Against its definition in 64 bits on the same weights.  Each of the block's products and norms is 1e-6 off (sums of up
    to 100 terms in 32 bits), a norm of a head that is nearly constant may enlarge that tenfold, and five of them follow each
    other: 1e-4 of the largest value, and twice that for gradients, which go through all of them twice."""

    torch.manual_seed(3)
    block = AttentionBlock(48, heads=3).to(cuda_device)
    args = [torch.randn(2, 100, 48, device=cuda_device) for _ in range(2)] + [torch.randn(2, 3, 16, 16, device=cuda_device)]
    mine = [a.clone().requires_grad_(True) for a in args]
    out = block(mine[0], mine[1], mine[2])
    ups = [torch.randn_like(o) for o in out]
    names, params = zip(*block.named_parameters())
    got = torch.autograd.grad(out, [*mine, *params], ups)
    wide = [a.double().requires_grad_(True) for a in args]
    want_out = plain_block(block, *wide)
    want = torch.autograd.grad(want_out, [*wide, *params], [u.double() for u in ups])
    for o, w in zip(out, want_out):
        assert float((o.double() - w).abs().max()) <= 1e-4 * float(w.abs().max())
    for name, g, w in zip(("stream", "normed", "state", *names), got, want):
        assert float((g.double() - w.double()).abs().max()) <= 2e-4 * float(w.abs().max()), name


@pytest.mark.parametrize("muon", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_training_runs(cuda_device, muon, bits):
    torch.manual_seed(0)
    model = Enhancer(width=64, blocks=2, mixer="attention").to(cuda_device)
    before = [p.detach().clone() for p in model.parameters()]
    losses = train(model, 4, batch=4, state_bits=bits, muon=muon)
    assert torch.isfinite(losses).all()
    assert all(not torch.equal(a, b) and torch.isfinite(b).all() for a, b in zip(before, model.parameters()))
    assert _lib.muon_check() == 0


def test_frame_by_frame_gives_the_same_masks(cuda_device):
    """The matrix products of one frame and of many may differ by their 32-bit rounding order (1e-6), which three blocks, their
    norms and memories of 500 frames may raise a hundredfold."""

    torch.manual_seed(1)
    model = Enhancer(mixer="attention").to(cuda_device)
    noisy = add_noise(speech_like(3, 32000, 16000, seed=5), 5.0, seed=6).to(cuda_device)
    magnitude = model.spectrum(noisy).abs()
    with torch.no_grad():
        whole, _ = model.masks(magnitude)
    assert float((model.stream_masks(magnitude) - whole).abs().max()) < 1e-4
