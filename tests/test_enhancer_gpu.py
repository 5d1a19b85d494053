"""The training operators together: the example's enhancer."""

import pytest
import torch

from examples.enhancer import Enhancer, train
from triton_pesq_b200.signals import add_noise, speech_like

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_training_lowers_the_loss(cuda_device, bits):
    """Over 80 steps on sixteen batches, whose noise levels repeat every
    eleven: means over the first and the last eleven compare like with like."""

    torch.manual_seed(0)
    model = Enhancer(width=64, blocks=2).to(cuda_device)
    losses = train(model, 88, batch=4, state_bits=bits)
    assert torch.isfinite(losses).all()
    assert float(losses[-11:].mean()) < 0.97 * float(losses[:11].mean())


def test_frame_by_frame_gives_the_same_masks(cuda_device):
    """The matrix products of one frame and of many may differ by their 32-bit
    rounding order (1e-6), which three blocks and a recurrence of memory 2000 may
    raise a hundredfold."""

    torch.manual_seed(1)
    model = Enhancer().to(cuda_device)
    noisy = add_noise(speech_like(3, 32000, 16000, seed=5), 5.0, seed=6).to(cuda_device)
    magnitude = model.spectrum(noisy).abs()
    with torch.no_grad():
        whole, _ = model.masks(magnitude)
    assert float((model.stream_masks(magnitude) - whole).abs().max()) < 1e-4


def test_operators_trace(cuda_device):
    """Shapes and types of the operators' fake kernels are those of the real ones."""

    from torch._subclasses.fake_tensor import FakeTensorMode

    from triton_pesq_b200 import adamw_step, gated_scan, norm_join

    def run(device):
        x = torch.zeros(2, 50, 24, device=device, dtype=torch.bfloat16)
        v = torch.ones(24, device=device)
        y, last = gated_scan(x, x, x, v)
        stream, normed = norm_join(x.float(), x, v, v, gate=x, scale=v)
        p = [torch.zeros(24, device=device)]
        m = torch.zeros(256, device=device)
        adamw_step(p, [v], m, m.clone(), torch.zeros(2, dtype=torch.int64, device=device))
        return y, last, stream, normed

    real = run(cuda_device)
    with FakeTensorMode():
        fake = run(cuda_device)
    for a, b in zip(real, fake):
        assert a.shape == b.shape and a.dtype == b.dtype and a.device == b.device
