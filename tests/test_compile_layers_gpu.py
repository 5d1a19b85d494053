"""The layer norm, the linear attention and Muon under tracing: the shapes of their fake kernels are the real ones, and a
compiled training step returns what the eager one returns."""

import pytest
import torch

from triton_pesq_b200 import _lib, layer_norm, linear_attention, muon_step, orthogonalize

pytestmark = pytest.mark.gpu

CHECKS = ("test_schema", "test_faketensor")
OPS = torch.ops.pesq_cuda


@pytest.fixture(autouse=True)
def _ops():
    _lib.load_ops()


@pytest.mark.parametrize("widths", [(8, 8), (48, 33), (128, 128), (0, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gated", [True, False])
def test_opcheck_linear_attention(cuda_device, widths, dtype, gated):
    key, value = widths
    q, v = (torch.randn(2, 150, 3, n, device=cuda_device).to(dtype) for n in (key, value))
    g = torch.zeros(2, 150, 3, device=cuda_device) if gated else torch.zeros(3, device=cuda_device)
    state = torch.zeros(2, 3, key, value, device=cuda_device)
    reset = torch.zeros(2, 150, dtype=torch.bool, device=cuda_device)
    for keep in (True, False):
        args = (q, q, v, g, state, reset, None, False, 0.5, keep)
        torch.library.opcheck(OPS.linear_attention_forward.default, args, test_utils=CHECKS)
    y, last, kept = OPS.linear_attention_forward(q, q, v, g, state, reset, None, False, 0.5, True)
    args = (q, q, v, g, state, reset, None, False, 0.5, kept, y, last)
    torch.library.opcheck(OPS.linear_attention_backward.default, args, test_utils=CHECKS)


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("shape,own", [((3, 20, 48), 1), ((3, 20, 4, 12), 2), ((48,), 1), ((2, 2, 2, 3, 5), 1)])
def test_opcheck_layer_norm(cuda_device, bias, shape, own):
    x = torch.randn(shape, device=cuda_device)
    w = torch.ones(shape[-own:], device=cuda_device)
    args = (x, w, w if bias else None, 1e-5, 1)
    torch.library.opcheck(OPS.layer_norm_forward.default, args, test_utils=CHECKS)
    torch.library.opcheck(OPS.layer_norm_backward.default, (*args, x.bfloat16()), test_utils=CHECKS)


def test_shapes_of_muon(cuda_device):
    from torch._subclasses.fake_tensor import FakeTensorMode

    torch.library.opcheck(OPS.orthogonalize.default, (torch.randn(2, 5, 9, device=cuda_device), 1.5, -0.5, 0.0, 1e-7, 2),
                          test_utils=CHECKS)
    with FakeTensorMode():
        p, g, m = ([torch.zeros(4, 6, device=cuda_device)] for _ in range(3))
        muon_step(p, g, m)
        assert orthogonalize(p[0]).shape == (4, 6)


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_compiled_training_step(cuda_device, backend):
    """Lengths that change between calls, too."""

    def step(h, weight, decay, norm, bias):
        q, k, v = torch.matmul(h, weight).unflatten(2, (4, 72)).split((16, 16, 40), dim=3)
        y, last = linear_attention(q, k, v, decay, scale=0.25)
        return layer_norm(y, norm, bias), last

    torch._dynamo.reset()
    compiled = torch.compile(step, backend=backend, fullgraph=True, dynamic=True)
    for steps in (300, 90, 64):
        g = torch.Generator(cuda_device).manual_seed(steps)
        args = [torch.randn(2, steps, 32, device=cuda_device, generator=g).bfloat16(),
                0.2 * torch.randn(32, 288, device=cuda_device, generator=g).bfloat16(),
                -0.1 * torch.rand(4, device=cuda_device, generator=g), 1 + 0.1 * torch.randn(4, 40, device=cuda_device, generator=g),
                0.1 * torch.randn(4, 40, device=cuda_device, generator=g)]
        results = []
        for fn in (step, compiled):
            leaves = [a.clone().requires_grad_(True) for a in args]
            out = fn(*leaves)
            results.append((*out, *torch.autograd.grad(sum(o.float().sum() for o in out), leaves)))
        for a, b in zip(*results):
            assert a.shape == b.shape and a.dtype == b.dtype
            if backend == "aot_eager":
                assert torch.equal(a, b)
            else:  # (the order of the products' sums may differ: bfloat16's rounding, a few times)
                assert float((a.float() - b.float()).norm()) <= 2.0**-6 * float(a.float().norm())
