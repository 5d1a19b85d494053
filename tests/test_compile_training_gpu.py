"""The training operators under tracing: the shapes of their fake kernels are
the real ones, for every layout of the streams, and a compiled training step
returns what the eager one returns."""

import pytest
import torch

from triton_pesq_b200 import _lib, gated_scan, norm_join

pytestmark = pytest.mark.gpu

CHECKS = ("test_schema", "test_faketensor")
OPS = torch.ops.pesq_cuda


@pytest.fixture(autouse=True)
def _ops():
    _lib.load_ops()


def streams(shape, dtype, device, boxes, seed=0):
    """Three streams that tensor copies take (``boxes``) or that lie off their alignment."""

    g = torch.Generator(device).manual_seed(seed)
    batch, steps, width = shape
    out = []
    for _ in range(3):
        t = torch.randn(batch, steps, width + (0 if boxes else 1), device=device, generator=g).to(dtype)
        out.append(t if boxes else t[:, :, 1:])
    return out


@pytest.mark.parametrize("shape", [(2, 1, 64), (2, 5, 64), (2, 300, 96), (3, 90, 33), (600, 40, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("boxes", [True, False])
def test_opcheck_gated_scan(cuda_device, shape, dtype, boxes):
    x, ig, rg = streams(shape, dtype, cuda_device, boxes)
    decay, state = torch.zeros(shape[2], device=cuda_device), torch.zeros(shape[0], shape[2], device=cuda_device)
    reset = torch.zeros(shape[:2], dtype=torch.bool, device=cuda_device)
    for keep in (True, False):
        args = (x, ig, rg, decay, state, reset, None, False, 8.0, keep)
        torch.library.opcheck(OPS.gated_scan_forward.default, args, test_utils=CHECKS)
    y, last, kept = OPS.gated_scan_forward(x, ig, rg, decay, state, reset, None, False, 8.0, True)
    args = (x, ig, rg, decay, state, reset, None, False, 8.0, kept, 0, y, last)
    torch.library.opcheck(OPS.gated_scan_backward.default, args, test_utils=CHECKS)


@pytest.mark.parametrize("shared", [True, False])
def test_opcheck_norm_join(cuda_device, shared):
    x = torch.randn(3, 20, 48, device=cuda_device)
    z, v = x.bfloat16(), torch.ones(48, device=cuda_device)
    gate = z[:, :1] if shared else z
    args = (x, z, gate, v, v, v, 1e-6, True, shared, 1)
    torch.library.opcheck(OPS.norm_join_forward.default, args, test_utils=CHECKS)
    torch.library.opcheck(OPS.norm_join_backward.default, (*args, x, z), test_utils=CHECKS)


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_compiled_training_step(cuda_device, backend):
    """Lengths that change between calls, too."""

    def step(h, weight, decay, post, stream):
        x, ig, rg = torch.matmul(h, weight).chunk(3, dim=2)
        y, last = gated_scan(x, ig, rg, decay)
        stream, normed = norm_join(stream, y, post, post, gate=x, scale=post)
        return stream, normed, last

    torch._dynamo.reset()
    compiled = torch.compile(step, backend=backend, fullgraph=True, dynamic=True)
    for steps in (300, 90, 64):
        g = torch.Generator(cuda_device).manual_seed(steps)
        args = [torch.randn(2, steps, 32, device=cuda_device, generator=g).bfloat16(),
                0.2 * torch.randn(32, 288, device=cuda_device, generator=g).bfloat16(),
                torch.randn(96, device=cuda_device, generator=g), 1 + 0.1 * torch.randn(96, device=cuda_device, generator=g),
                torch.randn(2, steps, 96, device=cuda_device, generator=g)]
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
