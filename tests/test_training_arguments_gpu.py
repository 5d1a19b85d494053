"""Arguments of the training operators' modules and of the ops beneath their gradients."""

import pytest
import torch

from triton_pesq_b200 import GatedScanCuda, NormJoinCuda, _lib

pytestmark = pytest.mark.gpu


def test_gradients_of_other_shapes_are_refused(cuda_device):
    _lib.load_ops()
    ops = torch.ops.pesq_cuda
    x, v, s = (torch.randn(shape, device=cuda_device) for shape in ((2, 40, 16), (16,), (2, 16)))
    y, last, kept = ops.gated_scan_forward(x, x, x, v, s, None, None, False, 8.0, True)
    rest = (x, x, x, v, s, None, None, False, 8.0)
    for dy, dlast in ((y[:, :8], last), (y, last[:1]), (y[0], last), (y.cpu(), last), (y, last.cpu())):
        with pytest.raises((RuntimeError, ValueError)):
            ops.gated_scan_backward(*rest, kept, 0, dy, dlast)
    for bad in (kept[:-16], kept.cpu(), kept[::2]):
        with pytest.raises((RuntimeError, ValueError)):
            ops.gated_scan_backward(*rest, bad, 0, y, last)
    join = (x, x, None, v, v, None, 1e-6, False, False, 0)
    for ds, dn in ((x[:, :8], x), (x, x[:1]), (x[0], x), (x.cpu(), x), (x, x.cpu())):
        with pytest.raises((RuntimeError, ValueError)):
            ops.norm_join_backward(*join, ds, dn)


def test_modules_in_sixteen_bits(cuda_device):
    """`.bfloat16()` on a model takes its vectors along: they are widened for the call, and their gradients come in their type."""

    x = torch.randn(2, 9, 16, device=cuda_device).bfloat16()
    scan, join = GatedScanCuda(16).to(cuda_device), NormJoinCuda(16).to(cuda_device)
    for module in (scan, join):
        for p in module.parameters():
            p.data = p.data.bfloat16().float()
    y, last = scan(x, x, x)
    out = join(x, y, x)
    scan.bfloat16(), join.bfloat16()
    y16, last16 = scan(x, x, x)
    out16 = join(x, y16, x)
    for a, b in zip((y, last, *out), (y16, last16, *out16)):
        assert torch.equal(a, b)
    sum(t.float().sum() for t in (*out16, last16)).backward()
    for p in (*scan.parameters(), *join.parameters()):
        assert p.grad.dtype == torch.bfloat16 and torch.isfinite(p.grad).all()
    scan.double(), join.double()
    for call in (lambda: scan(x, x, x), lambda: join(x, x, x)):
        with pytest.raises(RuntimeError, match="float32"):
            call()
