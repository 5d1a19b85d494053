"""The Newton-Schulz iteration is about as exact as in float32 products, whatever the matrices' sides: by the norm of what it is
away from 64 bits, half as much again at most (operands of 22 bits and sums that are cut off every 16 to 64 columns, against
operands of 24 and a rounding for every product).  Matrices of a few rows get as many in the stack as make up some 300 rows."""

import pytest
import torch

from test_muon_gpu import newton_schulz
from triton_pesq_b200 import _lib, orthogonalize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(16, 20, 200), (8, 37, 225), (6, 441, 48), (6, 52, 725), (5, 64, 64), (5, 506, 70), (4, 80, 1000),
                                   (3, 96, 288), (3, 128, 128), (2, 300, 300), (3, 100, 1100), (2, 385, 1155), (1, 700, 1000)])
def test_float32(cuda_device, shape):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape))).to(cuda_device)
    want = newton_schulz(x.double())
    allowed = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        plain = newton_schulz(x)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = allowed
    off, base = (float((t.double() - want).norm() / want.norm()) for t in (orthogonalize(x), plain))
    assert _lib.muon_check() == 0 and off <= 1.5 * base, (off, base)
