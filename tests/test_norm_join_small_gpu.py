"""The join's norms at the lower end of the range."""

import pytest
import torch

from triton_pesq_b200 import norm_join, pre_norm

pytestmark = pytest.mark.gpu


def test_small_rows_without_eps(cuda_device):
    """Rows of 1e-20, whose mean square, 1e-40, lies below the normal range in steps of 1.4e-45, eps = 0: normed
    to one.  1e-5 relative in the square's rounding, 1e-4 is allowed."""

    x = torch.full((1, 3, 40), 1e-20, device=cuda_device, requires_grad=True)
    one = torch.ones(40, device=cuda_device)
    assert float((pre_norm(x, one, eps=0.0) - 1).detach().abs().max()) <= 1e-4
    stream, normed = norm_join(torch.zeros_like(x), x, one, one, eps=0.0)
    assert float((stream - 1).detach().abs().max()) <= 1e-4 and float((normed - 1).detach().abs().max()) <= 1e-4
    (d,) = torch.autograd.grad(normed[..., 0].sum() + stream[..., 1].sum(), x)
    assert torch.isfinite(d).all()
