"""The training operators have no forward-mode derivatives, and say so."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from triton_pesq_b200 import gated_scan, norm_join, pre_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(cuda_device, grad):
    x, v, s = (torch.randn(shape, device=cuda_device) for shape in ((2, 5, 8), (8,), (2, 8)))
    calls = [(lambda *t: gated_scan(*t), (x, x, x, v, s)), (lambda a, b, c, d, e, f: norm_join(a, b, c, d, gate=e, scale=f), (x, x, v, v, x, v)),
             (pre_norm, (x, v))]
    for fn, args in calls:
        for k in range(len(args)):
            mine = [t.clone().requires_grad_(grad) for t in args]
            fn(*mine)
            with forward_ad.dual_level():
                mine[k] = forward_ad.make_dual(mine[k], torch.ones_like(mine[k]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    fn(*mine)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda t: gated_scan(t, x, x, v)[0], (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda t: norm_join(x, x, v, v, gate=t)[0], (x[:, :1],), (torch.ones_like(x[:, :1]),))
