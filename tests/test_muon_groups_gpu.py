"""Muon over more matrices than one launch takes: every one against the definition, those of a later launch too, which works in
the memory that an earlier one worked in.  Bounds as in test_muon_gpu.py."""

import pytest
import torch

from test_muon_gpu import matrix, near, newton_schulz, reference_step
from triton_pesq_b200 import _lib, muon_step, orthogonalize

pytestmark = pytest.mark.gpu


def workspace(rows, cols):
    n, m = (-(-x // 128) * 128 for x in sorted((rows, cols)))
    return 4 * (2 * n * m + 3 * n * n)


def test_large_matrices_of_several_launches(cuda_device):
    shapes = [(2100, 2200), (70, 90), (2100, 2200), (2200, 2100), (130, 2000), (2100, 2200)]
    # (two of the large ones go together, a third is past the limit of 256 MB)
    assert 2 * workspace(2100, 2200) < 256 << 20 < 3 * workspace(2100, 2200)
    x = [matrix(*s, seed=30 + i).to(cuda_device) for i, s in enumerate(shapes)]
    p = [matrix(*s, seed=50 + i).to(cuda_device) for i, s in enumerate(shapes)]
    before, m = [t.clone() for t in p], [torch.zeros_like(t) for t in p]
    muon_step(p, x, m, lr=1.0, weight_decay=0.0)
    assert _lib.muon_check() == 0
    for i, (a, b, g) in enumerate(zip(p, before, x)):
        want, momentum = reference_step(b.double(), g.double(), torch.zeros_like(g).double(), 1.0, decay=0.0)
        # (lr times the iteration's error; the parameters' roundings)
        near(a, want.cpu(), f"matrix {i}", scale=2.0)
        assert float((m[i].double() - momentum).abs().max()) <= 4 * 2.0**-24 * float(momentum.abs().max())


@pytest.mark.parametrize("shape", [(150, 20, 30), (300, 130, 40)])
def test_stacks_of_several_launches(cuda_device, shape):
    x = matrix(*shape, seed=9).to(cuda_device)
    got = orthogonalize(x)
    assert _lib.muon_check() == 0
    near(got, newton_schulz(x.double()).cpu(), "stack")


def test_what_is_written_twice_is_refused(cuda_device):
    p, g, m = (matrix(4, 6, seed=i).to(cuda_device) for i in range(3))
    before, version = [t.clone() for t in (p, m)], p._version
    flat = torch.zeros(40, device=cuda_device)
    for bad in (lambda: muon_step([p, p], [g, g], [m, m.clone()]), lambda: muon_step([p, p.clone()], [g, g], [m, m]),
                lambda: muon_step([p], [g], [p]), lambda: muon_step([flat[:24].view(4, 6), flat[12:36].view(4, 6)], [g, g], [m, m.clone()])):
        with pytest.raises(ValueError, match="share"):
            bad()
    for a, b in zip((p, m), before):
        assert torch.equal(a, b)
    assert p._version == version
    # (without a gradient a matrix is not written)
    muon_step([p, p], [g, g[:0]], [m, m])
    assert not torch.equal(p, before[0])
