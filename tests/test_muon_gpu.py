"""Muon and its Newton-Schulz iteration against their definition in 64 bits.

Bounds, on the norm of the difference (the largest element's is no larger).  A product's operands are 2^-23 off each and
its sum's roundings of random sign no more, so that a step adds 2^-21 of its matrix' norm at most.  The iteration enlarges what is
added by its polynomial's slope, at most 3.4445 a step on small singular values: 485 in five, of a matrix of norm 1
at first, which then grows to the result's norm with slopes around 1.  So 485 * 2^-21 and 20 * 2^-21 of the result's norm, and the
result's own rounding."""

import copy

import pytest
import torch

import train_reference as R
from triton_pesq_b200 import MuonCuda, _lib, muon_step, orthogonalize
from triton_pesq_b200.muon import COEFFICIENTS

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def newton_schulz(u, eps=1e-7, steps=5, coefficients=COEFFICIENTS):
    a, b, c = coefficients
    x = u.mT if u.shape[-2] > u.shape[-1] else u
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp_min(eps)
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.mT if u.shape[-2] > u.shape[-1] else x


def near(got, want, what="", scale=1.0):
    assert got.shape == want.shape
    g, w = got.detach().cpu().double(), want.double()
    assert torch.isfinite(g).all(), what
    size = torch.linalg.matrix_norm(w)
    allowed = scale * (485 + 20 * size) * 2.0**-21 + R.ROUND[got.dtype] * size
    off = torch.linalg.matrix_norm(g - w)
    assert (off <= allowed).all(), f"{what}: {off.max():.3e} against {allowed.max():.3e}"


def matrix(*shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (9, 1), (5, 5), (16, 64), (64, 16), (96, 288), (128, 128), (129, 127), (128, 64),
                                   (257, 96), (200, 640), (640, 200), (385, 385), (300, 1155)])
def test_iteration(cuda_device, shape):
    x = matrix(*shape, seed=sum(shape))
    near(orthogonalize(x.to(cuda_device)), newton_schulz(x.double()), "x")
    assert _lib.muon_check() == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(3, 40, 70), (2, 3, 130, 60), (140, 33)])
def test_types_and_stacks(cuda_device, dtype, shape):
    x = matrix(*shape, dtype=dtype)
    got = orthogonalize(x.to(cuda_device))
    assert got.dtype == dtype
    near(got, newton_schulz(x.double()), "x")
    near(orthogonalize(x.mT.to(cuda_device)), newton_schulz(x.double().mT), "a transpose")


def test_singular_values_come_near_one(cuda_device):
    x = matrix(150, 400, seed=3)
    s = torch.linalg.svdvals(orthogonalize(x.to(cuda_device)).double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


def test_scales_ranks_and_steps(cuda_device):
    """Matrices far from 1, below eps, of zeros, of few directions, other numbers of steps and coefficients."""

    x = matrix(60, 100, seed=4)
    for scale in (1e-30, 1e-4, 1e15, 1e30):
        near(orthogonalize((scale * x).to(cuda_device), eps=1e-36), newton_schulz((scale * x).double(), eps=1e-36), str(scale))
    small = 1e-12 * x
    near(orthogonalize(small.to(cuda_device)), newton_schulz(small.double()), "below eps")
    assert not orthogonalize(torch.zeros(60, 100, device=cuda_device)).any()
    low = matrix(200, 3, seed=5) @ matrix(3, 150, seed=6)
    near(orthogonalize(low.to(cuda_device)), newton_schulz(low.double()), "of rank 3")
    for steps in (1, 2, 3):
        near(orthogonalize(x.to(cuda_device), steps=steps), newton_schulz(x.double(), steps=steps), f"{steps} steps")
    cubic = (1.5, -0.5, 0.0)
    near(orthogonalize(x.to(cuda_device), steps=8, coefficients=cubic), newton_schulz(x.double(), steps=8, coefficients=cubic), "cubic")


def test_the_least_eps(cuda_device):
    """A reciprocal that is just in float32's range: 1 / eps is, 2^10 / eps is not."""

    x = 1e-37 * matrix(60, 100, seed=7)
    for eps in (2e-38, 1.2e-38):
        near(orthogonalize(x.to(cuda_device), eps=eps), newton_schulz(x.double(), eps=eps), "above eps")
        tiny = 1e-3 * x
        # (subnormal inputs are as exact as their last bit, 1.4e-45, beside a norm of some 1e-38)
        near(orthogonalize(tiny.to(cuda_device), eps=eps), newton_schulz(tiny.double(), eps=eps), "below eps")
    with pytest.raises(ValueError, match="eps"):
        orthogonalize(x.to(cuda_device), eps=1e-39)


def test_offsets_past_32_bits(cuda_device):
    """A matrix whose tiles lie more than 2^32 bytes into the workspace."""

    x = matrix(8192, 32768, seed=8).to(cuda_device)
    got = orthogonalize(x, steps=2)
    assert _lib.muon_check() == 0
    want = newton_schulz(x.double(), steps=2)
    size = torch.linalg.matrix_norm(want)
    off = torch.linalg.matrix_norm(got.double() - want)
    # (two steps' slopes: 3.4445^2 of what is added to a norm of 1, and 20 as above)
    assert off <= (12 + 20 * size) * 2.0**-21 + R.ROUND[F32] * size, (off, size)
    rows = torch.linalg.vector_norm(got.double() - want, dim=1) / torch.linalg.vector_norm(want, dim=1)
    assert rows.max() < 2.0**-15


def test_what_is_not_finite_stays_in_its_matrix(cuda_device):
    x = matrix(3, 70, 50).to(cuda_device)
    want = orthogonalize(x)
    x[1, 5, 7] = float("nan")
    got = orthogonalize(x)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and not torch.isfinite(got[1]).any()


def reference_step(p, g, m, lr, momentum=0.95, nesterov=True, decay=0.1, adjust="original"):
    m = momentum * m + (1 - momentum) * g
    x = newton_schulz(momentum * m + (1 - momentum) * g if nesterov else m)
    rows, cols = p.shape
    factor = max(1.0, rows / cols)**0.5 if adjust == "original" else 0.2 * max(rows, cols)**0.5
    return p * (1 - lr * decay) - lr * factor * x, m


SHAPES = [(96, 257), (288, 96), (96, 96), (257, 96), (130, 7), (1, 40)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", ["original", "match_rms_adamw"])
@pytest.mark.parametrize("with_copies", [False, True])
def test_step(cuda_device, dtype, nesterov, adjust, with_copies):
    if with_copies and dtype == F32:
        pytest.skip("copies are 16-bit")
    p = [matrix(*s, seed=i) for i, s in enumerate(SHAPES)]
    g = [(1e-3 * matrix(*s, seed=20 + i)).to(dtype) for i, s in enumerate(SHAPES)]
    m = [1e-3 * matrix(*s, seed=40 + i) for i, s in enumerate(SHAPES)]
    mine = [[t.to(cuda_device) for t in ts] for ts in (p, g, m)]
    copies = [torch.zeros_like(t) for t in mine[1]] if with_copies else None
    wide = [[t.double() for t in ts] for ts in (p, g, m)]
    lr = 0.02
    for _ in range(2):
        muon_step(*mine, lr=lr, nesterov=nesterov, adjust=adjust, copies=copies)
        for i in range(len(SHAPES)):
            wide[0][i], wide[2][i] = reference_step(wide[0][i], wide[1][i], wide[2][i], lr, nesterov=nesterov, adjust=adjust)
    for i, (rows, cols) in enumerate(SHAPES):
        factor = max(1.0, rows / cols)**0.5 if adjust == "original" else 0.2 * max(rows, cols)**0.5
        # two steps: an update's error each, of lr times the iteration's, and the parameters' own roundings
        off = torch.linalg.matrix_norm(mine[0][i].cpu().double() - wide[0][i])
        x = wide[0][i].shape[0]**0.5
        assert off <= 2 * lr * factor * (485 + 20 * min(rows, cols)**0.5 * 1.25) * 2.0**-21 + 4 * 2.0**-24 * torch.linalg.matrix_norm(wide[0][i]), (i, off)
        R.close(mine[2][i], wide[2][i], 4 * 2.0**-24, "momentum")
        if with_copies:
            assert torch.equal(copies[i], mine[0][i].to(dtype))
    assert _lib.muon_check() == 0


def test_many_matrices_go_in_several_launches(cuda_device):
    shapes = [(8 + i % 5, 9 + i % 7) for i in range(150)] + [(2100, 2200)] * 3
    x = [matrix(*s, seed=i) for i, s in enumerate(shapes)]
    p = [t.to(cuda_device) for t in x]
    m = [torch.zeros_like(t) for t in p]
    muon_step(p, [t.to(cuda_device) for t in x], m, lr=1.0, weight_decay=0.0)
    for i in (0, 77, 127, 128, 149):
        # (lr times the iteration's error; the parameters' roundings)
        want, _ = reference_step(x[i].double(), x[i].double(), torch.zeros_like(x[i]).double(), 1.0, decay=0.0)
        near(p[i], want, f"matrix {i}", scale=2.0)
    s = torch.linalg.svdvals(((x[150].to(cuda_device) - p[150])).double())
    assert float(s.max()) < 1.25 and float(s.median()) > 0.6
    assert torch.equal(p[150] - p[150], p[152] - p[152]) and _lib.muon_check() == 0


def test_grad_scale_and_missing_gradients(cuda_device):
    p, g = [matrix(20, 30, seed=i).to(cuda_device) for i in range(2)], [matrix(20, 30, seed=9).to(cuda_device), torch.empty(0, device=cuda_device)]
    m = [torch.zeros(20, 30, device=cuda_device) for _ in range(2)]
    before = [t.clone() for t in (*p, *m)]
    muon_step(p, g, m, grad_scale=torch.tensor([float("inf")], device=cuda_device))
    for a, b in zip((*p, *m), before):
        assert torch.equal(a, b)
    half = [t.clone() for t in p], [t.clone() for t in m]
    muon_step(p, g, m, grad_scale=torch.tensor([0.25], device=cuda_device))
    muon_step(half[0], [g[0] * 0.25, g[1]], half[1])
    assert torch.equal(p[0], half[0][0]) and torch.equal(m[0], half[1][0]) and not torch.equal(p[0], before[0])
    assert torch.equal(p[1], before[1]) and torch.equal(m[1], before[3])


def test_the_same_every_time_and_a_captured_step(cuda_device):
    p = [matrix(*s, seed=i).to(cuda_device) for i, s in enumerate(SHAPES)]
    g = [matrix(*s, seed=20 + i).to(cuda_device) for i, s in enumerate(SHAPES)]
    m = [torch.zeros_like(t) for t in p]
    runs = [([t.clone() for t in p], [t.clone() for t in m]) for _ in range(2)]
    for r in runs:
        for _ in range(3):
            muon_step(r[0], g, r[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        muon_step(p, g, m)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step(p, g, m)
    graph.replay()
    graph.replay()
    for a, b, c in zip(*[r[0] + r[1] for r in runs], p + m):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_two_streams_at_once(cuda_device):
    x = [matrix(3, 300, 500, seed=i).to(cuda_device) for i in range(2)]
    want = [orthogonalize(t) for t in x]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in x], []
    for t, stream in zip(x, streams):
        with torch.cuda.stream(stream):
            got.append(orthogonalize(t))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert _lib.muon_check() == 0


def test_optimiser(cuda_device):
    """Against muon_step by hand, in groups, with 16-bit parameters, saved, loaded and copied."""

    for dtype in (F32, BF16):
        params = [torch.nn.Parameter(matrix(*s, seed=i).to(cuda_device, dtype)) for i, s in enumerate(SHAPES[:4])]
        idle = torch.nn.Parameter(torch.ones(3, 4, device=cuda_device, dtype=dtype))
        opt = MuonCuda([{"params": params[:2], "lr": 0.05}, {"params": [*params[2:], idle], "nesterov": False}], lr=0.02)
        masters = [p.detach().float() for p in params]
        m = [torch.zeros_like(t) for t in masters]
        for step in range(3):
            for i, p in enumerate(params):
                p.grad = matrix(*p.shape, seed=100 * step + i).to(cuda_device, dtype)
            for part, kw in ((slice(0, 2), {"lr": 0.05}), (slice(2, 4), {"lr": 0.02, "nesterov": False})):
                muon_step(masters[part], [p.grad for p in params[part]], m[part], **kw)
            if step == 1:
                other = [torch.nn.Parameter(p.detach().clone()) for p in (*params, idle)]
                new = MuonCuda([{"params": other[:2]}, {"params": other[2:]}])
                new.load_state_dict(opt.state_dict())
                twin = copy.deepcopy(opt)
                for a, b in zip([p for q in twin.param_groups for p in q["params"]], (*params, idle)):
                    a.grad = None if b.grad is None else b.grad.clone()
                twin.step()
                for a, b in zip(other, params):
                    a.grad = b.grad.clone()
                new.step()
                for a, b in zip([p for q in twin.param_groups for p in q["params"]], other):
                    assert torch.equal(a, b)
            opt.step()
            for p, w in zip(params, masters):
                assert torch.equal(p, w.to(dtype))
            if step == 1:
                for a, b in zip(other, (*params, idle)):
                    assert torch.equal(a, b)
        assert torch.equal(idle, torch.ones_like(idle)) and idle not in opt.state
        assert opt.check_errors() == 0


def test_refusals(cuda_device):
    p, g, m = (matrix(4, 6, seed=i).to(cuda_device) for i in range(3))
    for bad in (lambda: muon_step([p.half()], [g], [m]), lambda: muon_step([p], [g.double()], [m]), lambda: muon_step([p], [g], [m.half()]),
                lambda: muon_step([p], [g], [m], copies=[p.half()]), lambda: muon_step([p], [g.half()], [m], copies=[p.bfloat16()]),
                lambda: muon_step([p.cpu()], [g], [m]), lambda: muon_step([p], [g.cpu()], [m]),
                lambda: muon_step([p.T], [g.T], [m.T]), lambda: muon_step([p, p.clone()], [g, g.half()], [m, m.clone()]),
                lambda: orthogonalize(p.double()), lambda: orthogonalize(torch.zeros(2, 32769, device=cuda_device)),
                lambda: MuonCuda([torch.nn.Parameter(torch.zeros(5, device=cuda_device))]),
                lambda: MuonCuda([torch.nn.Parameter(p.T)]), lambda: MuonCuda([torch.nn.Parameter(p.double())])):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: muon_step([p], [g, g], [m]), lambda: muon_step([p], [g], [m], copies=[p, p]), lambda: muon_step([p], [g[:2]], [m]),
                lambda: muon_step([p], [g], [m[:2]]), lambda: muon_step([p[0]], [g[0]], [m[0]]), lambda: muon_step([p], [g], [m], lr=-1.0),
                lambda: muon_step([p], [g], [m], momentum=1.0), lambda: muon_step([p], [g], [m], steps=0),
                lambda: muon_step([p], [g], [m], eps=0.0), lambda: muon_step([p], [g], [m], coefficients=(17.0, 0.0, 0.0)),
                lambda: muon_step([p], [g], [m], adjust="none"), lambda: orthogonalize(p[0]), lambda: orthogonalize(p, steps=101),
                lambda: orthogonalize(p, eps=float("nan"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        orthogonalize(None)
    param = torch.nn.Parameter(p.clone())
    param.grad = g
    opt = MuonCuda([param])
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="captur"):
                opt.step()
        finally:
            graph.capture_end()
    opt.step()
    with pytest.raises(ValueError):
        opt.load_state_dict({**opt.state_dict(), "state": {0: {"momentum": torch.zeros(3, 3)}}})
    assert orthogonalize(torch.zeros(0, 4, device=cuda_device)).shape == (0, 4)
    muon_step([], [], [])
