"""The norm-gate-residual join against its definition in 64 bits.

Bounds.  A row's sums run over at most 8192 values in 32 bits: partial sums of
eight, then a tree, 8 + 10 roundings of 6e-8 at worst, 1e-6; the approximate
exponential, reciprocal and root add 2^-22 each.  TOL is four times that.  The
backward subtracts projections of the gradient, which costs a few times as much
of what they are subtracted from (all of it, for a single channel): GTOL.  Vector gradients are sums of products over up to 10^4 rows in runs of
10 to 100: 100 * 6e-8, VTOL."""

import pytest
import torch

import train_reference as R
from triton_pesq_b200 import NormJoinCuda, norm_join, pre_norm

pytestmark = pytest.mark.gpu

TOL, GTOL, VTOL = 5e-6, 2e-5, 2e-5
NAMES = ("stream", "block", "post", "pre", "gate", "scale")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def inputs(batch, steps, width, stream, dtype, seed=0, gate="full", scale=True):
    g = torch.Generator().manual_seed(seed)
    x = (2 * torch.randn(batch, steps, width, generator=g)).to(stream)
    z = (0.5 * torch.randn(batch, steps, width, generator=g)).to(dtype)
    post, pre = 1 + 0.2 * torch.randn(width, generator=g), 1 + 0.2 * torch.randn(width, generator=g)
    gt = None
    if gate:
        gt = (1.5 * torch.randn(batch, 1 if gate == "shared" else steps, width, generator=g)).to(dtype)
    sc = 0.5 + 0.1 * torch.randn(width, generator=g) if scale else None
    ds, dn = torch.randn(batch, steps, width, generator=g).to(stream), torch.randn(batch, steps, width, generator=g).to(dtype)
    return [x, z, post, pre, gt, sc], ds, dn


def call(t, **kw):
    return norm_join(t[0], t[1], t[2], t[3], gate=t[4], scale=t[5], **kw)


def compare(tensors, ds, dn, device, place=None, **kw):
    place = place or (lambda t: t.to(device))
    mine = [None if t is None else place(t).requires_grad_(True) for t in tensors]
    stream, normed = call(mine, **kw)
    leaves = [t for t in mine if t is not None]
    got = torch.autograd.grad((stream, normed), leaves, (ds.to(device), dn.to(device)))
    wide = [None if t is None else t.double().requires_grad_(True) for t in tensors]
    ws, wn = R.norm_join(*wide, **kw)
    want = torch.autograd.grad((ws, wn), [t for t in wide if t is not None], (ds.double(), dn.double()))
    terms = torch.autograd.grad(R.norm_join(*wide, **kw, fixed=True), [t for t in wide if t is not None],
                                (ds.double(), dn.double()))
    assert stream.dtype == tensors[0].dtype and normed.dtype == tensors[1].dtype
    R.close(stream, ws, TOL, "stream")
    R.close(normed, wn, TOL, "normed")
    names = [n for n, t in zip(NAMES, tensors) if t is not None]
    for n, g, w, leaf, size in zip(names, got, want, leaves, terms):
        assert g.dtype == leaf.dtype
        R.close(g, w, GTOL if g.dim() == 3 else VTOL, "d " + n, size)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 7), (1, 5, 32), (3, 7, 33), (2, 40, 128), (1, 9, 257), (2, 33, 512),
                                   (1, 6, 1000), (2, 3, 2048)])
@pytest.mark.parametrize("activation", ["sigmoid", "silu"])
def test_outputs_and_gradients(cuda_device, types, shape, activation):
    tensors, ds, dn = inputs(*shape, *types, seed=sum(shape))
    compare(tensors, ds, dn, cuda_device, activation=activation)


@pytest.mark.parametrize("width", [3001, 4096, 5000, 8192, 8191])
def test_wide_rows(cuda_device, width):
    for types in ((F32, F32), (BF16, BF16)):
        tensors, ds, dn = inputs(1, 5, width, *types, seed=width)
        compare(tensors, ds, dn, cuda_device)


@pytest.mark.parametrize("gate", ["full", "shared", None])
@pytest.mark.parametrize("scale", [True, False])
@pytest.mark.parametrize("shape", [(3, 50, 24), (2, 1, 64), (5, 700, 100), (1, 2500, 385)])
def test_gates_and_scales(cuda_device, gate, scale, shape):
    for types in ((F32, F32), (F32, BF16)):
        tensors, ds, dn = inputs(*shape, *types, seed=3, gate=gate, scale=scale)
        compare(tensors, ds, dn, cuda_device)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("shape", [(2, 3001, 64), (3, 900, 256), (1, 2000, 896), (2, 500, 1600), (1, 500, 3000), (1, 400, 8192),
                                   (2, 3001, 61), (1, 2000, 900)])
@pytest.mark.parametrize("apart", [False, True])
def test_teams_that_take_several_rows(cuda_device, types, shape, apart):
    """More rows than the device holds teams for; with batch items apart,
    a team's rows stay within one."""

    tensors, ds, dn = inputs(*shape, *types, seed=8)
    place = None
    if apart:
        def place(t):
            if t.dim() < 3:
                return t.to(cuda_device)
            return torch.cat((t, torch.full_like(t[:, :3], float("nan"))), 1).to(cuda_device)[:, :-3]

        assert place(ds).stride(0) > shape[1] * shape[2]
    compare(tensors, ds, dn, cuda_device, place=place)


def test_other_broadcasts_of_the_gate(cuda_device):
    tensors, ds, dn = inputs(3, 20, 40, F32, F32, seed=4)
    for shape in ((40,), (1, 1, 40), (20, 40), (3, 20, 1)):
        t = list(tensors)
        t[4] = torch.randn(shape, generator=torch.Generator().manual_seed(5))
        mine = [v.to(cuda_device).requires_grad_(True) for v in t]
        got = torch.autograd.grad(call(mine), mine, (ds.to(cuda_device), dn.to(cuda_device)))
        wide = [v.double().requires_grad_(True) for v in t]
        want = torch.autograd.grad(R.norm_join(*wide), wide, (ds.double(), dn.double()))
        for n, g, w in zip(NAMES, got, want):
            R.close(g, w, VTOL, "d " + n)


def test_zero_rows_and_large_values(cuda_device):
    """A block row of zeros (the norm's eps alone), gates that are shut or
    open beyond the exponential's range, values near the type's largest."""

    tensors, ds, dn = inputs(2, 6, 64, F32, F32, seed=6)
    tensors[1][0, 0] = 0
    tensors[0][0, 1] = 0
    tensors[1][0, 1] = 0
    tensors[4][0, 2, ::2], tensors[4][0, 2, 1::2] = 300.0, -300.0
    tensors[0][1, 0] *= 1e6
    compare(tensors, ds, dn, cuda_device)
    half, ds, dn = inputs(1, 3, 64, F16, F16, seed=7)
    half[1][0, 0] = 60000.0
    compare(half, ds, dn, cuda_device)


def test_not_a_number_stays_in_its_row(cuda_device):
    tensors, _, _ = inputs(1, 4, 48, F32, F32, seed=8)
    for k in (0, 1, 4):
        t = [v.to(cuda_device) for v in tensors]
        t[k][0, 2, 5] = float("nan")
        stream, normed = call(t)
        assert torch.isnan(normed[0, 2]).all() and torch.isnan(stream[0, 2, 5])
        assert torch.isfinite(normed[0, :2]).all() and torch.isfinite(normed[0, 3]).all()


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16)])
def test_strides(cuda_device, types):
    tensors, ds, dn = inputs(3, 30, 64, *types, seed=9)
    dev = [t.to(cuda_device) for t in tensors]
    want = call(dev)
    packed = torch.cat([dev[1], dev[4].to(types[1])], dim=2)
    forms = [
        [dev[0], packed[..., :64], dev[2], dev[3], packed[..., 64:], dev[5]],
        [t if t.dim() < 3 else t.transpose(0, 1).contiguous().transpose(0, 1) for t in dev],
        [t if t.dim() < 3 else t.transpose(1, 2).contiguous().transpose(1, 2) for t in dev],
        [t if t.dim() < 3 else torch.nn.functional.pad(t, (1, 2))[..., 1:65] for t in dev],
        [t if t.dim() < 3 else t.repeat_interleave(2, dim=1)[:, ::2] for t in dev],
    ]
    for form in forms:
        for a, b in zip(call(form), want):
            R.close(a, b.double(), TOL, "strided")
    leaves = [t.detach().requires_grad_(True) for t in forms[3]]
    ds2 = torch.nn.functional.pad(ds, (3, 0)).to(cuda_device)[..., 3:]
    dn2 = dn.to(cuda_device).transpose(0, 1).contiguous().transpose(0, 1)
    got = torch.autograd.grad(call(leaves), leaves, (ds2, dn2))
    plain = [t.clone().requires_grad_(True) for t in dev]
    for n, a, b in zip(NAMES, got, torch.autograd.grad(call(plain), plain, (ds.to(cuda_device), dn.to(cuda_device)))):
        R.close(a, b.double(), GTOL, "d " + n)


def test_upstream_gradients_that_are_missing_or_broadcast(cuda_device):
    tensors, _, _ = inputs(2, 10, 24, F32, F32, seed=10)
    wide = [t.double().requires_grad_(True) for t in tensors]
    dev = [t.to(cuda_device).requires_grad_(True) for t in tensors]
    for pick in (0, 1):
        got = torch.autograd.grad(call(dev)[pick].sum(), dev, allow_unused=True)
        want = torch.autograd.grad(R.norm_join(*wide)[pick].sum(), wide, allow_unused=True)
        for n, g, w in zip(NAMES, got, want):
            zero = torch.zeros_like(dict(zip(NAMES, wide))[n])
            R.close(zero if g is None else g.cpu().float(), zero if w is None else w, VTOL, f"d {n} of {pick}")


def test_pre_norm(cuda_device):
    for stream, dtype in ((F32, F32), (F32, BF16), (F16, F16)):
        tensors, _, dn = inputs(2, 20, 72, stream, dtype, seed=11)
        x, w = tensors[0].to(cuda_device).requires_grad_(True), tensors[3].to(cuda_device).requires_grad_(True)
        y = pre_norm(x, w, dtype=dtype)
        assert y.dtype == dtype
        got = torch.autograd.grad(y, (x, w), dn.to(cuda_device))
        x64, w64 = tensors[0].double().requires_grad_(True), tensors[3].double().requires_grad_(True)
        _, want = R.norm_join(x64, None, None, w64)
        R.close(y, want, TOL, "normed")
        for g, v in zip(got, torch.autograd.grad(want, (x64, w64), dn.double())):
            R.close(g, v, GTOL, "gradient")


def test_gradient_against_differences(cuda_device):
    """Central differences along each gradient's own direction; the same reckoning
    as for the recurrence: 1 %."""

    tensors, ds, dn = inputs(2, 20, 40, F32, F32, seed=12)
    dev = [t.to(cuda_device) for t in tensors]
    ds, dn = ds.to(cuda_device), dn.to(cuda_device)

    def value(t):
        s, n = call(t)
        return float((s.double() * ds).sum() + (n.double() * dn).sum())

    leaves = [t.clone().requires_grad_(True) for t in dev]
    grads = torch.autograd.grad(call(leaves), leaves, (ds, dn))
    for k, n in enumerate(NAMES):
        way = grads[k] / grads[k].abs().max()
        up, down = list(dev), list(dev)
        up[k], down[k] = dev[k] + 1e-2 * way, dev[k] - 1e-2 * way
        slope, want = (value(up) - value(down)) / 2e-2, float((grads[k].double() * way).sum())
        assert abs(slope - want) <= 1e-2 * abs(want), f"{n}: {slope} against {want}"


def test_the_same_bits_every_time_on_any_stream_and_in_graphs(cuda_device):
    tensors, ds, dn = inputs(4, 500, 96, BF16, BF16, seed=13, gate="shared")
    dev = [t.to(cuda_device) for t in tensors]
    ds, dn = ds.to(cuda_device), dn.to(cuda_device)

    def once():
        leaves = [t.detach().requires_grad_(True) for t in dev]
        out = call(leaves)
        return (*out, *torch.autograd.grad(out, leaves, (ds, dn)))

    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    dev[0].mul_(2)
    again = once()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(held, again):
        assert torch.equal(a, b)


def test_offsets_beyond_32_bits(cuda_device):
    x = torch.randn(1, 1, 2048, device=cuda_device, dtype=BF16).expand(1, 2**20 + 3, 2048)
    w = torch.ones(2048, device=cuda_device)
    stream, normed = norm_join(x, x, w, w)
    assert stream.numel() > 2**31
    for t in (0, 2**19, 2**20 + 2):
        assert torch.equal(stream[0, t], stream[0, 1]) and torch.equal(normed[0, t], normed[0, 1])


def test_empty_sizes(cuda_device):
    for shape in ((0, 3, 8), (2, 0, 8)):
        tensors, ds, dn = inputs(*shape, F32, F32)
        dev = [t.to(cuda_device).requires_grad_(True) for t in tensors]
        out = call(dev)
        assert out[0].shape == shape and out[1].shape == shape
        grads = torch.autograd.grad(out, dev, (ds.to(cuda_device), dn.to(cuda_device)))
        assert not grads[2].any() and not grads[3].any() and not grads[5].any()


def test_refusals(cuda_device):
    tensors, _, _ = inputs(2, 3, 8, F32, F32)
    x, z, post, pre, gate, scale = (t.to(cuda_device) for t in tensors)
    with pytest.raises(TypeError):
        norm_join([1.0], z, post, pre)
    with pytest.raises(ValueError):
        norm_join(x, z, post, pre, activation="tanh")
    for bad in (x[0], x.double(), x.cpu(), x.half()):
        with pytest.raises(RuntimeError):
            norm_join(bad, z, post, pre)
    with pytest.raises(RuntimeError):
        norm_join(x, z.double(), post, pre)
    with pytest.raises(RuntimeError):
        norm_join(x, z, post.half(), pre)
    with pytest.raises(RuntimeError):
        norm_join(x, z, post, pre, gate=gate.bfloat16())
    with pytest.raises(RuntimeError):
        norm_join(x, z, post, pre.cpu())
    with pytest.raises(RuntimeError):
        norm_join(x, z, post, pre, gate=gate[:, :, :5])
    for kw in ({"eps": -1.0}, {"eps": float("nan")}, {"scale": scale[:3]}):
        with pytest.raises(ValueError):
            norm_join(x, z, post, pre, **kw)
    with pytest.raises(ValueError):
        norm_join(x, z[:, :2], post, pre)
    with pytest.raises(ValueError):
        norm_join(x, z, post[:3], pre)
    big = torch.zeros(1, 1, 8193, device=cuda_device)
    with pytest.raises(RuntimeError, match="8192"):
        norm_join(big, big, big[0, 0], big[0, 0])
    for kw in ({"channels": 0}, {"channels": 9000}, {"channels": 4, "activation": "x"}, {"channels": 4, "eps": -1}):
        with pytest.raises(ValueError):
            NormJoinCuda(**kw)
    module = NormJoinCuda(8).to(cuda_device)
    stream, _ = module(x, z, gate)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(stream.sum(), module.scale, create_graph=True)
