"""The layer norm against its definition in 64 bits.

Bounds.  A row's sums run over at most 8192 values in 32 bits: partial sums of eight, then a tree, 8 + 10 roundings of
6e-8 at worst, 1e-6, of which the mean's is relative to the row's mean absolute value (here at most a few
deviations); the approximate root adds 2^-22.  TOL is four times that.  The gradient subtracts projections, of values up to
the largest of dy times weight, over the root: GTOL, four times more.  Vector gradients are sums of products over up to
10^4 rows in runs of 10 to 100: 100 * 6e-8, VTOL, of the square root of the number of rows times the terms' size
(their sum of random signs), which `close` takes as the largest value."""

import pytest
import torch

import train_reference as R
from triton_pesq_b200 import LayerNormCuda, layer_norm

pytestmark = pytest.mark.gpu

TOL, GTOL, VTOL = 5e-6, 2e-5, 2e-5
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def definition(x, weight, bias, eps):
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + eps) * weight
    return y if bias is None else y + bias


def make(shape, vector, dtype, out, bias=True, seed=0, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (offset + 1.5 * torch.randn(shape, generator=g)).to(dtype)
    w = 1 + 0.2 * torch.randn(vector, generator=g)
    b = 0.3 * torch.randn(vector, generator=g) if bias else None
    dy = torch.randn(shape, generator=g).to(out)
    return x, w, b, dy


def compare(x, w, b, dy, device, place=None, eps=1e-5, scale=1.0):
    place = place or (lambda t: t.to(device))
    mine = [None if t is None else f(t).requires_grad_(True) for t, f in ((x, place), (w, lambda t: t.to(device)), (b, lambda t: t.to(device)))]
    y = layer_norm(*mine, eps=eps, dtype=dy.dtype)
    assert y.dtype == dy.dtype and y.shape == x.shape
    got = torch.autograd.grad(y, [t for t in mine if t is not None], place(dy))
    wide = [None if t is None else t.double().requires_grad_(True) for t in (x, w, b)]
    want_y = definition(*wide, eps)
    want = torch.autograd.grad(want_y, [t for t in wide if t is not None], dy.double())
    R.close(y, want_y, TOL * scale, "y")
    root = torch.sqrt(torch.var(x.double(), dim=-1, correction=0) + eps)
    terms = (dy.double() * w.double()).abs().amax() / root.min()
    for name, a, e in zip(("x", "weight", "bias"), got, want):
        R.close(a, e, (GTOL if name == "x" else VTOL) * scale, "d " + name, terms if name == "x" else dy.double().abs().max())


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)])
@pytest.mark.parametrize("shape", [(1, 1, 2), (2, 3, 7), (1, 5, 32), (3, 7, 33), (2, 40, 128), (1, 9, 257), (2, 33, 512),
                                   (1, 6, 1000), (2, 3, 2048)])
@pytest.mark.parametrize("bias", [True, False])
def test_outputs_and_gradients(cuda_device, types, shape, bias):
    compare(*make(shape, shape[-1:], *types, bias=bias, seed=sum(shape)), cuda_device)


@pytest.mark.parametrize("width", [3001, 4096, 5000, 8192, 8191])
def test_wide_rows(cuda_device, width):
    for types in ((F32, F32), (BF16, BF16)):
        compare(*make((1, 5, width), (width,), *types, seed=width), cuda_device)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("width", [1025, 1032, 1155, 1500, 1536, 1537, 2304, 2500, 2561, 4104, 5121, 6136, 6145, 8001])
def test_rows_of_several_warps(cuda_device, types, width):
    """Every number of warps, with rows enough that a team takes several."""

    compare(*make((2, 400, width), (width,), *types, seed=width), cuda_device)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("shape", [(2, 3, 1, 16), (2, 5, 2, 64), (3, 700, 14, 64), (1, 900, 9, 33), (2, 50, 17, 8), (1, 40, 300, 24),
                                   (1, 30, 5, 512), (2, 21, 3, 1500), (5, 1, 12, 77)])
@pytest.mark.parametrize("bias", [True, False])
def test_a_weight_for_each_head(cuda_device, types, shape, bias):
    compare(*make(shape, shape[-2:], *types, bias=bias, seed=sum(shape)), cuda_device)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("shape", [(2, 3001, 64), (3, 900, 256), (1, 2000, 896), (2, 500, 1600), (1, 400, 8192), (2, 3001, 61)])
def test_teams_that_take_several_rows(cuda_device, types, shape):
    compare(*make(shape, shape[-1:], *types, seed=8), cuda_device)


@pytest.mark.parametrize("heads", [None, 6])
def test_strides(cuda_device, heads):
    """Slices of a wider tensor, batch items apart, steps backward or shared, channels that are not adjacent."""

    shape = (3, 50, 40) if heads is None else (3, 50, heads, 40)
    x, w, b, dy = make(shape, shape[2:], F32, F32, seed=2)
    places = [
        lambda t: torch.cat((t, torch.full_like(t[:, :3], float("nan"))), 1).to(cuda_device)[:, :-3],
        lambda t: torch.cat((torch.full_like(t[..., :5], float("nan")), t), -1).to(cuda_device)[..., 5:],
        lambda t: t.transpose(0, 1).contiguous().to(cuda_device).transpose(0, 1),
        lambda t: t.transpose(1, -1).contiguous().to(cuda_device).transpose(1, -1),
    ]
    for place in places:
        compare(x, w, b, dy, cuda_device, place=place)
    mine = x.to(cuda_device)
    one = mine[:, :1].expand(shape)  # a step that all share
    want = layer_norm(one.contiguous(), w.to(cuda_device), b.to(cuda_device))
    assert torch.equal(layer_norm(one, w.to(cuda_device), b.to(cuda_device)), want)
    # a gradient that is broadcast
    leaf = mine.requires_grad_(True)
    y = layer_norm(leaf, w.to(cuda_device), b.to(cuda_device))
    got, = torch.autograd.grad(y.sum(), leaf, retain_graph=True)
    assert torch.equal(got, torch.autograd.grad(y, leaf, torch.ones_like(y))[0])


@pytest.mark.parametrize("dims", [1, 2, 5])
def test_other_numbers_of_dimensions(cuda_device, dims):
    shape = (2, 3, 2, 5, 24)[5 - dims:]
    compare(*make(shape, (24,), F32, F32, seed=dims), cuda_device)
    if dims >= 2:
        compare(*make(shape, shape[-2:], F32, F32, seed=dims), cuda_device)


def test_rows_without_spread_and_large_means(cuda_device):
    """Rows of one value (the eps alone), a single channel, and a mean a thousand deviations off, whose own rounding
    (20 roundings of 1500 deviations) is what the result may then be off by."""

    x, w, b, dy = make((2, 6, 64), (64,), F32, F32, seed=6)
    x[0, 0], x[0, 1] = 0.0, 2.0
    y = layer_norm(x.to(cuda_device), w.to(cuda_device), b.to(cuda_device))
    R.close(y[0, :2], b.double().expand(2, 64), TOL, "a row of one value")
    one = layer_norm(x[..., :1].to(cuda_device), w[:1].to(cuda_device), b[:1].to(cuda_device))
    assert torch.equal(one.cpu(), b[:1].expand(2, 6, 1))
    far = make((2, 6, 64), (64,), F32, F32, seed=7, offset=1500.0)
    y = layer_norm(*[t.to(cuda_device) for t in far[:3]])
    R.close(y, definition(*[t.double() for t in far[:3]], 1e-5), 20 * 6e-8 * 1500, "far from zero")
    big = make((2, 6, 64), (64,), F32, F32, seed=9)
    big[0].mul_(1e15)
    compare(*big, cuda_device)
    small = make((2, 6, 64), (64,), F32, F32, seed=9)
    small[0].mul_(1e-18)
    compare(*small, cuda_device, eps=0.0)


def test_not_a_number_stays_in_its_row(cuda_device):
    x, w, b, dy = (t.to(cuda_device) for t in make((1, 4, 48), (48,), F32, F32, seed=8))
    for bad in (float("nan"), float("inf")):
        x[0, 2, 5] = bad
        y = layer_norm(x, w, b)
        assert torch.isnan(y[0, 2]).all() and torch.isfinite(y[0, [0, 1, 3]]).all()


def test_the_same_every_time_and_a_captured_step(cuda_device):
    x, w, b, dy = (t.to(cuda_device) for t in make((4, 700, 6, 48), (6, 48), BF16, BF16, seed=1))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y = layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]  # (no graph of these leaves outlives the step)

    want = step()
    for a, e in zip(step(), want):
        assert torch.equal(a, e)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.mul_(-2.0)
    graph.replay()
    again = step()
    for a, e in zip(out, again):
        assert torch.equal(a, e)


def test_two_streams_at_once(cuda_device):
    inputs = [[t.to(cuda_device) for t in make((3, 900, 6, 48), (6, 48), BF16, BF16, seed=s)] for s in (5, 6)]

    def step(x, w, b, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = [step(*t) for t in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in inputs], []
    for t, stream in zip(inputs, streams):
        with torch.cuda.stream(stream):
            got.append([step(*t) for _ in range(10)])
    torch.cuda.synchronize()
    for runs, e in zip(got, want):
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(run, e))


def test_offsets_past_32_bits(cuda_device):
    """The last rows of more than 2^31 elements, and rows 2^31 elements and more apart, are what they are alone."""

    rows, width = (1 << 24) + 77, 128
    w, b = (torch.linspace(0.5, 1.5, width, device=cuda_device, requires_grad=True) for _ in range(2))
    x = torch.randn(1, rows, width, device=cuda_device, dtype=BF16).requires_grad_(True)
    y = layer_norm(x, w, b)
    dy = torch.zeros_like(y)
    tail = x.detach()[:, -50:].clone().requires_grad_(True)
    want = layer_norm(tail, w, b)
    assert torch.equal(y[:, -50:], want)
    dy[:, -50:] = 1 + torch.arange(width, device=cuda_device) % 3
    got = torch.autograd.grad(y, (x, w, b), dy)
    alone = torch.autograd.grad(want, (tail, w, b), dy[:, -50:].clone())
    assert torch.equal(got[0][:, -50:], alone[0]) and not got[0][:, :-50].any()
    for a, e in zip(got[1:], alone[1:]):
        R.close(a, e.double(), VTOL, "vectors")
    del x, y, dy, got
    far = torch.zeros((1 << 32) + 4096, device=cuda_device, dtype=BF16)
    for strides in (((1 << 32), 64, 1), (1024, 1 << 31, 1)):
        view = torch.as_strided(far, (2, 3, 64) if strides[1] == 64 else (4, 3, 64), strides)
        dense = torch.randn(view.shape, device=cuda_device, dtype=BF16)
        view.copy_(dense)
        assert torch.equal(layer_norm(view, w.detach()[:64], b.detach()[:64]), layer_norm(dense, w.detach()[:64], b.detach()[:64]))


def test_no_rows(cuda_device):
    for shape in ((0, 4, 8), (2, 0, 8), (2, 3, 0)):
        x = torch.zeros(shape, device=cuda_device, requires_grad=True)
        w = torch.ones(shape[-1], device=cuda_device, requires_grad=True)
        y = layer_norm(x, w)
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == x.shape and dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))


def test_module(cuda_device):
    for heads, shape in ((None, (2, 5, 24)), (4, (2, 5, 4, 24))):
        module = LayerNormCuda(24, heads=heads).to(cuda_device)
        x = torch.randn(shape, device=cuda_device)
        with torch.no_grad():
            module.weight.add_(torch.randn_like(module.weight))
        assert torch.equal(module(x), layer_norm(x, module.weight, module.bias))
        half = module.half()
        y = half(x.half())
        y.float().sum().backward()
        assert y.dtype == F16 and half.weight.grad.dtype == F16 and half.weight.grad.shape == half.weight.shape
    assert LayerNormCuda(8, bias=False).bias is None


def test_refusals(cuda_device):
    x, w = torch.zeros(2, 3, 8, device=cuda_device), torch.ones(8, device=cuda_device)
    for bad in (lambda: layer_norm(x, w.cpu()), lambda: layer_norm(x.double(), w), lambda: layer_norm(x, w.half()),
                lambda: layer_norm(x.half(), w, dtype=F32), lambda: layer_norm(x.half(), w, dtype=BF16),
                lambda: layer_norm(x, w, dtype=torch.float64), lambda: layer_norm(x, w, w.half()),
                lambda: layer_norm(torch.zeros(1, 8193, device=cuda_device), torch.ones(8193, device=cuda_device))):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: layer_norm(x, w[:7]), lambda: layer_norm(x, w, w[:7]), lambda: layer_norm(x, w, eps=-1.0),
                lambda: layer_norm(x, torch.ones(4, 8, device=cuda_device)),
                lambda: layer_norm(x, torch.ones((), device=cuda_device))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        layer_norm(None, w)
    leaf = x.requires_grad_(True)
    y = layer_norm(leaf, w)
    g, = torch.autograd.grad(y.sum(), leaf, create_graph=False, retain_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
    import torch.autograd.forward_ad as fw

    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        layer_norm(fw.make_dual(x.detach(), torch.ones_like(x)), w)
