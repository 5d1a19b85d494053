"""The gated linear recurrence against its definition in 64 bits.

Bounds.  Gates are evaluated to a few units in the last place and the
recurrence rounds once a step: over a memory of 1 / (1 - a) <= 2000 steps that
accumulates like a random walk to 45 * 6e-8 = 3e-6 of the values met, and the
backward passes through two such scans: TOL is seven times the one, GTOL three
times that."""

import pytest
import torch

import train_reference as R
from triton_pesq_b200 import GatedScanCuda, _lib, gated_scan

pytestmark = pytest.mark.gpu

TOL, GTOL = 2e-5, 6e-5
NAMES = ("x", "input_gate", "decay_gate", "decay", "state")


def inputs(batch, steps, width, dtype, seed=0, state=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(batch, steps, width, generator=g).to(dtype)
    ig = (2 * torch.randn(batch, steps, width, generator=g)).to(dtype)
    rg = (2 * torch.randn(batch, steps, width, generator=g)).to(dtype)
    a = 0.9 + 0.099 * torch.rand(width, generator=g)
    decay = torch.log(torch.expm1(-torch.log(a) / 8))
    s = torch.randn(batch, width, generator=g) if state else None
    dy = torch.randn(batch, steps, width, generator=g).to(dtype)
    dlast = torch.randn(batch, width, generator=g)
    return [x, ig, rg, decay, s], dy, dlast


def compare(tensors, dy, dlast, device, reset=None, lengths=None, reverse=False, rate=8.0):
    """Outputs and all gradients, on the device and in 64 bits; the padded
    steps of the device's inputs hold NaN."""

    mine = [None if t is None else t.to(device) for t in tensors]
    if lengths is not None:
        pad = torch.arange(dy.shape[1])[None, :] >= lengths[:, None]
        for k in range(3):
            mine[k] = mine[k].clone()
            mine[k][pad.to(device)] = float("nan")
    mine = [None if t is None else t.requires_grad_(True) for t in mine]
    on = lambda t: None if t is None else t.to(device)  # noqa: E731
    y, last = gated_scan(*mine, reset=on(reset), lengths=on(lengths), reverse=reverse, rate=rate)
    leaves = [t for t in mine if t is not None]
    ddy = dy.to(device)
    if lengths is not None:
        ddy[pad.to(device)] = float("nan")
    got = torch.autograd.grad((y, last), leaves, (ddy, dlast.to(device)))

    wide = [None if t is None else t.double().requires_grad_(True) for t in tensors]
    wy, wl = R.gated_scan(*wide, reset, lengths, reverse, rate)
    want = torch.autograd.grad((wy, wl), [t for t in wide if t is not None], (dy.double(), dlast.double()),
                               allow_unused=True)
    assert y.dtype == tensors[0].dtype and last.dtype == torch.float32
    R.close(y, wy, TOL, "y")
    R.close(last, wl, TOL, "last")
    for name, g, w, t in zip([n for n, t in zip(NAMES, tensors) if t is not None], got, want, leaves):
        assert g.dtype == t.dtype
        R.close(g, torch.zeros(g.shape, dtype=torch.float64) if w is None else w, GTOL, "d " + name)
    assert _lib.gated_scan_check() == 0


SHAPES = [(1, 1, 1), (3, 1, 70), (2, 2, 33), (2, 8, 64), (1, 9, 66), (2, 64, 31), (1, 65, 129), (3, 130, 40),
          (1, 333, 2), (2, 1000, 96)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("reverse", [False, True])
def test_outputs_and_gradients(cuda_device, dtype, shape, reverse):
    tensors, dy, dlast = inputs(*shape, dtype, seed=sum(shape), state=shape[0] != 1)
    compare(tensors, dy, dlast, cuda_device, reverse=reverse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steps", [1, 7, 64, 200])
@pytest.mark.parametrize("reverse", [False, True])
def test_resets(cuda_device, dtype, steps, reverse):
    tensors, dy, dlast = inputs(4, steps, 50, dtype, seed=steps)
    reset = torch.rand(4, steps, generator=torch.Generator().manual_seed(1)) < 0.1
    reset[0] = True
    reset[1] = False
    reset[2, 0] = True
    reset[2, -1] = True
    compare(tensors, dy, dlast, cuda_device, reset=reset, reverse=reverse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("steps", [1, 6, 130])
@pytest.mark.parametrize("reverse", [False, True])
def test_lengths_with_nan_in_the_padding(cuda_device, dtype, steps, reverse):
    lengths = torch.tensor([0, 1, steps, steps // 2, steps - 1])
    tensors, dy, dlast = inputs(5, steps, 34, dtype, seed=steps + 1)
    reset = torch.rand(5, steps, generator=torch.Generator().manual_seed(2)) < 0.05
    compare(tensors, dy, dlast, cuda_device, lengths=lengths, reverse=reverse)
    compare(tensors, dy, dlast, cuda_device, lengths=lengths, reset=reset, reverse=reverse)


# every way through the rows: whole rows of single channels and of pairs, by boxes and by lanes; rows cut in
# both directions or in the backward alone; rows of one CTA; many single steps
WAYS = [((100, 40, 512), torch.float32), ((230, 33, 512), torch.bfloat16), ((100, 20, 1202), torch.float32),
        ((100, 20, 1202), torch.float16), ((30, 50, 448), torch.float32), ((50, 150, 416), torch.bfloat16),
        ((50, 100, 401), torch.float16), ((3, 700, 128), torch.float32), ((3, 700, 128), torch.bfloat16),
        ((9, 500, 72), torch.bfloat16), ((80, 1, 4096), torch.float32), ((100, 1, 1601), torch.bfloat16)]


@pytest.mark.parametrize("shape, dtype", WAYS)
@pytest.mark.parametrize("masks, reverse", [(False, False), (True, False), (True, True)])
def test_ways_through_the_rows(cuda_device, shape, dtype, masks, reverse):
    batch, steps, _ = shape
    tensors, dy, dlast = inputs(*shape, dtype, seed=sum(shape))
    lengths = reset = None
    if masks:
        g = torch.Generator().manual_seed(3)
        lengths = torch.randint(0, steps + 1, (batch,), generator=g)
        reset = torch.rand(batch, steps, generator=g) < 0.02
    compare(tensors, dy, dlast, cuda_device, lengths=lengths, reset=reset, reverse=reverse)


def test_lengths_beyond_the_row_and_below_zero(cuda_device):
    tensors, _, _ = inputs(2, 20, 8, torch.float32)
    dev = [t.to(cuda_device) for t in tensors]
    y, last = gated_scan(*dev, lengths=torch.tensor([500, -3], device=cuda_device, dtype=torch.int32))
    full, fl = gated_scan(*dev)
    assert torch.equal(y[0], full[0]) and torch.equal(last[0], fl[0])
    assert not y[1].any() and torch.equal(last[1], dev[4][1])


def test_a_reset_drops_a_state_that_is_not_finite(cuda_device):
    for steps in (3, 300):
        tensors, _, _ = inputs(1, steps, 40, torch.float32)
        dev = [t.to(cuda_device) for t in tensors]
        dev[0][0, 0] = float("nan")
        reset = torch.zeros(1, steps, dtype=torch.bool, device=cuda_device)
        reset[0, 2] = True
        y, last = gated_scan(*dev, reset=reset)
        assert torch.isnan(y[0, :2]).all() and torch.isfinite(y[0, 2:]).all() and torch.isfinite(last).all()


def test_extreme_logits(cuda_device):
    """Saturated gates: an open decay gate of a fast channel (a = 0), a shut
    one (a = 1, beta = 0 and no gradient through it), shut input gates."""

    batch, steps, width = 1, 70, 64
    x = torch.randn(batch, steps, width, generator=torch.Generator().manual_seed(4))
    rg, ig = torch.zeros(batch, steps, width), torch.zeros(batch, steps, width)
    rg[..., :16], rg[..., 16:32] = 200.0, -200.0
    ig[..., ::2], ig[..., 1::4] = 300.0, -300.0
    decay = torch.linspace(-30, 30, width)
    tensors = [x, ig, rg, decay, torch.randn(batch, width, generator=torch.Generator().manual_seed(5))]
    compare(tensors, torch.ones(batch, steps, width), torch.ones(batch, width), cuda_device)


def test_not_a_number_stays_visible(cuda_device):
    tensors, _, _ = inputs(1, 5, 6, torch.float32)
    for k in range(3):
        dev = [t.to(cuda_device) for t in tensors]
        dev[k][0, 1, 2] = float("nan")
        y, last = gated_scan(*dev)
        assert torch.isnan(y[0, 1:, 2]).all() and torch.isnan(last[0, 2])
        assert torch.isfinite(y[0, 0]).all() and torch.isfinite(y[..., :2]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(cuda_device, dtype):
    """Slices of one projection, rows of a longer buffer, every second step,
    a time-major tensor, channels that are not adjacent, one gate for all rows."""

    (x, ig, rg, decay, state), dy, dlast = inputs(3, 90, 64, dtype, seed=9)
    dev = [t.to(cuda_device) for t in (x, ig, rg, decay, state)]
    want, wl = gated_scan(*dev)

    packed = torch.cat(dev[:3], dim=2).chunk(3, dim=2)
    odd = torch.zeros(3, 91, 193, dtype=dtype, device=cuda_device)
    odd[:, 1:, 1:65], odd[:, 1:, 65:129], odd[:, 1:, 129:] = dev[:3]
    sliced = [odd[:, 1:, 1 + 64 * k:65 + 64 * k] for k in range(3)]
    twice = [t.repeat_interleave(2, dim=1)[:, ::2] for t in dev[:3]]
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in dev[:3]]
    apart = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in dev[:3]]
    for form in (packed, sliced, twice, major, apart):
        y, last = gated_scan(*form, *dev[3:])
        assert torch.equal(y, want) and torch.equal(last, wl)

    shared = dev[1][:1].expand(3, 90, 64).detach().requires_grad_(True)
    leaf = dev[1][:1].clone().requires_grad_(True)
    y, _ = gated_scan(dev[0], leaf.expand(3, 90, 64), dev[2], *dev[3:])
    (g,) = torch.autograd.grad(y, leaf, dy.to(cuda_device))
    z, _ = gated_scan(dev[0], shared, dev[2], *dev[3:])
    (full,) = torch.autograd.grad(z, shared, dy.to(cuda_device))
    assert torch.equal(y, z)
    R.close(g, full.double().sum(0, keepdim=True), 2.0**-7 if dtype == torch.bfloat16 else 1e-6, "shared gate")


def test_upstream_gradients_that_are_missing_or_broadcast(cuda_device):
    (x, ig, rg, decay, state), _, _ = inputs(2, 70, 20, torch.float32, seed=3)
    wide = [t.double().requires_grad_(True) for t in (x, ig, rg, decay, state)]
    dev = [t.to(cuda_device).requires_grad_(True) for t in (x, ig, rg, decay, state)]
    for pick in (0, 1):
        got = torch.autograd.grad(gated_scan(*dev)[pick].sum(), dev)
        want = torch.autograd.grad(R.gated_scan(*wide)[pick].sum(), wide)
        for n, g, w in zip(NAMES, got, want):
            R.close(g, w, GTOL, f"d {n} of output {pick}")


def test_gradient_against_differences(cuda_device):
    """Central differences of a weighted sum of the outputs along a random
    direction.  Step 1e-2: the third derivative leaves about 1e-4 relative, the
    32-bit forward's error 3e-6 / 1e-2 = 3e-4 of the outputs' norm over the
    derivative: 1 % is allowed."""

    (x, ig, rg, decay, state), dy, dlast = inputs(2, 150, 24, torch.float32, seed=6)
    dev = [t.to(cuda_device) for t in (x, ig, rg, decay, state)]
    dy, dlast = dy.to(cuda_device), dlast.to(cuda_device)
    g = torch.Generator(cuda_device).manual_seed(7)

    def value(ts):
        y, last = gated_scan(*ts)
        return float((y.double() * dy).sum() + (last.double() * dlast).sum())

    leaves = [t.clone().requires_grad_(True) for t in dev]
    y, last = gated_scan(*leaves)
    grads = torch.autograd.grad((y, last), leaves, (dy, dlast))
    for k in range(5):
        way = grads[k] + grads[k].norm() / grads[k].numel() ** 0.5 * torch.randn(dev[k].shape, device=cuda_device,
                                                                                 generator=g)
        way = way / way.abs().max()
        up, down = list(dev), list(dev)
        up[k], down[k] = dev[k] + 1e-2 * way, dev[k] - 1e-2 * way
        slope = (value(up) - value(down)) / 2e-2
        want = float((grads[k].double() * way).sum())
        assert abs(slope - want) <= 1e-2 * abs(want), f"{NAMES[k]}: {slope} against {want}"


def test_pieces_and_single_steps_continue_a_sequence(cuda_device):
    (x, ig, rg, decay, state), _, _ = inputs(2, 150, 48, torch.float32, seed=8)
    dev = [t.to(cuda_device) for t in (x, ig, rg, decay, state)]
    want, wl = gated_scan(*dev)
    s, parts = dev[4], []
    for lo, hi in ((0, 1), (1, 2), (2, 70), (70, 70), (70, 79), (79, 150)):
        y, s = gated_scan(*[t[:, lo:hi] for t in dev[:3]], dev[3], s)
        parts.append(y)
    R.close(torch.cat(parts, dim=1), want.double(), TOL, "pieces")
    R.close(s, wl.double(), TOL, "state")
    module = GatedScanCuda(48).to(cuda_device)
    module.decay.data.copy_(dev[3])
    s = dev[4]
    with torch.no_grad():
        for t in range(5):
            y, s = module.step(dev[0][:, t], dev[1][:, t], dev[2][:, t], s)
            R.close(y, want[:, t].double(), TOL, "step")
    assert module.check_errors() == 0


def test_empty_sizes(cuda_device):
    for shape in ((0, 5, 4), (2, 0, 4), (2, 5, 0)):
        tensors, _, _ = inputs(*shape, torch.float32)
        dev = [t.to(cuda_device).requires_grad_(True) for t in tensors]
        y, last = gated_scan(*dev)
        assert y.shape == shape and torch.equal(last, dev[4])
        grads = torch.autograd.grad(y.sum() + 2 * last.sum(), dev)
        assert torch.equal(grads[4], torch.full_like(dev[4], 2.0)) and not grads[3].any()
    y, last = gated_scan(*dev[:4])
    assert not last.any()


def test_long_rows_give_the_same_bits_every_time(cuda_device):
    """A row long enough to be cut into strips."""

    tensors, dy, dlast = inputs(1, 20000, 40, torch.float32, seed=12)
    dev = [t.to(cuda_device).requires_grad_(True) for t in tensors]

    def once():
        y, last = gated_scan(*dev)
        return (y, last, *torch.autograd.grad((y, last), dev, (dy.to(cuda_device), dlast.to(cuda_device))))

    first = once()
    for _ in range(5):
        for a, b in zip(once(), first):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits(cuda_device):
    """An output of more than 2**31 elements, and inputs that far apart."""

    batch, steps, width = 33000, 64, 1040
    (x, ig, rg, decay, _), _, _ = inputs(1, steps, width, torch.bfloat16, seed=14)
    dev = [t.to(cuda_device).expand(batch, steps, width) for t in (x, ig, rg)]
    y, last = gated_scan(*dev, decay.to(cuda_device))
    one, _ = gated_scan(*[t[:1] for t in dev], decay.to(cuda_device))
    assert y.numel() > 2**31
    for b in (0, batch // 2, batch - 1):
        assert torch.equal(y[b], one[0])
    del y, last
    far = torch.zeros(2**31 + steps * width, dtype=torch.bfloat16, device=cuda_device)
    rows = far.as_strided((2, steps, width), (2**31, width, 1))
    rows.copy_(dev[0][:2])
    z, _ = gated_scan(rows, dev[1][:2], dev[2][:2], decay.to(cuda_device))
    assert torch.equal(z[1], one[0]) and torch.equal(z[0], one[0])


def test_other_streams_and_graphs(cuda_device):
    tensors, dy, dlast = inputs(2, 300, 64, torch.float32, seed=15)
    dev = [t.to(cuda_device).requires_grad_(True) for t in tensors]
    dy, dlast = dy.to(cuda_device), dlast.to(cuda_device)

    def once():
        leaves = [t.detach().requires_grad_(True) for t in dev]  # (whose gradients come in on this stream)
        y, last = gated_scan(*leaves)
        return (y, last, *torch.autograd.grad((y, last), leaves, (dy, dlast)))

    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
        once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    with torch.no_grad():
        dev[0].mul_(2)
    again = once()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(held, again):
        assert torch.equal(a, b)


def test_threads_that_have_not_used_the_device(cuda_device):
    """The backward of a first pass runs on such a thread of autograd's."""

    import threading

    tensors, _, _ = inputs(2, 100, 64, torch.bfloat16, seed=16)
    dev = [t.to(cuda_device) for t in tensors]
    want, got = gated_scan(*dev)[0], []
    thread = threading.Thread(target=lambda: got.append(gated_scan(*dev)[0]))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert len(got) == 1 and torch.equal(got[0], want)


def test_refusals(cuda_device):
    tensors, _, _ = inputs(2, 4, 6, torch.float32)
    x, ig, rg, decay, state = (t.to(cuda_device) for t in tensors)
    with pytest.raises(TypeError):
        gated_scan([1.0], ig, rg, decay)
    for bad in (x[0], x.double(), x.cpu()):
        with pytest.raises(RuntimeError):
            gated_scan(bad, ig, rg, decay)
    with pytest.raises(RuntimeError):
        gated_scan(x, ig.bfloat16(), rg, decay)
    with pytest.raises(RuntimeError):
        gated_scan(x, ig, rg.cpu(), decay)
    with pytest.raises(RuntimeError):
        gated_scan(x, ig, rg, decay.half())
    with pytest.raises(RuntimeError):
        gated_scan(x, ig, rg, decay, state.double())
    with pytest.raises(RuntimeError):
        gated_scan(x, ig, rg, decay, reset=torch.zeros(2, 4, device=cuda_device))
    with pytest.raises(RuntimeError):
        gated_scan(x, ig, rg, decay, lengths=torch.zeros(2, device=cuda_device))
    for kw in ({"state": state[:1]}, {"reset": torch.zeros(2, 5, device=cuda_device, dtype=torch.bool)},
               {"lengths": torch.zeros(3, device=cuda_device, dtype=torch.int64)}, {"rate": 0.0}, {"rate": -1.0},
               {"rate": float("nan")}):
        with pytest.raises(ValueError):
            gated_scan(x, ig, rg, decay, **kw)
    with pytest.raises(ValueError):
        gated_scan(x, ig[:, :3], rg, decay)
    with pytest.raises(ValueError):
        gated_scan(x, ig, rg, decay[:3])
    x.requires_grad_(True)
    y, _ = gated_scan(x, ig, rg, decay)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dense_first", [False, True])
def test_saved_streams_that_come_back_in_another_layout(cuda_device, dtype, dense_first):
    """Hooks on what autograd saves (offloading, say) may hand the backward
    tensors of other strides than the forward's."""

    def strided(t):
        out = torch.empty(t.shape[0], t.shape[1], t.shape[2] + 1, dtype=t.dtype, device=t.device)[..., 1:]
        return out.copy_(t)

    tensors, dy, dlast = inputs(2, 90, 64, dtype, seed=6)
    dev = [t.to(cuda_device) for t in tensors]
    relay = strided if dense_first else torch.Tensor.contiguous
    if not dense_first:
        dev[:3] = [strided(t) for t in dev[:3]]
    dev = [t.requires_grad_(True) for t in dev]
    streams = lambda t: t.dim() == 3 and t.dtype == dtype  # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), lambda t: relay(t) if streams(t) else t):
        y, last = gated_scan(*dev)
    got = torch.autograd.grad((y, last), dev, (dy.to(cuda_device), dlast.to(cuda_device)))
    wide = [t.double().requires_grad_(True) for t in tensors]
    wy, wl = R.gated_scan(*wide, None, None, False, 8.0)
    want = torch.autograd.grad((wy, wl), wide, (dy.double(), dlast.double()))
    for name, g, w in zip(NAMES, got, want):
        R.close(g, w, GTOL, "d " + name)


@pytest.mark.parametrize("steps", [90, 300, 1000])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dense_first", [False, True])
def test_saved_streams_in_another_layout_with_lengths(cuda_device, steps, reverse, dense_first):
    """The states that the forward keeps serve a backward of any layout, wherever the rows end: the same bits as
    with one layout in both."""

    def strided(t):
        out = torch.empty(t.shape[0], t.shape[1], t.shape[2] + 1, dtype=t.dtype, device=t.device)[..., 1:]
        return out.copy_(t)

    lengths = torch.tensor([0, 1, 7, 8, 9, 15, 16, 17, 23, 24, 25, 31, 32, 33, 63, steps - 9, steps - 8, steps - 1, steps])
    tensors, dy, dlast = inputs(len(lengths), steps, 64, torch.float32, seed=7)
    dev, dy, dlast = [t.to(cuda_device) for t in tensors], dy.to(cuda_device), dlast.to(cuda_device)
    first, then = (torch.Tensor.contiguous, strided) if dense_first else (strided, torch.Tensor.contiguous)

    def call(at_first, later):
        leaves = [(at_first(t) if t.dim() == 3 else t).detach().requires_grad_(True) for t in dev]
        relay = lambda t: later(t) if t.dim() == 3 else t  # noqa: E731
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), relay):
            y, last = gated_scan(*leaves, lengths=lengths.to(cuda_device), reverse=reverse)
        return torch.autograd.grad((y, last), leaves, (dy, dlast))

    want = call(then, then)
    # states of a forward of which nothing is known
    lasts = (*[first(t) for t in dev[:3]], *dev[3:], None, lengths.to(cuda_device), reverse, 8.0)
    _, _, kept = torch.ops.pesq_cuda.gated_scan_forward(*lasts, True)
    laters = (*[then(t) for t in dev[:3]], *lasts[3:])
    for a, b in zip(torch.ops.pesq_cuda.gated_scan_backward(*laters, kept, 0, dy, dlast), want):
        R.close(a, b.double(), 1e-5, "of an unknown forward")
    for name, a, b in zip(NAMES, call(first, then), want):
        if name == "decay":  # (a sum over strips, whose number is the layout's)
            R.close(a, b.double(), 1e-5, name)
        else:
            R.close(a, b.double(), 1e-6, name)
