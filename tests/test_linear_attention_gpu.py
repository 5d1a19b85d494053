"""The linear attention against its definition in 64 bits, step by step, with gradients by autograd.

Bounds.  Sums are 32 bits: a chunk's products over up to 128 channels or 64 steps, and the carried state, whose
roundings decay with it (a head that forgets by 0.998 a step holds some 500 of them): under 600 roundings of 6e-8 of random
sign, 25 * 6e-8.  What is computed goes through the matrix instructions in two terms: 2^-17 off beside bfloat16 inputs
(a product of two such factors twice that), 2^-21 otherwise; of random sign again, but bounded here as if it were not.
That makes TOL, relative to the largest value of the output (`close` adds the rounding to 16 bits).  A decay's gradient
sums products of two outputs over a chunk's or a row's steps; its terms are larger than it: DTOL, ten times that, of the largest
value of the steps' gradients."""

import pytest
import torch

import train_reference as R
from triton_pesq_b200 import LinearAttentionCuda, linear_attention

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 5e-6, F16: 5e-6, BF16: 2e-5}
DTOL = {t: 10 * v for t, v in TOL.items()}


def definition(q, k, v, g, state=None, reset=None, lengths=None, reverse=False, scale=1.0):
    """S_t = exp(g_t) S_{t-1} + k_t v_t^T, y_t = scale S_t^T q_t, step by step."""

    batch, steps, heads, key = q.shape
    S = torch.zeros(batch, heads, key, v.shape[3], dtype=torch.float64) if state is None else state
    g = g.expand(batch, steps, heads) if g.dim() == 1 else g
    ys = [None] * steps
    for t in range(steps - 1, -1, -1) if reverse else range(steps):
        a = torch.exp(g[:, t])
        if reset is not None:
            a = torch.where(reset[:, t, None], 0.0, a)
        new = a[..., None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        y = scale * (q[:, t, :, None, :] @ new)[:, :, 0]
        if lengths is not None:
            live = t < lengths
            y = torch.where(live[:, None, None], y, 0.0)
            S = torch.where(live[:, None, None, None], new, S)
        else:
            S = new
        ys[t] = y
    return (torch.stack(ys, dim=1) if steps else v.clone()), S


def make(batch, steps, heads, key, value, dtype, gated=False, reset=False, lengths=False, state=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, dy = (torch.randn(batch, steps, heads, n, generator=g).to(dtype) for n in (key, key, value, value))
    if gated:
        decay = -torch.nn.functional.softplus(2 * torch.randn(batch, steps, heads, generator=g) - 2.0)
    else:
        decay = torch.log1p(-torch.exp2(-2.0 - 7.0 * torch.rand(heads, generator=g)))
    s = torch.randn(batch, heads, key, value, generator=g) if state else None
    dlast = torch.randn(batch, heads, key, value, generator=g)
    kw = {"scale": key**-0.5}
    if reset:
        kw["reset"] = torch.rand(batch, steps, generator=g) < 0.03
    if lengths:
        n = torch.randint(0, steps + 1, (batch,), generator=g)
        n[0] = 0
        if batch > 1:
            n[1] = steps
        kw["lengths"] = n
    return [q, k, v, decay, s], dy, dlast, kw


def on(device, kw):
    return {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}


def compare(tensors, dy, dlast, kw, device, place=None, reverse=False, train=True):
    place = place or (lambda t: t.to(device))
    dtype = tensors[0].dtype
    mine = [None if t is None else (place(t) if i < 3 else t.to(device)) for i, t in enumerate(tensors)]
    wide = [None if t is None else t.double() for t in tensors]
    if train:
        for t in (*mine, *wide):
            if t is not None:
                t.requires_grad_(True)
    y, last = linear_attention(*mine, **on(device, kw), reverse=reverse)
    wy, wlast = definition(*wide, **kw, reverse=reverse)
    assert y.dtype == dtype and last.dtype == F32
    R.close(y, wy, TOL[dtype], "y")
    R.close(last, wlast, TOL[dtype], "last")
    if not train:
        return
    leaves, wleaves = ([t for t in ts if t is not None] for ts in (mine, wide))
    got = torch.autograd.grad((y, last), leaves, (place(dy), dlast.to(device)))
    want = torch.autograd.grad((wy, wlast), wleaves, (dy.double(), dlast.double()))
    for name, a, e in zip(("q", "k", "v", "log_decay", "state"), got, want):
        assert a.dtype == (dtype if name in "qkv" else F32) and a.shape == e.shape
        terms = None
        if name == "log_decay":  # its terms: the state's products with its gradient, of key * value values each
            size = float(wlast.detach().abs().max()) * float(dlast.abs().max())
            terms = torch.full((1,), max(size, float(e.abs().max())) , dtype=torch.float64)
        R.close(a, e, DTOL[dtype] if name == "log_decay" else TOL[dtype] * 2, "d " + name, terms)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (2, 3, 2, 8, 8), (1, 16, 1, 16, 32), (2, 64, 3, 32, 32), (1, 65, 2, 33, 17),
                                   (2, 100, 2, 64, 64), (1, 200, 1, 48, 128), (1, 130, 2, 128, 40), (1, 129, 1, 128, 128),
                                   (1, 90, 3, 7, 5), (1, 77, 1, 96, 65)])
@pytest.mark.parametrize("gated", [False, True])
def test_outputs_and_gradients(cuda_device, dtype, shape, gated):
    compare(*make(*shape, dtype, gated=gated, seed=sum(shape)), cuda_device)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("masks", ["reset", "lengths", "both"])
def test_masks_and_directions(cuda_device, dtype, gated, reverse, masks):
    case = make(3, 150, 2, 24, 40, dtype, gated=gated, reset=masks != "lengths", lengths=masks != "reset", seed=5)
    compare(*case, cuda_device, reverse=reverse)
    case = make(3, 150, 2, 24, 40, dtype, gated=gated, reset=masks != "lengths", lengths=masks != "reset", seed=6, state=False)
    compare(*case, cuda_device, reverse=reverse, train=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1500, 1, 32, 32), (1, 2000, 2, 64, 48), (2, 1100, 1, 128, 128)])
@pytest.mark.parametrize("gated,reverse", [(False, False), (True, False), (True, True)])
def test_rows_in_parts(cuda_device, dtype, shape, gated, reverse):
    compare(*make(*shape, dtype, gated=gated, reset=gated, lengths=reverse, seed=9), cuda_device, reverse=reverse)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,gated,reverse", [((45, 390, 10, 16, 24), True, True), ((30, 400, 10, 24, 16), False, False),
                                                 ((23, 385, 10, 16, 72), True, False)])
def test_rows_left_over_from_full_rounds(cuda_device, dtype, shape, gated, reverse):
    """A few rows more than the device holds at once, of the forward, of the backward, and of two CTAs a row: cut, the others whole."""

    compare(*make(*shape, dtype, gated=gated, reset=gated, seed=10), cuda_device, reverse=reverse)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("steps", [1, 2, 7, 8, 9])
@pytest.mark.parametrize("widths", [(64, 64), (31, 33), (128, 100), (5, 3)])
def test_few_steps(cuda_device, dtype, steps, widths):
    for seed in range(2):
        case = make(3, steps, 2, *widths, dtype, gated=seed == 1, reset=seed == 1, lengths=seed == 1, seed=seed)
        compare(*case, cuda_device, train=False, reverse=seed == 1)
        compare(*case, cuda_device)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_stream_step_by_step_is_the_sequence(cuda_device, dtype):
    """Both forms against the definition; the state that one leaves is taken on by the other."""

    (q, k, v, g, s), _, _, kw = make(2, 90, 3, 32, 48, dtype, gated=True)
    wy, wlast = definition(*[t.double() for t in (q, k, v, g, s)], **kw)
    q, k, v, g, s = (t.to(cuda_device) for t in (q, k, v, g, s))
    ys, state = [], s
    for t in range(70):
        y, state = linear_attention(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], g[:, t:t + 1], state, **kw)
        ys.append(y)
    y, state = linear_attention(q[:, 70:], k[:, 70:], v[:, 70:], g[:, 70:], state, **kw)
    R.close(torch.cat([*ys, y], dim=1), wy, TOL[dtype], "y")
    R.close(state, wlast, TOL[dtype], "last")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_strides(cuda_device, dtype):
    """Slices of one projection, heads before steps, batch items apart, odd offsets, shared heads, not adjacent channels."""

    (q, k, v, g, s), dy, dlast, kw = make(2, 70, 3, 24, 24, dtype)
    places = [
        lambda t: torch.cat((t, torch.full_like(t, float("nan"))), 3).to(cuda_device)[..., :24],
        lambda t: t.transpose(1, 2).contiguous().to(cuda_device).transpose(1, 2),
        lambda t: torch.cat((torch.full_like(t[..., :1], float("nan")), t), 3).to(cuda_device)[..., 1:],
        lambda t: torch.cat((torch.full_like(t[..., :2], float("nan")), t), 3).to(cuda_device)[..., 2:],
        lambda t: t.transpose(1, 3).contiguous().to(cuda_device).transpose(1, 3),
        lambda t: t.flip(1).to(cuda_device).flip(1),
    ]
    for place in places:
        compare([q, k, v, g, s], dy, dlast, kw, cuda_device, place=place)
    # keys and values of one head for all, whose gradients torch sums
    leaves = [t.to(cuda_device).requires_grad_(True) for t in (q, k[:, :, :1], v[:, :, :1])]
    y, _ = linear_attention(leaves[0], leaves[1].expand(q.shape), leaves[2].expand(v.shape), g.to(cuda_device), **kw)
    got = torch.autograd.grad(y, leaves, dy.to(cuda_device))
    wide = [t.double().requires_grad_(True) for t in (q, k[:, :, :1], v[:, :, :1])]
    wy, _ = definition(wide[0], wide[1].expand(q.shape), wide[2].expand(v.shape), g.double(), **kw)
    want = torch.autograd.grad(wy, wide, dy.double())
    # (three gradients rounded to the type, then their sum)
    for a, e in zip(got, want):
        R.close(a, e, TOL[dtype] * 2 + 4 * R.ROUND[dtype], "a shared head's gradient")
    # and a gradient that is broadcast, or missing
    leaf = q.to(cuda_device).requires_grad_(True)
    y, last = linear_attention(leaf, k.to(cuda_device), v.to(cuda_device), g.to(cuda_device), **kw)
    a, = torch.autograd.grad(y.sum(), leaf, retain_graph=True)
    assert torch.equal(a, torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)[0])
    none, = torch.autograd.grad(last.sum(), leaf)
    assert torch.equal(none, torch.zeros_like(none))


def test_what_masks_hide_is_not_read(cuda_device):
    for dtype in (F32, BF16):
        (q, k, v, g, s), dy, dlast, kw = make(3, 140, 2, 32, 32, dtype, gated=True, lengths=True, seed=3)
        clean = [t.to(cuda_device) for t in (q, k, v, g, s, dy)]
        dirty = [t.clone() for t in clean]
        past = (torch.arange(140)[None] >= kw["lengths"][:, None]).to(cuda_device)
        for t in (*dirty[:4], dirty[5]):
            t[past] = float("nan")
        outs = []
        for t in (clean, dirty):
            leaves = [x.requires_grad_(True) for x in t[:5]]
            y, last = linear_attention(*leaves, **on(cuda_device, kw))
            outs.append([y.detach(), last.detach(), *torch.autograd.grad((y, last), leaves, (t[5], dlast.to(cuda_device)))])
        for a, e in zip(*outs):
            assert torch.equal(a, e)


def test_decays_at_their_limits(cuda_device):
    """No decay, decays of zero (as -inf and as far below zero), steps that decay by e^-50: and a state before that is not
    a number stays behind a reset."""

    for dtype in (F32, BF16, F16):
        (q, k, v, g, s), dy, dlast, kw = make(2, 150, 3, 32, 32, dtype, gated=True, seed=4)
        g[:, :, 0] = 0.0
        g[:, 5::31, 1] = float("-inf")
        g[:, 17::13, 1] = -1e30
        g[:, ::3, 2] = -50.0
        k, v = (0.3 * k.float()).to(dtype), (0.3 * v.float()).to(dtype)
        mine = [t.to(cuda_device).requires_grad_(True) for t in (q, k, v, g, s)]
        y, last = linear_attention(*mine, **kw)
        got = torch.autograd.grad((y, last), mine, (dy.to(cuda_device), dlast.to(cuda_device)))
        # (the same function of the decays' factors: autograd through exp(-inf) is 0 too)
        wide = [t.double().requires_grad_(True) for t in (q, k, v, g, s)]
        wy, wlast = definition(*wide, **kw)
        want = torch.autograd.grad((wy, wlast), wide, (dy.double(), dlast.double()))
        R.close(y, wy, TOL[dtype], "y")
        R.close(last, wlast, TOL[dtype], "last")
        for name, a, e in zip(("q", "k", "v", "log_decay", "state"), got, want):
            terms = None
            if name == "log_decay":
                terms = wlast.detach().abs().max().reshape(1) * dlast.abs().max()
                terms = torch.maximum(terms, e.abs().max())
            R.close(a, e, DTOL[dtype] if name == "log_decay" else 2 * TOL[dtype], "d " + name, terms)
    reset = torch.zeros(2, 150, dtype=torch.bool, device=cuda_device)
    reset[:, 0] = True
    bad = torch.full_like(s, float("nan")).to(cuda_device)
    with torch.no_grad():
        for n in (150, 4):
            args = [t.detach()[:, :n] for t in mine[:4]]
            y, last = linear_attention(*args, bad, reset=reset[:, :n], **kw)
            want = linear_attention(*args, reset=reset[:, :n], **kw)
            assert torch.equal(y, want[0]) and torch.equal(last, want[1])


def test_large_values_in_float16(cuda_device):
    """Products and states beyond float16's range, results within it."""

    (q, k, v, g, s), dy, dlast, kw = make(1, 100, 1, 64, 64, F16, state=False, seed=2)
    q, k, v = (200.0 * q.float()).half(), (200.0 * k.float()).half(), (1e-3 * v.float()).half()
    dy = (1e-3 * dy.float()).half()
    compare([q, k, v, g, None], dy, 1e-3 * dlast, {"scale": 0.05}, cuda_device)


def test_gradients_against_differences(cuda_device):
    """Central differences in 32 bits of a function that is smooth: steps of 2^-6, whose square times the third derivative (a few
    times the gradient's size here) is 1e-3 of it, and rounding of 1e-6 of the sum over 2^-6 less than that."""

    (q, k, v, g, s), dy, dlast, kw = make(1, 80, 1, 8, 8, F32, gated=True, reset=True, seed=11)
    base = [t.to(cuda_device) for t in (q, k, v, g, s)]
    dy, dlast, kw = dy.to(cuda_device), dlast.to(cuda_device), on(cuda_device, kw)

    def f(ts):
        y, last = linear_attention(*ts, **kw)
        return (y.double() * dy).sum() + (last.double() * dlast).sum()

    leaves = [t.clone().requires_grad_(True) for t in base]
    grads = torch.autograd.grad(f(leaves), leaves)
    gen = torch.Generator().manual_seed(1)
    for i, gr in enumerate(grads):
        move = torch.randn(base[i].shape, generator=gen).to(cuda_device)
        move /= move.norm()
        want = float((gr.double() * move).sum())
        with torch.no_grad():
            up, down = ([t + sgn * 2.0**-6 * move if j == i else t for j, t in enumerate(base)] for sgn in (1, -1))
            got = float(f(up) - f(down)) * 2.0**5
        assert abs(got - want) <= 5e-3 * float(gr.double().norm()), (i, got, want)


def test_the_same_every_time_and_a_captured_step(cuda_device):
    for shape in ((2, 300, 3, 64, 64), (1, 1000, 1, 32, 48)):
        (q, k, v, g, s), dy, dlast, kw = make(*shape, BF16, seed=1)
        leaves = [t.to(cuda_device).requires_grad_(True) for t in (q, k, v, g, s)]
        dy, dlast = dy.to(cuda_device), dlast.to(cuda_device)

        def step():
            y, last = linear_attention(*leaves, **kw)
            return [y.detach(), last.detach(), *torch.autograd.grad((y, last), leaves, (dy, dlast))]

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
            leaves[0].mul_(-2.0)
        graph.replay()
        for a, e in zip(out, step()):
            assert torch.equal(a, e)


def test_two_streams_at_once(cuda_device):
    cases = [make(1, 1300, 2, 64, 64, BF16, seed=i) for i in range(2)]
    inputs = [[t.to(cuda_device) for t in c[0]] for c in cases]
    want = [linear_attention(*t, **c[3]) for t, c in zip(inputs, cases)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], []
    for t, c, stream in zip(inputs, cases, streams):
        with torch.cuda.stream(stream):
            got.append(linear_attention(*t, **c[3]))
    torch.cuda.synchronize()
    for a, e in zip(got, want):
        assert torch.equal(a[0], e[0]) and torch.equal(a[1], e[1])


@pytest.mark.parametrize("shape", [(3, 400, 4, 64, 64), (2, 300, 2, 128, 100), (1, 1300, 2, 32, 16)])
def test_states_beside_bfloat16_are_of_32_bits(cuda_device, shape):
    """The last state and the first one's gradient, by their norm.  Three terms hold 24 bits, and a state is a chunk's sum (in
    four to eight pieces, each cut off at 2^-23 of it) and a decay a chunk: some ten roundings of random sign, 10**0.5 * 2^-23."""

    (q, k, v, decay, state), dy, dlast, kw = make(*shape, BF16, gated=True, seed=12)
    mine = [t.to(cuda_device) for t in (q, k, v, decay)]
    first, wide = state.to(cuda_device).requires_grad_(True), state.double().requires_grad_(True)
    y, last = linear_attention(*mine, first, **kw)
    wy, wlast = definition(*(t.double() for t in (q, k, v, decay)), wide, **kw)
    got = torch.autograd.grad((y, last), first, (dy.to(cuda_device), dlast.to(cuda_device)))[0]
    want = torch.autograd.grad((wy, wlast), wide, (dy.double(), dlast.double()))[0]
    for name, x, e in (("last", last, wlast), ("d state", got, want)):
        off = float((x.detach().cpu().double() - e).norm() / e.norm())
        assert off <= 10**0.5 * 2.0**-23, (name, off)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_offsets_past_32_bits(cuda_device, dtype):
    """The last steps of operands of more than 2^31 elements, and operands whose steps, heads and rows lie as far apart."""

    steps, heads, width, tail = (1 << 20) + 200, 32, 64, 300
    x = torch.randn(1, steps, heads, width, device=cuda_device, dtype=dtype) * 0.3
    decay = torch.linspace(-0.6, -0.4, heads, device=cuda_device)
    v = x.detach().requires_grad_(True)
    y, last = linear_attention(x, x, v, decay)
    # (what came 128 steps before is e^-51 of what it was)
    end = x[:, -tail:].cpu().double()
    wv = end.clone().requires_grad_(True)
    want, wlast = definition(end, end, wv, decay.cpu().double())
    R.close(y[:, -tail + 128:], want[:, 128:], TOL[dtype], "y")
    R.close(last, wlast, TOL[dtype], "last")
    dlast = torch.randn_like(last)
    got = torch.autograd.grad(last, v, dlast)[0]
    alone = torch.autograd.grad(wlast, wv, dlast.cpu().double())[0]
    R.close(got[:, -tail:], alone, TOL[dtype] * 2, "dv")
    assert not got[:, :1000].any()
    del x, v, y, got
    far = torch.zeros((1 << 32) + (1 << 14), device=cuda_device, dtype=dtype)
    for strides in ((1 << 32, 256, 64, 1), (1 << 13, 1 << 30, 64, 1), (1 << 13, 64, 1 << 31, 1)):
        shape = (2, 5 if strides[1] == 1 << 30 else 30, 3 if strides[2] == 1 << 31 else 2, 64)
        last_at = sum((n - 1) * s for n, s in zip(shape, strides))
        if last_at >= far.numel():
            shape = (2, 4, 2, 64)
        view = torch.as_strided(far, shape, strides)
        dense = torch.randn(shape, device=cuda_device, dtype=dtype)
        view.copy_(dense)
        decay = torch.linspace(-0.5, -0.1, shape[2], device=cuda_device)
        for n in (shape[1], 1):
            v, d = view[:, :n], dense[:, :n]
            for a, e in zip(linear_attention(v, v, v, decay), linear_attention(d, d, d, decay)):
                assert torch.equal(a, e)


def test_nothing_to_do(cuda_device):
    for shape in ((0, 4, 2, 8, 8), (2, 0, 2, 8, 8), (2, 3, 0, 8, 8), (2, 3, 2, 0, 8), (2, 3, 2, 8, 0)):
        (q, k, v, g, s), dy, dlast, kw = make(*shape[:3], max(shape[3], 1), max(shape[4], 1), F32)
        q, k, v, s = q[..., :shape[3]], k[..., :shape[3]], v[..., :shape[4]], s[:, :, :shape[3], :shape[4]]
        leaves = [t.to(cuda_device).requires_grad_(True) for t in (q, k, v, g, s)]
        y, last = linear_attention(*leaves)
        assert torch.equal(last, leaves[4]) and y.shape == v.shape and not y.any()
        grads = torch.autograd.grad(y.sum() + last.sum(), leaves)
        assert torch.equal(grads[4], torch.ones_like(grads[4])) and not any(x.any() for x in grads[:4])


def test_module(cuda_device):
    module = LinearAttentionCuda(3, 16).to(cuda_device)
    (q, k, v, _, s), _, _, kw = make(2, 40, 3, 16, 24, F32)
    q, k, v, s = (t.to(cuda_device) for t in (q, k, v, s))
    a = torch.exp(module.log_decay())
    assert torch.allclose(a[[0, -1]].cpu(), torch.tensor([0.875, 0.998]), atol=1e-6)
    y, last = module(q, k, v, s)
    want = linear_attention(q, k, v, module.log_decay(), s, scale=0.25)
    assert torch.equal(y, want[0]) and torch.equal(last, want[1])
    (y.sum() + last.sum()).backward()
    assert module.decay.grad.shape == (3,)
    with torch.no_grad():
        y1, last1 = module.step(q[:, 0], k[:, 0], v[:, 0], s)
        want = linear_attention(q[:, :1], k[:, :1], v[:, :1], module.log_decay(), s, scale=0.25)
    assert torch.equal(y1, want[0][:, 0]) and torch.equal(last1, want[1])


def test_refusals(cuda_device):
    (q, k, v, g, s), _, _, _ = make(2, 5, 3, 8, 12, F32)
    q, k, v, g, s = (t.to(cuda_device) for t in (q, k, v, g, s))
    wide = torch.zeros(1, 2, 1, 129, device=cuda_device)
    for bad in (lambda: linear_attention(q.double(), k.double(), v.double(), g), lambda: linear_attention(q, k.half(), v, g),
                lambda: linear_attention(q, k, v, g.half()), lambda: linear_attention(q, k, v, g, s.half()),
                lambda: linear_attention(q, k.cpu(), v, g), lambda: linear_attention(q[0], k[0], v[0], g),
                lambda: linear_attention(q, k, v, g, reset=torch.zeros(2, 5, device=cuda_device)),
                lambda: linear_attention(q, k, v, g, lengths=torch.zeros(2, device=cuda_device)),
                lambda: linear_attention(wide, wide, wide, g[:1])):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: linear_attention(q, k[:, :4], v, g), lambda: linear_attention(q, k, v[:, :, :2], g),
                lambda: linear_attention(q, k, v, g[:2]), lambda: linear_attention(q, k, v, g.expand(2, 4, 3)),
                lambda: linear_attention(q, k, v, g, s[:1]), lambda: linear_attention(q, k, v, g, scale=float("nan")),
                lambda: linear_attention(q, k, v, g, reset=torch.zeros(2, 4, dtype=torch.bool, device=cuda_device)),
                lambda: linear_attention(q, k, v, g, lengths=torch.zeros(3, dtype=torch.int64, device=cuda_device))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        linear_attention(None, k, v, g)
    leaf = q.requires_grad_(True)
    y, _ = linear_attention(leaf, k, v, g)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
    import torch.autograd.forward_ad as fw

    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        linear_attention(fw.make_dual(q.detach(), torch.ones_like(q)), k, v, g)
