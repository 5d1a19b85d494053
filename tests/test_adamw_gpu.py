"""The AdamW step against its definition in 64 bits.

Bounds.  A step is a dozen 32-bit operations on a value, the division and the
hyperparameters approximate to 2^-21: of the moments, 4 * 2^-24 of the two terms
that make them (which may cancel); of the parameter, one rounding of it plus 2^-19 of the update, which is at most
lr * (1 - b1) / sqrt(1 - b2) = 3.2 lr here (and 1 / sqrt(1 - b2) = 32 lr where an old
second moment is zero).  Over n steps these add up.  Eight bits: a value is within
half a step of float8 (1/16 of itself, or 2^-10 of the block's unit), a root within
a whole one."""

import pytest
import torch

import train_reference as R
from triton_pesq_b200 import AdamWCuda, adamw_step

pytestmark = pytest.mark.gpu

BLOCK = 256
SIZES = [(1,), (0,), (255,), (256,), (257,), (3, 5), (40, 33), (1000,), (129, 129), (2,)]


def build(sizes, device, bits=32, dtype=torch.float32, seed=0, shift=0, copies=False):
    """Parameters as views of a buffer (``shift`` values off its alignment), state after some steps."""

    g = torch.Generator().manual_seed(seed)
    numel = [torch.Size(s).numel() for s in sizes]
    padded = [-(-n // BLOCK) * BLOCK for n in numel]
    total = sum(padded)
    flat = torch.randn(total + shift, generator=g).to(device)
    at, params, grads, marks = 0, [], [], []
    for s, n, w in zip(sizes, numel, padded):
        params.append(flat[shift + at:shift + at + n].view(s))
        grads.append((1e-2 * torch.randn(s, generator=g)).to(dtype).to(device))
        marks.append(slice(at, at + n))
        at += w
    m, v = torch.zeros(total), torch.zeros(total)
    for k in marks:
        m[k] = 1e-3 * torch.randn(m[k].shape, generator=g)
        v[k] = (1e-2 * torch.randn(m[k].shape, generator=g)) ** 2
    out = {"params": params, "grads": grads, "marks": marks, "scales": None, "copies": None,
           "step": torch.tensor([4, 0], device=device)}
    if copies:
        out["copies"] = [p.to(dtype) for p in params]
    if bits == 32:
        out["m"], out["v"] = m.to(device), v.to(device)
    else:
        both = torch.stack([m, v.sqrt()]).view(2, -1, BLOCK)
        scales = both.abs().amax(2) / 448
        code = (both / scales.clamp_min(1e-30)[:, :, None]).to(torch.float8_e4m3fn).view(2, -1)
        out["m"], out["v"], out["scales"] = code[0].to(device), code[1].to(device), scales.to(device)
    return out


def run(s, **kw):
    adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], scales=s["scales"], copies=s["copies"], **kw)


def values(s):
    """The moments' values in 64 bits."""

    m, v = s["m"].cpu().double(), s["v"].cpu().double()
    if s["scales"] is not None:
        spread = s["scales"].cpu().double().repeat_interleave(BLOCK, dim=1)
        m, v = m * spread[0], (v * spread[1]) ** 2
    return m, v


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shift", [0, 1])
def test_one_step(cuda_device, bits, dtype, shift):
    copies = dtype != torch.float32
    s = build(SIZES, cuda_device, bits, dtype, seed=1, shift=shift, copies=copies)
    old = [p.cpu().double() for p in s["params"]]
    m0, v0 = values(s)
    kw = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
    run(s, **kw)
    m1, v1 = values(s)
    assert s["step"].tolist() == [5, 0]
    for i, k in enumerate(s["marks"]):
        if old[i].numel() == 0:
            continue
        g = s["grads"][i].cpu().double().reshape(-1)
        wp, wm, wv = R.adamw(old[i].reshape(-1), g, m0[k], v0[k], 5, 3e-3, (0.9, 0.99), 1e-6, 0.1)
        p = s["params"][i].cpu().double().reshape(-1)
        update = (wp - old[i].reshape(-1)).abs()
        assert ((p - wp).abs() <= 2.0**-23 * wp.abs() + 2.0**-19 * update).all()
        if copies:
            assert torch.equal(s["copies"][i], s["params"][i].to(dtype))
        if bits == 32:
            terms = 0.9 * m0[k].abs() + 0.1 * g.abs()
            for got, want, size in ((m1[k], wm, terms), (v1[k], wv, wv)):
                assert ((got - want).abs() <= 2.0**-22 * (size + 1e-3 * want.abs().max())).all()
        else:
            for got, want, share in ((m1[k], wm, 1 / 16), (v1[k].sqrt(), wv.sqrt(), 1 / 8)):
                n = want.numel()
                unit = torch.nn.functional.pad(want.abs(), (0, -n % BLOCK)).view(-1, BLOCK).amax(1) / 448
                unit = unit.repeat_interleave(BLOCK)[:n]
                allowed = torch.maximum(share * want.abs(), share * 2.0**-6 * unit) * 1.001
                assert ((got - want).abs() <= allowed).all()


def test_many_steps_follow_the_definition(cuda_device):
    """200 steps in 32 bits: the parameter moves by at most 3.2 lr a step, and 200
    roundings of it and of 2^-19 of the moves add up."""

    s = build([(300,), (7, 11)], cuda_device, seed=2)
    s["m"].zero_(), s["v"].zero_(), s["step"].zero_()
    p = [q.cpu().double() for q in s["params"]]
    m, v = [torch.zeros_like(q) for q in p], [torch.zeros_like(q) for q in p]
    g = torch.Generator().manual_seed(3)
    for t in range(1, 201):
        for i, q in enumerate(s["grads"]):
            q.copy_(torch.randn(q.shape, generator=g) * (1 if t % 3 else 0.01))
            p[i], m[i], v[i] = R.adamw(p[i], q.cpu().double(), m[i], v[i], t, 1e-2)
        run(s, lr=1e-2)
    assert s["step"].tolist() == [200, 0]
    for q, w in zip(s["params"], p):
        assert float((q.cpu().double() - w).abs().max()) <= 200 * (2.0**-24 * float(w.abs().max()) + 2.0**-19 * 3.2e-2)


def test_eight_bit_root_is_rounded_without_bias(cuda_device):
    """A root that decays by 1/2000 a step would be held by nearest rounding.  The
    mean over 4096 equal values of what is kept has to follow it: a rounding is
    at most a step of 1/8 off, 1/16 in standard deviation, 1/1000 in the mean's, of which
    five are allowed a step, adding like a random walk over 300 steps."""

    n = 4096
    p, g = [torch.zeros(n, device=cuda_device)], [torch.zeros(n, device=cuda_device)]
    scales = torch.ones(2, n // BLOCK, device=cuda_device)
    m = torch.zeros(n, device=cuda_device).to(torch.float8_e4m3fn)
    v = torch.full((n,), 10.0, device=cuda_device)
    v[::BLOCK] = 400.0  # sets the scale, which would carry equal values along
    v = v.to(torch.float8_e4m3fn)
    g[0][::BLOCK] = 400.0
    step = torch.zeros(2, dtype=torch.int64, device=cuda_device)
    for t in range(300):
        adamw_step(p, g, m, v, step, scales=scales, seed=11)
    root = (v.float().view(-1, BLOCK) * scales[1][:, None])[:, 1:]
    want = 10.0 * 0.999**150
    assert abs(float(root.mean()) - want) <= 5 * 0.001 * 300**0.5 * want
    assert len(torch.unique(root)) > 1


def test_eight_bit_rounding_depends_on_its_seed_only(cuda_device):
    def once(seed):
        s = build(SIZES, cuda_device, 8, seed=4)
        run(s, seed=seed)
        return s

    a, b, c = once(1), once(1), once(2)
    assert torch.equal(a["v"].view(torch.uint8), b["v"].view(torch.uint8))
    assert not torch.equal(a["v"].view(torch.uint8), c["v"].view(torch.uint8))
    assert torch.equal(a["m"].view(torch.uint8), c["m"].view(torch.uint8))
    for x, y in zip(a["params"], c["params"]):
        assert torch.equal(x, y)


def test_eight_bit_roots_do_not_vanish_and_zeros_stay(cuda_device):
    n = 2 * BLOCK
    p = [torch.zeros(n, device=cuda_device)]
    g = [torch.full((n,), 1e-7, device=cuda_device)]
    g[0][0], g[0][BLOCK:] = 1.0, 0.0
    m, v = (torch.zeros(n, device=cuda_device).to(torch.float8_e4m3fn) for _ in range(2))
    scales, step = torch.zeros(2, 2, device=cuda_device), torch.zeros(2, dtype=torch.int64, device=cuda_device)
    adamw_step(p, g, m, v, step, scales=scales)
    assert (v[1:BLOCK].float() == 2.0**-9).all()
    assert not v[BLOCK:].float().any() and not scales[:, 1].any() and not p[0][BLOCK:].any()
    assert torch.isfinite(p[0]).all()


@pytest.mark.parametrize("count", [96, 97, 800, 801, 1700])
def test_many_tensors(cuda_device, count):
    """As many as one launch takes, and more."""

    sizes = [(1 + (7 * i) % 300,) for i in range(count)]
    s = build(sizes, cuda_device, seed=5)
    old, (m0, v0) = [p.cpu().double() for p in s["params"]], values(s)
    run(s)
    assert s["step"].tolist() == [5, 0]
    for i in list(range(0, count, 37)) + [count - 1]:
        k = s["marks"][i]
        wp, wm, _ = R.adamw(old[i], s["grads"][i].cpu().double(), m0[k], v0[k], 5)
        assert ((s["params"][i].cpu().double() - wp).abs() <= 2.0**-23 * wp.abs() + 2.0**-19 * (wp - old[i]).abs()).all()
        terms = 0.9 * m0[k].abs() + 0.1 * s["grads"][i].cpu().double().abs()
        assert ((s["m"][k].cpu().double() - wm).abs() <= 2.0**-22 * (terms + 1e-6)).all()


def test_missing_gradients_leave_their_tensor(cuda_device):
    for bits in (32, 8):
        s = build(SIZES, cuda_device, bits, seed=6)
        before = [p.clone() for p in s["params"]]
        kept = s["m"].view(torch.uint8).clone()
        for i in (2, 7):
            s["grads"][i] = torch.empty(0, device=cuda_device)
        run(s)
        for i, p in enumerate(s["params"]):
            k = s["marks"][i]
            if p.numel() == 0:
                continue
            same = torch.equal(p, before[i])
            assert same == (i in (2, 7))
            if i in (2, 7):
                width = s["m"].element_size()
                assert torch.equal(s["m"].view(torch.uint8)[k.start * width:k.stop * width],
                                   kept[k.start * width:k.stop * width])


def test_grad_scale_and_skipped_steps(cuda_device):
    a, b = build(SIZES, cuda_device, seed=7), build(SIZES, cuda_device, seed=7)
    for g in b["grads"]:
        g.mul_(0.25)
    run(a, grad_scale=torch.tensor(0.25, device=cuda_device))
    run(b)
    for x, y in zip(a["params"], b["params"]):
        assert torch.equal(x, y)
    for bad in (float("inf"), float("nan")):
        before = [p.clone() for p in a["params"]]
        run(a, grad_scale=torch.tensor([bad], device=cuda_device))
        assert a["step"].tolist() == [5, 0]
        assert all(torch.equal(x, y) for x, y in zip(a["params"], before))


def test_not_a_number_stays_visible(cuda_device):
    for bits in (32, 8):
        s = build([(600,), (30,)], cuda_device, bits, seed=8)
        s["grads"][0][300] = float("nan")
        run(s)
        assert torch.isnan(s["params"][0][300]) and torch.isfinite(s["params"][0][:256]).all()
        assert torch.isfinite(s["params"][1]).all()
        m, _ = values(s)
        assert torch.isnan(m[300]) and torch.isfinite(m[:256]).all()


def test_dense_copies_of_strided_gradients(cuda_device):
    a, b = build([(40, 33)], cuda_device, seed=9), build([(40, 33)], cuda_device, seed=9)
    b["grads"][0] = b["grads"][0].t().contiguous().t()
    run(a)
    run(b)
    assert torch.equal(a["params"][0], b["params"][0])


def test_offsets_beyond_32_bits(cuda_device):
    n = 2**31 + 512
    p = torch.ones(n, device=cuda_device)
    g = torch.ones(1, device=cuda_device, dtype=torch.bfloat16).expand(n).contiguous()
    m, v = (torch.zeros(n, device=cuda_device, dtype=torch.float8_e4m3fn) for _ in range(2))
    scales, step = torch.zeros(2, n // BLOCK, device=cuda_device), torch.zeros(2, dtype=torch.int64, device=cuda_device)
    adamw_step([p], [g], m, v, step, scales=scales, lr=0.5, weight_decay=0.0)
    for k in (0, 2**31 - 1, 2**31, n - 1):
        assert abs(float(p[k]) - 0.5) < 1e-5 and abs(float(m[k].float()) - 448) < 1e-5
    assert step.tolist() == [1, 0]


def test_graphs_count_their_steps(cuda_device):
    a, b = build(SIZES, cuda_device, 8, seed=10), build(SIZES, cuda_device, 8, seed=10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(a)
    for _ in range(3):
        graph.replay()
        run(b)
    assert a["step"].tolist() == b["step"].tolist() == [7, 0]
    for x, y in zip(a["params"], b["params"]):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(a)
    torch.cuda.current_stream().wait_stream(side)
    run(b)
    for x, y in zip(a["params"], b["params"]):
        assert torch.equal(x, y)


def networks(device, dtype=torch.float32):
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(20, 33), torch.nn.Tanh(), torch.nn.Linear(33, 5))
    return net.to(device, dtype)


@pytest.mark.parametrize("bits", [32, 8])
def test_optimiser_against_torch(cuda_device, bits):
    """Fifteen steps of two groups.  In 32 bits as close as the steps' own
    bounds; in 8 bits a step is off by the moments' rounding, 1/8 of it at most: a quarter
    of the distance moved, by norm."""

    mine, wide = networks(cuda_device), networks("cpu", torch.float64)
    wide.load_state_dict({k: v.cpu().double() for k, v in mine.state_dict().items()})
    start = [p.detach().cpu().double().clone() for p in mine.parameters()]
    split = lambda n: [{"params": n[0].parameters(), "lr": 2e-2}, {"params": n[2].parameters(), "weight_decay": 0.2}]  # noqa: E731
    opt, want = AdamWCuda(split(mine), lr=1e-2, state_bits=bits), torch.optim.AdamW(split(wide), lr=1e-2)
    g = torch.Generator().manual_seed(1)
    for _ in range(15):
        x = torch.randn(64, 20, generator=g, dtype=torch.float64)
        want.zero_grad()
        wide(x).square().mean().backward()
        want.step()
        opt.zero_grad()
        for p, q in zip(mine.parameters(), wide.parameters()):  # the same gradients
            p.grad = q.grad.float().to(cuda_device)
        opt.step()
    for p, q, s in zip(mine.parameters(), wide.parameters(), start):
        off, moved = (p.detach().cpu().double() - q.detach()).norm(), (q.detach() - s).norm()
        assert off <= (1e-4 if bits == 32 else 0.25) * moved


def test_optimiser_sixteen_bit_parameters_and_saved_state(cuda_device):
    for bits in (32, 8):
        net = networks(cuda_device, torch.bfloat16)
        opt = AdamWCuda(net.parameters(), lr=1e-2, state_bits=bits, seed=3)

        def advance(net, opt, n, seed):
            g = torch.Generator(cuda_device).manual_seed(seed)
            for _ in range(n):
                opt.zero_grad()
                for p in net.parameters():
                    p.grad = torch.randn(p.shape, device=cuda_device, generator=g).to(p.dtype)
                opt.step()

        advance(net, opt, 3, 1)
        for p in net.parameters():
            assert torch.equal(p, opt.state[p]["master"].to(p.dtype))
        other = networks(cuda_device, torch.bfloat16)
        other.load_state_dict(net.state_dict())
        again = AdamWCuda(other.parameters(), lr=1e-2, state_bits=bits, seed=3)
        again.load_state_dict(opt.state_dict())
        advance(net, opt, 4, 2)
        advance(other, again, 4, 2)
        for p, q in zip(net.parameters(), other.parameters()):
            assert torch.equal(p, q) and torch.equal(opt.state[p]["master"], again.state[q]["master"])


def test_optimiser_marks_its_parameters_as_changed(cuda_device):
    w = torch.nn.Parameter(torch.ones(4, device=cuda_device))
    opt = AdamWCuda([w])
    y = (w * w).sum()
    w.grad = torch.ones_like(w)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals(cuda_device):
    s = build([(8,)], cuda_device)
    p, g, m, v, t = s["params"], s["grads"], s["m"], s["v"], s["step"]
    for kw in ({"lr": -1.0}, {"eps": -1.0}, {"weight_decay": -1.0}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)},
               {"copies": [p[0], p[0]]}, {"grad_scale": torch.ones(2, device=cuda_device)}):
        with pytest.raises(ValueError):
            adamw_step(p, g, m, v, t, **kw)
    with pytest.raises(ValueError):
        adamw_step(p, [], m, v, t)
    with pytest.raises(ValueError):
        adamw_step(p, [g[0][:4]], m, v, t)
    with pytest.raises(ValueError):
        adamw_step(p, g, m[:100], v[:100], t)
    eight = m.to(torch.float8_e4m3fn)
    with pytest.raises(ValueError):
        adamw_step(p, g, eight, eight.clone(), t)
    for args in (([p[0].half()], g, m, v, t), (p, [g[0].double()], m, v, t), (p, g, m, v, t[:1]), (p, g, m, eight, t),
                 ([p[0].cpu()], g, m, v, t), (p, [g[0].cpu()], m, v, t),
                 ([torch.zeros(8, 2, device=cuda_device)[:, 0]], g, m, v, t)):
        with pytest.raises(RuntimeError):
            adamw_step(*args)
    with pytest.raises(RuntimeError):  # too short for two tensors
        adamw_step(p * 2, g * 2, m, v, t)
    with pytest.raises(RuntimeError):
        adamw_step(p, g, m, v, t, copies=[p[0].bfloat16()])
    with pytest.raises(ValueError):
        AdamWCuda([torch.nn.Parameter(p[0].clone())], state_bits=16)
    with pytest.raises(ValueError):
        AdamWCuda([torch.nn.Parameter(p[0].clone())], lr=-1)
    with pytest.raises(RuntimeError):
        AdamWCuda([torch.nn.Parameter(p[0].double())])
