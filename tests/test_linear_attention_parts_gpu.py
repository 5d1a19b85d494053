"""The linear attention's rows that are cut in parts, with states that last longer than a part: parts that make the states they
begin from themselves (up to four) and parts that a join makes them for, of several chunks each, in both directions.  Bounds
as in test_linear_attention_gpu.py; the definition runs on the GPU in 64 bits."""

import ctypes

import pytest
import torch

from test_linear_attention_gpu import compare, definition, make, on
from triton_pesq_b200 import _lib, linear_attention

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def parts_of(tensors, kw, backward):
    """(parts, chunks) of a row, from the workspace of a call whose rows are all cut: a state and a factor for each part."""

    q, v, decay = tensors[0], tensors[2], tensors[3]
    code = {F32: _lib.F32, BF16: _lib.BF16, F16: _lib.F16}[q.dtype]
    batch, steps, heads, key = q.shape
    d = _lib.LinearAttentionDesc(batch=batch, steps=steps, heads=heads, key=key, value=v.shape[3], dtype=code, scale=1.0,
                                 decay_shared=decay.dim() == 1, lengths=16 if "lengths" in kw else None)
    sizes = [ctypes.c_size_t() for _ in range(3)]
    _lib.check(_lib.library().pesq_linear_attention_sizes(ctypes.byref(d), *[ctypes.byref(n) for n in sizes]), "sizes")
    dk, dv = (32 if n <= 32 else 64 if n <= 64 else 128 for n in (key, v.shape[3]))
    chunk = 32 if q.dtype == F32 and dk == dv == 128 else 64
    rows, chunks = batch * heads, -(-steps // chunk)
    size = sizes[2].value if backward else sizes[0].value
    if backward and decay.dim() == 1:
        size -= -(-rows * chunks * 8 // 16) * 16
    for parts in range(2, chunks + 1):
        if -(-rows * parts * dk * dv * 4 // 16) * 16 + -(-rows * parts * 4 // 16) * 16 == size:
            return parts, chunks
    assert size == 0
    return 1, chunks


def slow(case, device, factor=0.02):
    """The case on the GPU, its decays of the data so slow that a state lasts for hundreds of steps."""

    tensors, dy, dlast, kw = case
    if tensors[3].dim() == 3:
        tensors[3] = factor * tensors[3]
    return [t.to(device) for t in tensors], dy.to(device), dlast.to(device), on(device, kw)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,forward,backward", [((8, 500, 12, 64, 64), 4, 3), ((12, 500, 8, 24, 40), 4, 3), ((8, 380, 12, 16, 33), 3, 3),
                                                    ((6, 1000, 10, 128, 100), 1, 2), ((6, 420, 10, 100, 72), 1, 2)])
@pytest.mark.parametrize("gated,reset,reverse", [(False, False, False), (True, False, True), (True, True, False), (False, True, True)])
def test_parts_that_make_their_own_states(cuda_device, dtype, shape, forward, backward, gated, reset, reverse):
    case = slow(make(*shape, dtype, gated=gated, reset=reset, seed=21), cuda_device)
    if reset:
        case[3]["reset"] &= torch.rand(shape[:2], generator=torch.Generator().manual_seed(3)).to(cuda_device) < 0.05
    for way, want in ((False, forward), (True, backward)):
        parts, chunks = parts_of(case[0], case[3], way)
        assert parts == want and (parts == 1 or chunks > parts), (parts, chunks)
    compare(*case, cuda_device, reverse=reverse)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(4, 3000, 12, 24, 40), (2, 1500, 8, 128, 128), (2, 3001, 10, 64, 48)])
@pytest.mark.parametrize("gated,reset,reverse", [(False, False, False), (True, False, True), (True, True, False)])
def test_joined_parts_of_several_chunks(cuda_device, dtype, shape, gated, reset, reverse):
    case = slow(make(*shape, dtype, gated=gated, reset=reset, seed=22), cuda_device)
    if reset:
        case[3]["reset"] &= torch.rand(shape[:2], generator=torch.Generator().manual_seed(4)).to(cuda_device) < 0.05
    for way in (False, True):
        parts, chunks = parts_of(case[0], case[3], way)
        assert parts > 4 and chunks >= 2 * parts - 2, (parts, chunks)
    compare(*case, cuda_device, reverse=reverse)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reverse", [False, True])
def test_parts_past_a_row_s_length(cuda_device, dtype, reverse):
    """Rows that end within a part, at a part's end, before the last parts, and at once."""

    case = slow(make(5, 3000, 10, 24, 40, dtype, lengths=True, seed=23), cuda_device)
    parts, chunks = parts_of(case[0], case[3], False)
    assert parts > 4 and chunks >= 2 * parts - 2, (parts, chunks)
    per = -(-chunks // parts) * 64
    case[3]["lengths"] = torch.tensor([0, 3000, 3 * per, 3 * per + 65, 70], device=cuda_device)
    compare(*case, cuda_device, reverse=reverse)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(3, 400, 4, 64, 64), (2, 300, 2, 64, 100), (8, 500, 12, 64, 64), (2, 1500, 8, 24, 40)])
def test_gradients_of_decays_by_their_norm(cuda_device, dtype, shape):
    """A decay's gradient sums products of a state or its gradient with an input, and of the two: three sums whose errors have
    nothing to do with each other.  Beside bfloat16 an operand of two terms is 2^-18 off at most; of the others products of
    two tf32 terms leave out 3 * 2^-22 at most, and the states' own roundings are sqrt(10) * 2^-23."""

    (q, k, v, decay, state), dy, dlast, kw = slow(make(*shape, dtype, gated=True, seed=24), cuda_device, 0.2)
    mine, wide = decay.clone().requires_grad_(True), decay.double().requires_grad_(True)
    out = linear_attention(q, k, v, mine, state, **kw)
    want_out = definition(*(t.double() for t in (q, k, v)), wide, state.double(), **kw)
    got = torch.autograd.grad(out, mine, (dy, dlast))[0].double()
    want = torch.autograd.grad(want_out, wide, (dy.double(), dlast.double()))[0]
    off = float((got - want).norm() / want.norm())
    term = 2.0**-18 if dtype == BF16 else 3 * 2.0**-22 + 10**0.5 * 2.0**-23
    assert off <= 3**0.5 * term, off


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(2, 150, 3, 32, 32), (2, 150, 3, 128, 128), (1, 1500, 2, 64, 48)])
def test_gradients_behind_a_reset_see_nothing_of_the_state(cuda_device, dtype, shape):
    """A state that is not a number, of rows that forget it at their first step: every gradient is what it is without."""

    (q, k, v, decay, state), dy, dlast, kw = make(*shape, dtype, gated=True, seed=25)
    reset = torch.zeros(shape[:2], dtype=torch.bool, device=cuda_device)
    reset[:, 0] = True
    outs = []
    for s in (torch.full_like(state, float("nan")), torch.zeros_like(state)):
        leaves = [t.to(cuda_device).requires_grad_(True) for t in (q, k, v, decay, s)]
        out = linear_attention(*leaves, reset=reset, **kw)
        outs.append([*(t.detach() for t in out), *torch.autograd.grad(out, leaves, (dy.to(cuda_device), dlast.to(cuda_device)))])
    for a, e in zip(*outs):
        assert torch.isfinite(e).all() and torch.equal(a, e)
    assert not outs[0][-1].any()
