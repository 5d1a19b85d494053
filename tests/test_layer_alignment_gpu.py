"""The layer operators' C entries with results and operands that are aligned to no more than their checks ask for."""

import ctypes

import pytest
import torch

from triton_pesq_b200 import _lib, layer_norm, linear_attention, muon_step, orthogonalize

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CODES = {F32: _lib.F32, BF16: _lib.BF16, F16: _lib.F16}


def place(t, off):
    """t's values as a dense tensor that begins `off` elements past a 512-byte boundary, with a canary on both sides."""

    room = torch.full((off + t.numel() + 8,), 7.0, dtype=t.dtype, device=t.device)
    assert room.data_ptr() % 512 == 0
    room[off:off + t.numel()] = t.flatten()
    return room, room[off:off + t.numel()].view(t.shape)


def untouched(room, off, numel):
    return bool((room[:off] == 7).all()) and bool((room[off + numel:] == 7).all())


def heads(t):
    return _lib.Heads(data=t.data_ptr(), batch_stride=t.stride(0), step_stride=t.stride(1), head_stride=t.stride(2))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("key,value", [(32, 24), (33, 47), (24, 33)])
@pytest.mark.parametrize("steps", [5, 130])
def test_attention(cuda_device, dtype, key, value, steps):
    """Results of even width two elements past a boundary, of odd width one: as the torch entry's, bit for bit."""

    g = torch.Generator().manual_seed(1)
    batch, count = 2, 3
    q, k = (torch.randn(batch, steps, count, key, generator=g).to(dtype).to(cuda_device) for _ in range(2))
    v, dy = (torch.randn(batch, steps, count, value, generator=g).to(dtype).to(cuda_device) for _ in range(2))
    decay = torch.tensor([-0.1, -0.5, -0.01], device=cuda_device)
    state, dlast = (torch.randn(batch, count, key, value, generator=g).to(cuda_device) for _ in range(2))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, decay, state)]
    want = linear_attention(*leaves)
    grads = torch.autograd.grad(want, leaves, (dy, dlast))
    lib, stream = _lib.library(), torch.cuda.current_stream().cuda_stream
    d = _lib.LinearAttentionDesc(batch=batch, steps=steps, heads=count, key=key, value=value, dtype=CODES[dtype], scale=1.0,
                                 decay_shared=1, q=heads(q), k=heads(k), v=heads(v), decay_head_stride=1)
    # (32-bit operands one element past a boundary)
    inputs = [place(t, 1)[1] for t in (decay, state, dlast)]
    d.log_decay, d.state = inputs[0].data_ptr(), inputs[1].data_ptr()
    sizes = [ctypes.c_size_t() for _ in range(3)]
    _lib.check(lib.pesq_linear_attention_sizes(ctypes.byref(d), *[ctypes.byref(n) for n in sizes]), "sizes")
    work, kept, back = (torch.empty(n.value + 16, dtype=torch.uint8, device=cuda_device) for n in sizes)
    off = {key: 2 if key % 2 == 0 else 1, value: 2 if value % 2 == 0 else 1}
    rooms = [(place(torch.zeros_like(t), o), o, e) for t, o, e in
             ((v, off[value], want[0]), (state, 1, want[1]), (q, off[key], grads[0]), (q, off[key], grads[1]), (v, off[value], grads[2]),
              (decay, 1, grads[3]), (state, 1, grads[4]))]
    y, last, dq, dk, dv, ddecay, dstate = (ctypes.c_void_p(r[0][1].data_ptr()) for r in rooms)
    _lib.check(lib.pesq_linear_attention_forward(ctypes.byref(d), ctypes.c_void_p(stream), y, last, ctypes.c_void_p(kept.data_ptr()),
                                                 kept.numel(), ctypes.c_void_p(work.data_ptr()), work.numel()), "forward")
    _lib.check(lib.pesq_linear_attention_backward(ctypes.byref(d), ctypes.c_void_p(stream), ctypes.c_void_p(kept.data_ptr()), kept.numel(),
                                                  heads(dy), ctypes.c_void_p(inputs[2].data_ptr()), dq, dk, dv, ddecay, dstate,
                                                  ctypes.c_void_p(back.data_ptr()), back.numel()), "backward")
    for ((room, got), o, e) in rooms:
        assert torch.equal(got, e) and untouched(room, o, got.numel())


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16)])
@pytest.mark.parametrize("width", [64, 33, 1155])
def test_layer_norm(cuda_device, dtype, out, width):
    """All operands and results one element past a boundary.  Sums may run in another order than those of whole pieces of 16
    bytes: ten roundings of 32 bits of the largest value (times four for what a gradient is the difference of, times the root of 150 rows for
    the vectors' sums), and one to the type."""

    g = torch.Generator().manual_seed(2)
    batch, steps = 3, 50
    x = torch.randn(batch, steps, 1, width, generator=g).to(dtype).to(cuda_device)
    dy = torch.randn(batch, steps, 1, width, generator=g).to(out).to(cuda_device)
    weight, bias = (torch.randn(width, generator=g).to(cuda_device) for _ in range(2))
    leaves = [x.clone().requires_grad_(True), weight.clone().requires_grad_(True), bias.clone().requires_grad_(True)]
    want = layer_norm(*leaves, dtype=out)
    grads = torch.autograd.grad(want, leaves, dy)
    lib, stream = _lib.library(), torch.cuda.current_stream().cuda_stream
    x, dy, weight, bias = (place(t, 1)[1] for t in (x, dy, weight, bias))
    d = _lib.LayerNormDesc(batch=batch, steps=steps, heads=1, width=width, dtype=CODES[dtype], out_dtype=CODES[out], eps=1e-5, x=heads(x),
                           weight=weight.data_ptr(), bias=bias.data_ptr())
    size = ctypes.c_size_t()
    _lib.check(lib.pesq_layer_norm_workspace(ctypes.byref(d), ctypes.byref(size)), "workspace")
    work = torch.empty(size.value, dtype=torch.uint8, device=cuda_device)
    rooms = [(place(torch.zeros_like(e), 1), e) for e in (want, *grads)]
    y, dx, dweight, dbias = (ctypes.c_void_p(r[0][1].data_ptr()) for r in rooms)
    _lib.check(lib.pesq_layer_norm_forward(ctypes.byref(d), ctypes.c_void_p(stream), y), "forward")
    _lib.check(lib.pesq_layer_norm_backward(ctypes.byref(d), ctypes.c_void_p(stream), heads(dy), dx, dweight, dbias,
                                            ctypes.c_void_p(work.data_ptr()), work.numel()), "backward")
    for (room, got), e in rooms:
        allowed = torch.finfo(e.dtype).eps * e.abs().double() + 10 * 2.0**-24 * float(e.detach().abs().max()) * (12 if e.dim() == 1 else 4)
        assert bool(((got.double() - e.double()).abs() <= allowed).all()) and untouched(room, 1, got.numel())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(96, 257), (385, 200)])
def test_muon(cuda_device, dtype, shape):
    """Tensors one element past a boundary, through the torch entries: the same bits."""

    g = torch.Generator().manual_seed(3)
    param, momentum, grad = (torch.randn(shape, generator=g).to(cuda_device) for _ in range(3))
    grad = grad.to(dtype)
    copy = None if dtype == F32 else torch.zeros_like(grad)
    tensors = [param, grad, momentum, *([] if copy is None else [copy])]
    rooms = [place(t, 1) for t in tensors]
    moved = [r[1] for r in rooms]
    for p, gr, m, *c in (tensors, moved):
        muon_step([p], [gr], [m], copies=c or None, lr=0.1)
    for a, e, (room, _) in zip(moved, tensors, rooms):
        assert torch.equal(a, e) and untouched(room, 1, e.numel())
    assert torch.equal(orthogonalize(place(grad, 1)[1]), orthogonalize(grad)) and _lib.muon_check() == 0
