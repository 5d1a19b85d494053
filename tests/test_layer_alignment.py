"""Operands of the layer operators' C entries that are less aligned than what the kernels load and store: refused on the host,
before any launch.  The addresses are not memory: where there is a GPU the tests are skipped, so that nothing is ever launched on
them."""

import ctypes

import pytest
import torch

from triton_pesq_b200 import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="a call that is not refused would be launched")

INVALID = 1
ONE = ctypes.c_void_p(64)


def at(address):
    return ctypes.c_void_p(address)


def attention(dtype, key, value, **kw):
    x = _lib.Heads(data=64, batch_stride=19200, step_stride=192, head_stride=64)
    d = _lib.LinearAttentionDesc(batch=2, steps=100, heads=3, key=key, value=value, dtype=dtype, scale=1.0, q=x, k=x, v=x, log_decay=64)
    for k, v in kw.items():
        setattr(d, k, v)
    return ctypes.byref(d), x


def attention_forward(d, y=ONE, last=ONE):
    return _lib.library().pesq_linear_attention_forward(d, None, y, last, None, 0, ONE, 1 << 40)


def attention_backward(d, dy, dq=ONE, dk=ONE, dv=ONE, ddecay=ONE, dstate=ONE, dlast=ONE):
    return _lib.library().pesq_linear_attention_backward(d, None, ONE, 1 << 40, dy, dlast, dq, dk, dv, ddecay, dstate, ONE, 1 << 40)


@pytest.mark.parametrize("dtype,size", [(_lib.F32, 4), (_lib.BF16, 2), (_lib.F16, 2)])
def test_attention_results_of_even_width_are_stored_in_pairs(dtype, size):
    """Two adjacent elements of a row of even width are one store; rows of odd width go element by element."""

    for off in (size, size // 2, 1):
        d, x = attention(dtype, 64, 48)
        assert attention_forward(d, y=at(64 + off)) == INVALID
        for name in ("dq", "dk", "dv"):
            assert attention_backward(d, x, **{name: at(64 + off)}) == INVALID, (name, off)
    for off in (size // 2, 1):
        d, x = attention(dtype, 33, 47)
        assert attention_forward(d, y=at(64 + off)) == INVALID
        for name in ("dq", "dk", "dv"):
            assert attention_backward(d, x, **{name: at(64 + off)}) == INVALID, (name, off)


def test_attention_operands_are_aligned_to_their_types():
    good, x = attention(_lib.F32, 64, 48)
    for dtype, off in ((_lib.F32, 2), (_lib.BF16, 1)):
        odd = _lib.Heads(data=64 + off, batch_stride=19200, step_stride=192, head_stride=64)
        for name in ("q", "k", "v"):
            d, _ = attention(dtype, 64, 48, **{name: odd})
            assert attention_forward(d) == INVALID and attention_backward(d, x) == INVALID, name
        d, _ = attention(dtype, 64, 48)
        assert attention_backward(d, odd) == INVALID
    for name, address in (("log_decay", 66), ("state", 66), ("lengths", 68)):
        d, _ = attention(_lib.BF16, 64, 48, **{name: address})
        assert attention_forward(d) == INVALID and attention_backward(d, x) == INVALID, name
    assert attention_forward(good, last=at(66)) == INVALID
    for name in ("dlast", "ddecay", "dstate"):
        assert attention_backward(good, x, **{name: at(66)}) == INVALID, name


def test_layer_norm_operands_are_aligned_to_their_types():
    lib = _lib.library()

    def call(out=_lib.BF16, x=64, weight=64, bias=64, dy=64, dx=64, dweight=64, dbias=64, y=64):
        """Of float32, with gradients of `out`: (the forward's answer, the backward's)."""

        d = _lib.LayerNormDesc(batch=2, steps=3, heads=1, width=64, dtype=_lib.F32, out_dtype=out, eps=1e-6, weight=weight, bias=bias,
                               x=_lib.Heads(data=x, batch_stride=192, step_stride=64, head_stride=64))
        g = _lib.Heads(data=dy, batch_stride=192, step_stride=64, head_stride=64)
        return (lib.pesq_layer_norm_forward(ctypes.byref(d), None, at(y)),
                lib.pesq_layer_norm_backward(ctypes.byref(d), None, g, at(dx), at(dweight), at(dbias), ONE, 1 << 40))

    for name in ("x", "weight", "bias"):
        assert call(**{name: 66}) == (INVALID, INVALID), name
    assert call(y=65, dy=65) == (INVALID, INVALID)
    assert call(out=_lib.F32, y=66, dy=66) == (INVALID, INVALID)
    for name in ("dx", "dweight", "dbias"):
        assert call(y=65, **{name: 66}) == (INVALID, INVALID), name


def test_muon_tensors_are_aligned_to_their_types():
    lib = _lib.library()

    def step(dtype=_lib.BF16, **kw):
        d = _lib.MuonDesc(grad_dtype=dtype, nesterov=1, adjust=0, steps=5, momentum=0.95, lr=0.02, weight_decay=0.1, eps=1e-7, a=3.4, b=-4.8,
                          c=2.0, grad_scale=kw.pop("grad_scale", None))
        t = (_lib.MuonTensor * 1)(_lib.MuonTensor(**{**dict(param=64, grad=64, momentum=64, copy=None, rows=100, cols=200), **kw}))
        return lib.pesq_muon_step(ctypes.byref(d), t, 1, None, ONE, 1 << 40)

    for kw in ({"param": 66}, {"momentum": 66}, {"grad": 65}, {"copy": 65}, {"grad_scale": 66}, {"dtype": _lib.F32, "grad": 66}):
        assert step(**kw) == INVALID, kw
    for dtype, off in ((_lib.F32, 2), (_lib.F16, 1)):
        o = _lib.OrthogonalizeDesc(count=2, rows=100, cols=200, dtype=dtype, steps=5, eps=1e-7, a=3.4, b=-4.8, c=2.0)
        assert lib.pesq_orthogonalize(ctypes.byref(o), None, at(64 + off), ONE, ONE, 1 << 40) == INVALID
        assert lib.pesq_orthogonalize(ctypes.byref(o), None, ONE, at(64 + off), ONE, 1 << 40) == INVALID
