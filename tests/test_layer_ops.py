"""What the layer norm, the linear attention and Muon refuse without a GPU, and their C entries' checks."""

import ctypes

import pytest
import torch

from triton_pesq_b200 import LayerNormCuda, _lib, layer_norm


def test_layer_norm_without_a_gpu():
    x, v = torch.zeros(1, 2, 4), torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU"):
        layer_norm(x, v)
    for kw in ({"channels": 0}, {"channels": 8193}, {"channels": 4, "eps": -1.0}, {"channels": 4, "heads": 0},
               {"channels": 1024, "heads": 1025}):
        with pytest.raises(ValueError):
            LayerNormCuda(**kw)
    assert "channels=5" in repr(LayerNormCuda(5)) and LayerNormCuda(5, heads=3).weight.shape == (3, 5)


def test_layer_norm_entry_checks_its_descriptor():
    lib = _lib.library()

    def make(**kw):
        d = _lib.LayerNormDesc(batch=2, steps=3, heads=1, width=64, dtype=_lib.F32, out_dtype=_lib.BF16, eps=1e-6)
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    size = ctypes.c_size_t()
    assert lib.pesq_layer_norm_workspace(ctypes.byref(make()), ctypes.byref(size)) == _lib.PESQ_OK and size.value > 0
    for bad in ({"batch": 0}, {"steps": -1}, {"heads": 0}, {"width": 0}, {"dtype": 5}, {"dtype": _lib.F16}, {"out_dtype": -1},
                {"eps": -1.0}, {"eps": float("nan")}):
        assert lib.pesq_layer_norm_workspace(ctypes.byref(make(**bad)), ctypes.byref(size)) == 1, bad
    for large in ({"width": 8193}, {"heads": 1 << 15}, {"steps": 1 << 32}, {"batch": 1 << 31}):
        assert lib.pesq_layer_norm_workspace(ctypes.byref(make(**large)), ctypes.byref(size)) == 2, large
    assert lib.pesq_layer_norm_workspace(ctypes.byref(make()), None) == 1
    one = ctypes.c_void_p(16)
    assert lib.pesq_layer_norm_forward(None, None, one) == 1
    assert lib.pesq_layer_norm_forward(ctypes.byref(make()), None, one) == 1  # no x
    x = _lib.Heads(data=16, batch_stride=192, step_stride=64, head_stride=64)
    d = make(x=x, weight=16)
    assert lib.pesq_layer_norm_forward(ctypes.byref(d), None, None) == 1
    none = _lib.Heads(data=None)
    assert lib.pesq_layer_norm_backward(ctypes.byref(d), None, none, one, one, None, one, 1 << 30) == 1
    assert lib.pesq_layer_norm_backward(ctypes.byref(d), None, x, one, one, None, one, 8) == _lib.PESQ_ERR_WORKSPACE
    assert lib.pesq_layer_norm_backward(ctypes.byref(d), None, x, one, one, None, ctypes.c_void_p(24), 1 << 30) == 3
