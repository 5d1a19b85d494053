"""What the layer norm, the linear attention and Muon refuse without a GPU, and their C entries' checks."""

import ctypes

import pytest
import torch

from triton_pesq_b200 import (LayerNormCuda, LinearAttentionCuda, MuonCuda, _lib, layer_norm, linear_attention, muon_step,
                              orthogonalize)


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


@pytest.mark.parametrize("heads,width", [(1, 1), (1, 8192), (14, 64), (128, 8192), (1000, 64), (16384, 64), (1 << 20, 1), (100000, 7)])
@pytest.mark.parametrize("steps", [1, 1000, 1 << 20])
def test_layer_norm_workspace_stays_small(heads, width, steps):
    """One CTA's sums are of its own heads: twice as many vectors as CTAs at most, however many heads there are."""
    d = _lib.LayerNormDesc(batch=1, steps=steps, heads=heads, width=width, dtype=_lib.F32, out_dtype=_lib.F32, eps=0.0)
    size = ctypes.c_size_t()
    assert _lib.library().pesq_layer_norm_workspace(ctypes.byref(d), ctypes.byref(size)) == _lib.PESQ_OK
    assert 2 * 4 * heads * width <= size.value <= 1 << 25


def test_linear_attention_without_a_gpu():
    x = torch.zeros(1, 2, 3, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        linear_attention(x, x, x, torch.zeros(3))
    for kw in ({"heads": 0, "key": 4}, {"heads": 2, "key": 0}, {"heads": 2, "key": 129}, {"heads": 2, "key": 4, "slow": 1.0},
               {"heads": 2, "key": 4, "fast": 0.99, "slow": 0.9}):
        with pytest.raises(ValueError):
            LinearAttentionCuda(**kw)
    module = LinearAttentionCuda(5, 16)
    a = torch.exp(module.log_decay())
    assert (a[1:] > a[:-1]).all() and "heads=5" in repr(module)
    assert float(torch.exp(LinearAttentionCuda(1, 16).log_decay())) == pytest.approx(0.875)


def test_linear_attention_entry_checks_its_descriptor():
    lib = _lib.library()

    def make(**kw):
        d = _lib.LinearAttentionDesc(batch=2, steps=100, heads=3, key=64, value=48, dtype=_lib.BF16, scale=1.0)
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    def sizes(d):
        out = [ctypes.c_size_t() for _ in range(3)]
        return lib.pesq_linear_attention_sizes(ctypes.byref(d), *[ctypes.byref(n) for n in out]), [n.value for n in out]

    assert sizes(make())[0] == _lib.PESQ_OK
    for bad in ({"batch": 0}, {"steps": 0}, {"heads": -1}, {"key": 0}, {"value": 0}, {"dtype": 3}, {"scale": float("nan")},
                {"scale": float("inf")}):
        assert sizes(make(**bad))[0] == 1, bad
    for large in ({"key": 129}, {"value": 129}, {"batch": 1 << 22}, {"batch": 1 << 40}, {"steps": 1 << 31}):
        assert sizes(make(**large))[0] == 2, large
    assert lib.pesq_linear_attention_sizes(ctypes.byref(make()), None, None, None) == 1
    # a state of 32 bits before every chunk of 64 steps (of 32 where float32 keys and values are wide), of padded widths
    for kw, chunks, width in (({}, 2, 64 * 64), ({"dtype": _lib.F32}, 2, 64 * 64), ({"key": 128, "value": 100}, 2, 128 * 128),
                              ({"key": 128, "value": 100, "dtype": _lib.F32}, 4, 128 * 128), ({"key": 3, "value": 33}, 2, 32 * 64)):
        assert sizes(make(**kw))[1][1] == 2 * 3 * chunks * width * 4
    # short rows need no workspace, long ones that are few do, and a head's decay gradient always
    assert sizes(make())[1][::2] == [0, 0]
    assert sizes(make(decay_shared=1))[1][2] > 0
    long = make(steps=5000)
    assert min(sizes(long)[1]) > 0
    one, odd = ctypes.c_void_p(16), ctypes.c_void_p(18)
    x = _lib.Heads(data=16, batch_stride=19200, step_stride=192, head_stride=64)
    none = _lib.Heads(data=None)
    full = dict(q=x, k=x, v=x, log_decay=16)

    def forward(d, y=one, kept=None, kept_bytes=0, ws=one, ws_bytes=1 << 30):
        return lib.pesq_linear_attention_forward(ctypes.byref(d), None, y, one, kept, kept_bytes, ws, ws_bytes)

    assert forward(make()) == 1 and forward(make(**full), y=None) == 1 and forward(make(**full), y=odd) == 1
    assert forward(make(**{**full, "q": _lib.Heads(data=17)})) == 1
    assert forward(make(**full), kept=one, kept_bytes=100) == _lib.PESQ_ERR_WORKSPACE
    assert forward(make(steps=5000, **full), ws=None, ws_bytes=0) == _lib.PESQ_ERR_WORKSPACE

    def backward(d, kept=one, kept_bytes=1 << 30, dy=x, dq=one, ws=one, ws_bytes=1 << 30):
        return lib.pesq_linear_attention_backward(ctypes.byref(d), None, kept, kept_bytes, dy, None, dq, one, one, one, None,
                                                  ws, ws_bytes)

    assert backward(make(**full), dy=none) == 1 and backward(make(**full), dq=None) == 1 and backward(make(**full), dq=odd) == 1
    assert backward(make(**full), kept=None) == 3 and backward(make(**full), kept_bytes=64) == 3
    assert backward(make(decay_shared=1, **full), ws=None) == 3


def test_muon_without_a_gpu():
    p = torch.nn.Parameter(torch.ones(4, 4))
    p.grad = torch.ones(4, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        MuonCuda([p]).step()
    with pytest.raises((RuntimeError, NotImplementedError)):
        orthogonalize(p)
    with pytest.raises((RuntimeError, NotImplementedError)):
        muon_step([p.detach()], [p.grad], [torch.zeros(4, 4)])
    for kw in ({"lr": -1.0}, {"momentum": 1.0}, {"weight_decay": -0.1}, {"coefficients": (1.0, 2.0)}, {"coefficients": (20.0, 0.0, 0.0)},
               {"eps": 0.0}, {"eps": float("inf")}, {"steps": 0}, {"steps": 101}, {"adjust": "x"}):
        with pytest.raises(ValueError):
            MuonCuda([torch.nn.Parameter(torch.ones(2, 2))], **kw)
    for bad in (torch.ones(3), torch.ones(2, 2, 2), torch.ones(0, 3), torch.ones(2, 3).T, torch.ones(2, 2).double()):
        with pytest.raises(RuntimeError):
            MuonCuda([torch.nn.Parameter(bad)])
    good = MuonCuda([p])
    with pytest.raises(ValueError, match="momentum"):
        good.load_state_dict({**good.state_dict(), "state": {0: {"momentum": torch.zeros(4, 4), "master": torch.zeros(4, 4)}}})


def test_muon_entry_checks_its_descriptor():
    lib = _lib.library()
    size = ctypes.c_size_t()

    def workspace(count=1, rows=100, cols=200, param=16, grad=16, momentum=16, copy=None, **kw):
        d = _lib.MuonDesc(grad_dtype=_lib.F32, nesterov=1, adjust=0, steps=5, momentum=0.95, lr=0.02, weight_decay=0.1, eps=1e-7, a=3.4,
                          b=-4.8, c=2.0)
        for k, v in kw.items():
            setattr(d, {"beta": "momentum"}.get(k, k), v)
        t = (_lib.MuonTensor * 1)(_lib.MuonTensor(param=param, grad=grad, momentum=momentum, copy=copy, rows=rows, cols=cols))
        return lib.pesq_muon_workspace(ctypes.byref(d), t, count, ctypes.byref(size)), d, t

    assert workspace()[0] == _lib.PESQ_OK
    # X before and after a step, A, b + c A and the polynomial, in tiles of 128, 4 bytes a value; a norm's sums and a counter
    assert size.value == (2 * 128 * 256 + 3 * 128 * 128) * 4 + 8 * -(-100 * 200 // 8192) + 16
    for bad in ({"count": -1}, {"rows": 0}, {"cols": 0}, {"param": None}, {"momentum": None}, {"copy": 16}, {"grad_dtype": 3},
                {"steps": 0}, {"steps": 101}, {"adjust": 2}, {"beta": 1.0}, {"beta": float("nan")}, {"lr": -1.0},
                {"weight_decay": float("nan")}, {"eps": 0.0}, {"eps": float("inf")}, {"a": 17.0}, {"b": float("nan")}):
        assert workspace(**bad)[0] == 1, bad
    assert workspace(rows=32769)[0] == 2 and workspace(cols=1 << 40)[0] == 2
    assert workspace(grad=None, param=None)[0] == _lib.PESQ_OK and size.value == 0
    _, d, t = workspace()
    assert lib.pesq_muon_workspace(ctypes.byref(d), t, 1, None) == 1
    assert lib.pesq_muon_step(ctypes.byref(d), t, 1, None, None, 0) == _lib.PESQ_ERR_WORKSPACE
    assert lib.pesq_muon_step(ctypes.byref(d), t, 1, None, ctypes.c_void_p(8), 1 << 40) == _lib.PESQ_ERR_WORKSPACE
    assert lib.pesq_muon_step(None, None, 0, None, None, 0) == 1
    o = _lib.OrthogonalizeDesc(count=2, rows=100, cols=200, dtype=_lib.BF16, steps=5, eps=1e-7, a=3.4, b=-4.8, c=2.0)
    assert lib.pesq_orthogonalize_workspace(ctypes.byref(o), ctypes.byref(size)) == _lib.PESQ_OK
    assert lib.pesq_orthogonalize(ctypes.byref(o), None, None, ctypes.c_void_p(16), ctypes.c_void_p(16), 1 << 40) == 1
    assert lib.pesq_orthogonalize(ctypes.byref(o), None, ctypes.c_void_p(16), ctypes.c_void_p(16), ctypes.c_void_p(16), 100) == 3
    o.count = 0
    assert lib.pesq_orthogonalize_workspace(ctypes.byref(o), ctypes.byref(size)) == 1
