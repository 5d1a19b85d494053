"""What the training operators refuse without a GPU, and their C entries' checks."""

import ctypes

import pytest
import torch

from triton_pesq_b200 import (AdamWCuda, GatedScanCuda, NormJoinCuda, _lib, adamw_step, gated_scan, norm_join,
                              pre_norm)


def test_cpu_tensors_are_refused():
    x, v = torch.zeros(1, 2, 4), torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU"):
        gated_scan(x, x, x, v)
    with pytest.raises(RuntimeError, match="GPU"):
        norm_join(x, x, v, v)
    with pytest.raises(RuntimeError, match="GPU"):
        pre_norm(x, v)
    p = torch.nn.Parameter(torch.ones(4))
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU"):
        AdamWCuda([p]).step()
    with pytest.raises((RuntimeError, NotImplementedError)):
        adamw_step([p], [p.grad], torch.zeros(256), torch.zeros(256), torch.zeros(2, dtype=torch.int64))


def test_module_arguments():
    for kw in ({"channels": 0}, {"channels": 4, "rate": 0}, {"channels": 4, "fast": 0.9, "slow": 1.0},
               {"channels": 4, "fast": 0.99, "slow": 0.9}):
        with pytest.raises(ValueError):
            GatedScanCuda(**kw)
    module = GatedScanCuda(5)
    a = torch.exp(-module.rate * torch.nn.functional.softplus(module.decay))
    assert ((a > 0.899) & (a < 0.9991)).all()
    join = NormJoinCuda(5, scale=None)
    assert join.scale is None and "channels=5" in repr(join)
    for kw in ({"state_bits": 4}, {"lr": -1.0}, {"betas": (1.0, 0.5)}, {"eps": -1e-8}, {"weight_decay": -1.0}):
        with pytest.raises(ValueError):
            AdamWCuda([torch.nn.Parameter(torch.ones(2))], **kw)


def _scan(**kw):
    d = _lib.GatedScanDesc(batch=2, steps=100, width=64, dtype=_lib.BF16, rate=8.0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _sizes(d):
    out = [ctypes.c_size_t() for _ in range(3)]
    status = _lib.library().pesq_gated_scan_sizes(ctypes.byref(d), *[ctypes.byref(n) for n in out])
    return status, [n.value for n in out]


def test_gated_scan_entry_checks_its_descriptor():
    lib = _lib.library()
    assert _sizes(_scan())[0] == _lib.PESQ_OK
    for bad in ({"batch": 0}, {"steps": 0}, {"width": -1}, {"dtype": 3}, {"dtype": -1}, {"rate": 0.0},
                {"rate": float("nan")}, {"rate": float("inf")}):
        assert _sizes(_scan(**bad))[0] == _lib.PESQ_ERR_INVALID_ARGUMENT, bad
    for large in ({"batch": 65536}, {"width": 1 << 25}, {"steps": 1 << 31}):
        assert _sizes(_scan(**large))[0] == 2, large
    # refused before anything is launched
    d, one = _scan(), ctypes.c_void_p(16)
    assert lib.pesq_gated_scan_forward(None, None, one, one, None, 0, one, 1 << 30) == _lib.PESQ_ERR_INVALID_ARGUMENT
    assert lib.pesq_gated_scan_forward(ctypes.byref(d), None, None, one, None, 0, one, 1 << 30) == 1
    assert lib.pesq_gated_scan_forward(ctypes.byref(d), None, one, one, None, 0, one, 1 << 30) == 1
    assert "NULL" in _lib.last_error()
    long = _scan(steps=1000)  # cut into strips; 100 steps go through one CTA, which needs no workspace
    assert _sizes(d)[1][0] == 0 and _sizes(long)[1][0] > 0
    assert lib.pesq_gated_scan_forward(ctypes.byref(long), None, one, one, None, 0, None, 0) == _lib.PESQ_ERR_WORKSPACE
    dy = _lib.Stream(data=None, batch_stride=0, step_stride=0)
    assert lib.pesq_gated_scan_backward(ctypes.byref(d), None, None, 0, dy, None, one, one, one, one, None, one,
                                        1 << 30) == _lib.PESQ_ERR_WORKSPACE


def test_gated_scan_entry_checks_what_boxes_need_of_results():
    """Streams that are copied in boxes ask for results that are 16-byte aligned."""
    lib = _lib.library()
    one, off = ctypes.c_void_p(16), ctypes.c_void_p(24)
    dense = _lib.Stream(data=16, batch_stride=100 * 64, step_stride=64)
    d = _scan(x=dense, input_gate=dense, decay_gate=dense)
    assert lib.pesq_gated_scan_forward(ctypes.byref(d), None, off, one, None, 0, one, 1 << 30) == 1
    assert "aligned" in _lib.last_error()
    for k in range(3):
        out = [off if i == k else one for i in range(3)]
        assert lib.pesq_gated_scan_backward(ctypes.byref(d), None, one, 1 << 30, dense, None, *out, one, None, one,
                                            1 << 30) == 1
        assert "aligned" in _lib.last_error()


def test_gated_scan_keeps_one_state_a_chunk():
    for steps, width in ((1, 7), (8, 64), (9, 64), (1000, 96)):
        d = _scan(batch=3, steps=steps, width=width)
        status, (_, kept, _) = _sizes(d)
        assert status == _lib.PESQ_OK
        chunks = -(-steps // (1 if steps == 1 else 8))
        assert kept == -(-3 * chunks * width * 4 // 16) * 16


def test_norm_join_entry_checks_its_descriptor():
    lib = _lib.library()

    def make(**kw):
        d = _lib.NormJoinDesc(batch=2, steps=3, width=64, stream_dtype=_lib.F32, dtype=_lib.BF16, eps=1e-6)
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    size = ctypes.c_size_t()
    assert lib.pesq_norm_join_workspace(ctypes.byref(make()), ctypes.byref(size)) == _lib.PESQ_OK and size.value > 0
    for bad in ({"batch": 0}, {"width": 0}, {"dtype": 5}, {"stream_dtype": _lib.F16}, {"activation": 2}, {"eps": -1.0},
                {"eps": float("nan")}, {"gate_shared": 1}):
        assert lib.pesq_norm_join_workspace(ctypes.byref(make(**bad)), ctypes.byref(size)) == 1, bad
    assert lib.pesq_norm_join_workspace(ctypes.byref(make(width=8193)), ctypes.byref(size)) == 2
    assert lib.pesq_norm_join_forward(ctypes.byref(make()), None, None, None) == 1


def test_adamw_entry_checks_its_descriptor():
    lib = _lib.library()

    def step(count=1, n=256, param=16, grad=16, copy=None, **kw):
        d = _lib.AdamwDesc(grad_dtype=_lib.F32, state_bits=32, units=1, moment1=16, moment2=16, step=16, beta1=0.9,
                           beta2=0.999, lr=1e-3, eps=1e-8, weight_decay=0.0)
        for k, v in kw.items():
            setattr(d, k, v)
        t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(param=param, grad=grad, copy=copy, n=n))
        return lib.pesq_adamw_step(ctypes.byref(d), t, count, None)

    assert lib.pesq_adamw_step(None, None, 0, None) == 1
    for bad in ({"count": -1}, {"n": -1}, {"param": None}, {"copy": 16}, {"grad_dtype": 4}, {"state_bits": 16},
                {"state_bits": 8}, {"moment1": None}, {"moment2": 8}, {"step": None}, {"beta1": 1.0}, {"beta2": -0.1},
                {"beta1": float("nan")}, {"lr": -1.0}, {"eps": float("nan")}, {"weight_decay": -0.5}):
        assert step(**bad) == 1, bad
    assert step(n=257) == _lib.PESQ_ERR_WORKSPACE


def test_gated_scan_keeps_the_same_whatever_the_layout():
    """A tracer has shapes alone to go by."""
    for steps, width in ((1, 64), (16, 64), (90, 64), (1000, 96), (300, 33)):
        want = _sizes(_scan(batch=3, steps=steps, width=width))[1][1]
        for dtype in (_lib.F32, _lib.BF16):
            for at, stride in ((0, width), (16, width), (8, 3 * width), (2, width + 1)):
                layout = _lib.Stream(data=4096 + at, batch_stride=steps * stride, step_stride=stride)
                d = _scan(batch=3, steps=steps, width=width, dtype=dtype, x=layout, input_gate=layout, decay_gate=layout)
                assert _sizes(d)[1][1] == want


def test_gated_scan_says_how_far_apart_it_keeps_its_states():
    """As far as chunks, which follow from the layout; a backward that needs them closer refuses them."""
    lib, one = _lib.library(), ctypes.c_void_p(4096)
    here, most = ctypes.c_int32(), ctypes.c_int32()
    boxes = _lib.Stream(data=4096, batch_stride=100 * 64, step_stride=64)
    lanes = _lib.Stream(data=4096 + 2, batch_stride=100 * 64, step_stride=64)
    cases = ((boxes, 100, 64, 16, 16), (lanes, 100, 64, 8, 16), (lanes, 100, 63, 8, 8), (lanes, 10, 64, 8, 8), (boxes, 1, 64, 1, 1))
    for stream, steps, width, want, longest in cases:
        d = _scan(steps=steps, width=width, x=stream, input_gate=stream, decay_gate=stream)
        assert lib.pesq_gated_scan_kept_steps(ctypes.byref(d), ctypes.byref(here), ctypes.byref(most)) == _lib.PESQ_OK
        assert (here.value, most.value) == (want, longest)
    assert lib.pesq_gated_scan_kept_steps(ctypes.byref(d), None, ctypes.byref(most)) == 1
    d = _scan(x=lanes, input_gate=lanes, decay_gate=lanes, kept_steps=16)
    none = _lib.Stream(data=None, batch_stride=0, step_stride=0)
    assert lib.pesq_gated_scan_backward(ctypes.byref(d), None, one, 1 << 30, none, None, one, one, one, one, None, one,
                                        1 << 30) == 1
    assert "too far apart" in _lib.last_error()


def test_rates_that_no_call_takes_are_refused_by_the_module():
    for rate in (1.1e6, float("inf"), float("nan"), -1.0):
        with pytest.raises(ValueError, match="1e6"):
            GatedScanCuda(4, rate=rate)
    assert _sizes(_scan(rate=1e6))[0] == _lib.PESQ_OK
    assert _sizes(_scan(rate=1.1e6))[0] == _lib.PESQ_ERR_INVALID_ARGUMENT and "1e6" in _lib.last_error()
