"""A Muon step works on all matrices at the same time: what two of them would write is refused before any launch.  (The
addresses are not memory: skipped where there is a GPU, so that nothing is ever launched on them.)"""

import ctypes

import pytest
import torch

from triton_pesq_b200 import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="a call that is not refused would be launched")

ROWS, COLS = 32, 64
BYTES = ROWS * COLS * 4


def step(*tensors):
    """The answer to a step over (param, momentum, copy), with bfloat16 gradients."""

    d = _lib.MuonDesc(grad_dtype=_lib.BF16, nesterov=1, adjust=0, steps=5, momentum=0.95, lr=0.02, weight_decay=0.1, eps=1e-7, a=3.4, b=-4.8, c=2.0)
    table = (_lib.MuonTensor * len(tensors))(*(_lib.MuonTensor(param=p, grad=1 << 40, momentum=m, copy=c, rows=ROWS, cols=COLS) for p, m, c in tensors))
    return _lib.library().pesq_muon_step(ctypes.byref(d), table, len(tensors), None, ctypes.c_void_p(1 << 41), 1 << 40)


def test_what_is_written_twice_is_refused():
    a, b, c, d = (BYTES * k for k in range(1, 5))
    for bad in ([(a, b, None), (a, c, None)], [(a, b, None), (c, b, None)], [(a, a, None)], [(a, b, a)], [(a, b, c), (d, 5 * BYTES, c)],
                [(a, c, None), (a + BYTES - 4, 8 * BYTES, None)], [(a, c, None), (8 * BYTES, 9 * BYTES, c - BYTES // 2 + 2)]):
        assert step(*bad) == 1, bad
    # neighbours in one buffer get as far as the launch, which there is no device for
    assert step((a, b, c), (c + BYTES // 2, d + BYTES // 2, 8 * BYTES)) == 4
