"""``layer_norm`` / ``LayerNormCuda``: layer norm with its gradients, beside the
rms norms of :mod:`~triton_pesq_b200.norm_join` (csrc/layer_norm.cuh)::

    y = (x - mean(x)) / sqrt(mean((x - mean(x))**2) + eps) * weight + bias

over the last dimension, with one weight for all rows, or one for each head of
``[..., head, channel]`` (the norm of an attention's heads).  Statistics and sums
are float32, and a result is the same, to the last bit, every time.  The reference has no counterpart (its networks
are its users').
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

__all__ = ["layer_norm", "LayerNormCuda"]

_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}

_op = None


def _load():
    global _op
    if _op is None:
        _lib.load_ops()
        _op = torch.ops.pesq_cuda.layer_norm.default
    return _op


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
               dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Layer norm over the last dimension.

    Parameters
    ----------
    x
        ``[..., channel]``, float32, bfloat16 or float16, at most 8192 channels.  Of up to three dimensions
        (four with heads) any strides are read where they lie; a tensor whose channels are not adjacent is copied.
    weight, bias
        float32 ``[channel]``, or ``[head, channel]`` for ``x`` of ``[..., head, channel]`` (up to 2**20 values).
    eps
        Added to the mean square.
    dtype
        Of the result: the type of ``x``, or 16 bits beside a float32 ``x``.

    Returns
    -------
    A tensor of the shape of ``x``.  Differentiable once, in reverse mode, in ``x``, ``weight`` and ``bias``.
    """

    op = _op or _load()
    if not isinstance(x, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("`x` and `weight` must be torch.Tensors")
    code = -1
    if dtype is not None:
        code = _CODES.get(dtype)
        if code is None:
            raise RuntimeError(f"The CUDA layer norm supports float32, bfloat16 and float16, not {dtype}.")
    return op(x, weight, bias, eps, code)


class LayerNormCuda(torch.nn.Module):
    """The norm with its parameters.

    Parameters
    ----------
    channels : int
        Width of the last dimension, at most 8192
    heads : Optional[int]
        Heads of ``[..., head, channel]`` with a weight each, ``None`` for one weight
    eps : float
        Added to the mean square
    bias : bool
        Whether there is a bias

    Attributes
    ----------
    weight, bias : torch.nn.Parameter
        float32 ``[channels]`` or ``[heads, channels]``, ones and zeros; of a module in 16 bits they are widened for the call
    """

    def __init__(self, channels: int, heads: Optional[int] = None, eps: float = 1e-5, bias: bool = True):
        super().__init__()
        if not 1 <= int(channels) <= 8192:
            raise ValueError("`channels` has to be between 1 and 8192.")
        if heads is not None and not 1 <= int(heads) <= (1 << 20) // int(channels):
            raise ValueError("`heads` has to be positive, and `heads` times `channels` at most 2**20.")
        if not eps >= 0:
            raise ValueError("`eps` must not be negative.")
        self.channels, self.heads, self.eps = int(channels), None if heads is None else int(heads), float(eps)
        shape = (self.channels,) if heads is None else (self.heads, self.channels)
        self.weight = torch.nn.Parameter(torch.ones(shape))
        self.bias = torch.nn.Parameter(torch.zeros(shape)) if bias else None
        _load()

    def forward(self, x: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """See :func:`layer_norm`."""

        return layer_norm(x, _lib.widened(self.weight), _lib.widened(self.bias), eps=self.eps, dtype=dtype)

    def extra_repr(self) -> str:
        return f"channels={self.channels}, heads={self.heads}, eps={self.eps}, bias={self.bias is not None}"
