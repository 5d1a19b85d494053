"""``norm_join`` / ``NormJoinCuda``: what lies between two blocks of a network,
in one pass over the data (csrc/norm_join.cuh)::

    stream' = stream + scale * act(gate) * post_weight * block / rms(block)
    normed = pre_weight * stream' / rms(stream')

with ``rms(v) = sqrt(mean(v**2) + eps)`` over the channels.  ``pre_norm`` is the
norm alone, for the first block.  Sums and statistics are float32; the stream may be
float32 beside 16-bit blocks.  The reference has no counterpart (its networks are
its users').
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

__all__ = ["norm_join", "pre_norm", "NormJoinCuda"]

ACTIVATIONS = ("sigmoid", "silu")
_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}

_op = None


def _load():
    global _op
    if _op is None:
        _lib.load_ops()
        _op = torch.ops.pesq_cuda.norm_join.default
    return _op


def _code(dtype) -> int:
    code = _CODES.get(dtype)
    if code is None:
        raise RuntimeError(f"The CUDA norm join supports float32, bfloat16 and float16, not {dtype}.")
    return code


def norm_join(stream: torch.Tensor, block: torch.Tensor, post_weight: torch.Tensor, pre_weight: torch.Tensor, *,
              gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, eps: float = 1e-6,
              activation: str = "sigmoid") -> Tuple[torch.Tensor, torch.Tensor]:
    """Join a block's output with the residual stream, and norm it for the next block.

    Parameters
    ----------
    stream
        ``[batch, step, channel]``, float32 or of the block's type; at most 8192
        channels, any strides (a tensor whose channels are not adjacent is copied).
    block
        The block's output, the same shape, float32, bfloat16 or float16.
    post_weight, pre_weight
        float32 ``[channel]``: of the norm after the block and before the next.
    gate
        Logits in the block's type, of its shape or broadcast to it; ``[batch, 1,
        channel]`` is one gate for all steps, whose gradient the kernels sum.
    scale
        float32 ``[channel]``: the residual scale.
    activation
        ``"sigmoid"`` or ``"silu"``, of the gate.

    Returns
    -------
    ``(stream', normed)``, in the types of ``stream`` and ``block``.  Differentiable
    once, in reverse mode, in every operand.
    """

    op = _op or _load()
    if not isinstance(stream, torch.Tensor) or not isinstance(block, torch.Tensor):
        raise TypeError("`stream` and `block` must be torch.Tensors")
    if activation not in ACTIVATIONS:
        raise ValueError(f"Unknown activation `{activation}`, pick one of {ACTIVATIONS}.")
    return op(stream, block, gate, post_weight, pre_weight, scale, eps, activation == "silu", _code(block.dtype))


def pre_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6,
             dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``weight * x / rms(x)`` over the channels of ``[batch, step, channel]``,
    in ``dtype`` (the type of ``x``; 16 bits beside a float32 ``x``)."""

    op = _op or _load()
    if not isinstance(x, torch.Tensor):
        raise TypeError("`x` must be a torch.Tensor")
    return op(x, None, None, None, weight, None, eps, False, _code(x.dtype if dtype is None else dtype))[1]


class NormJoinCuda(torch.nn.Module):
    """The join with its parameters.

    Parameters
    ----------
    channels : int
        Width of the stream, at most 8192
    eps : float
        Added to the mean square
    activation : str
        ``"sigmoid"`` or ``"silu"``, of the gate
    scale : Optional[float]
        Initial residual scale, ``None`` for a join without one

    Attributes
    ----------
    post_weight, pre_weight : torch.nn.Parameter
        float32 ``[channels]``, ones
    scale : Optional[torch.nn.Parameter]
        float32 ``[channels]``; the vectors of a module in 16 bits are widened for the call
    """

    def __init__(self, channels: int, eps: float = 1e-6, activation: str = "sigmoid", scale: Optional[float] = 1.0):
        super().__init__()
        if not 1 <= int(channels) <= 8192:
            raise ValueError("`channels` has to be between 1 and 8192.")
        if activation not in ACTIVATIONS:
            raise ValueError(f"Unknown activation `{activation}`, pick one of {ACTIVATIONS}.")
        if not eps >= 0:
            raise ValueError("`eps` must not be negative.")
        self.channels, self.eps, self.activation = int(channels), float(eps), activation
        self.post_weight = torch.nn.Parameter(torch.ones(self.channels))
        self.pre_weight = torch.nn.Parameter(torch.ones(self.channels))
        self.scale = None if scale is None else torch.nn.Parameter(torch.full((self.channels,), float(scale)))
        _load()

    def forward(self, stream: torch.Tensor, block: torch.Tensor,
                gate: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """See :func:`norm_join`."""

        return norm_join(stream, block, _lib.widened(self.post_weight), _lib.widened(self.pre_weight), gate=gate,
                         scale=_lib.widened(self.scale), eps=self.eps, activation=self.activation)

    def extra_repr(self) -> str:
        return f"channels={self.channels}, eps={self.eps}, activation={self.activation}"
