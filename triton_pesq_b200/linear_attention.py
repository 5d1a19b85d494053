"""``linear_attention`` / ``LinearAttentionCuda``: linear attention with a decay
for each head, the recurrence of :mod:`~triton_pesq_b200.gated_scan` with a
matrix as its state.

Per row and head, in scan order::

    S = exp(log_decay) * S + outer(k, v),   y = scale * q @ S

Sequences run in chunks of 64 steps on the tensor cores, and in parts that are
joined where rows are few; a call of a few steps with ``state`` is the streaming form
(csrc/linear_attention.cuh).  The state, the decays and every sum are float32
whatever the streams' type.  Products take what was computed as terms: all
bits of it where the result is float32 beside bfloat16, 2^-18 of it left out where the
result is rounded to bfloat16 itself, 2^-22 beside float16 and float32.  A result is the same,
to the last bit, every time.  The reference has no counterpart (its networks are its users').
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

__all__ = ["linear_attention", "LinearAttentionCuda"]

_op = None


def _load():
    global _op
    if _op is None:
        _lib.load_ops()
        _op = torch.ops.pesq_cuda.linear_attention.default
    return _op


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                     state: Optional[torch.Tensor] = None, *, reset: Optional[torch.Tensor] = None,
                     lengths: Optional[torch.Tensor] = None, reverse: bool = False,
                     scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Linear attention with a decay for each head, along dimension 1.

    Parameters
    ----------
    q, k
        ``[batch, step, head, key]``, float32, bfloat16 or float16, one type, up to 128 channels and 2^22 heads over the batch.  Any strides:
        slices of one projection, or heads that are shared by expansion, are read where they lie (a tensor whose channels
        are not adjacent is copied).
    v
        ``[batch, step, head, value]`` in their type, up to 128 channels.
    log_decay
        float32 ``[head]``, or ``[batch, step, head]`` for decays that the data sets: the logarithm of the factor
        that the state takes at a step, 0 or less (-inf forgets it).
    state
        float32 ``[batch, head, key, value]``, the state before the first step (zeros).
    reset
        bool ``[batch, step]``: the step forgets the state, so that several utterances can share a row.
    lengths
        int64 or int32 ``[batch]``: steps at or past a row's length leave its state as it is and give ``y = 0``;
        what the inputs hold there is not read.
    reverse
        Scan from the last step to the first.
    scale
        Factor of the result.

    Returns
    -------
    ``(y, last)``: ``[batch, step, head, value]`` in the type of ``v``, and the float32 state after the last step.
    Differentiable once, in reverse mode, in all inputs but the masks.

    Inputs have to be finite (but for ``log_decay``, and where ``lengths`` masks them): a step's value that is not may
    reach every step of its chunk of 64, earlier ones and those behind a reset too.
    """

    op = _op or _load()
    if not isinstance(q, torch.Tensor):
        raise TypeError("`q` must be a torch.Tensor")
    return op(q, k, v, log_decay, state, reset, lengths, reverse, scale)


class LinearAttentionCuda(torch.nn.Module):
    """The attention with a learned decay for each head.

    Parameters
    ----------
    heads : int
        Number of heads
    key : int
        Channels of a head's queries and keys, at most 128; the result is scaled by ``key**-0.5``
    reverse : bool
        Scan from the last step to the first
    fast, slow : float
        The initial decays: their distances from 1 are spaced evenly in the logarithm between these values' distances

    Attributes
    ----------
    decay : torch.nn.Parameter
        float32 ``[heads]``: the log decay is ``-softplus(decay)``; of a module in 16 bits it is widened for the call
    """

    def __init__(self, heads: int, key: int, reverse: bool = False, fast: float = 0.875, slow: float = 0.998):
        super().__init__()
        if int(heads) < 1:
            raise ValueError("`heads` has to be positive.")
        if not 1 <= int(key) <= 128:
            raise ValueError("`key` has to be between 1 and 128.")
        if not 0 < fast <= slow < 1:
            raise ValueError("The initial decays have to satisfy 0 < fast <= slow < 1.")
        self.heads, self.key, self.reverse = int(heads), int(key), bool(reverse)
        ends = torch.log(1 - torch.tensor([fast, slow], dtype=torch.float64))
        decay = 1 - torch.exp(torch.linspace(float(ends[0]), float(ends[1]), self.heads, dtype=torch.float64))
        self.decay = torch.nn.Parameter(torch.log(torch.expm1(-torch.log(decay))).float())
        _load()

    def log_decay(self) -> torch.Tensor:
        """The heads' log decays, float32 ``[heads]``."""

        return -torch.nn.functional.softplus(_lib.widened(self.decay))

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, state: Optional[torch.Tensor] = None,
                reset: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Sequences ``[batch, step, head, channel]``; see :func:`linear_attention`."""

        return linear_attention(q, k, v, self.log_decay(), state, reset=reset, lengths=lengths, reverse=self.reverse,
                                scale=self.key**-0.5)

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
             state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """One step ``[batch, head, channel]`` of a stream: its output and the state after it."""

        y, last = self(q.unsqueeze(1), k.unsqueeze(1), v.unsqueeze(1), state)
        return y.squeeze(1), last

    def extra_repr(self) -> str:
        return f"heads={self.heads}, key={self.key}, reverse={self.reverse}"
