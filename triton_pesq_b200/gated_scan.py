"""``gated_scan`` / ``GatedScanCuda``: a gated linear recurrence over long
sequences, the time-varying sibling of :class:`~triton_pesq_b200.iir.IIRCuda`
for the networks that are trained on the loss.

Per row and channel, in scan order::

    r = sigmoid(decay_gate),  i = sigmoid(input_gate)
    log a = -rate * softplus(decay) * r
    h = a * h + sqrt(1 - a**2) * i * x,   y = h

Rows and channels side by side, and steps in strips where those are few
(csrc/gated_scan.cuh); the state, the gates and every sum are float32 whatever
the streams' type, and a result is the same, to the last bit, every time.  A call of one step
with ``state`` is the streaming form.  The reference has fixed-coefficient
recurrences only (torch_pesq/triton_ops/iir.py).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

__all__ = ["gated_scan", "GatedScanCuda"]

_op = None


def _load():
    global _op
    if _op is None:
        _lib.load_ops()
        _op = torch.ops.pesq_cuda.gated_scan.default
    return _op


def gated_scan(x: torch.Tensor, input_gate: torch.Tensor, decay_gate: torch.Tensor, decay: torch.Tensor,
               state: Optional[torch.Tensor] = None, *, reset: Optional[torch.Tensor] = None,
               lengths: Optional[torch.Tensor] = None, reverse: bool = False,
               rate: float = 8.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gated linear recurrence along dimension 1.

    Parameters
    ----------
    x, input_gate, decay_gate
        ``[batch, step, channel]``, float32, bfloat16 or float16, one type, up to 2**24 channels.  Any
        strides: slices of one projection are read where they lie (a tensor
        whose channels are not adjacent is copied).  The gates are logits.
    decay
        float32 ``[channel]``.
    state
        float32 ``[batch, channel]``, the state before the first step (zeros).
    reset
        bool ``[batch, step]``: the step forgets the state (``a = 0`` whatever its decay gate), so that
        several utterances can share a row.
    lengths
        int64 or int32 ``[batch]``: steps at or past a row's length leave its
        state as it is and give ``y = 0``; what the inputs hold there is not read.
    reverse
        Scan from the last step to the first.
    rate
        Factor of the log decay, above 0 and up to 1e6.

    Returns
    -------
    ``(y, last)``: ``[batch, step, channel]`` in the type of ``x``, and the
    float32 state after the last step.  Differentiable once, in reverse mode, in all inputs but
    the masks.
    """

    op = _op or _load()
    if not isinstance(x, torch.Tensor):
        raise TypeError("`x` must be a torch.Tensor")
    return op(x, input_gate, decay_gate, decay, state, reset, lengths, reverse, rate)


class GatedScanCuda(torch.nn.Module):
    """The recurrence with its decay parameter.

    Parameters
    ----------
    channels : int
        Width of the recurrence
    rate : float
        Factor of the log decay, above 0 and up to 1e6
    reverse : bool
        Scan from the last step to the first
    fast, slow : float
        The initial decays are uniform between these values at an open gate

    Attributes
    ----------
    decay : torch.nn.Parameter
        float32 ``[channels]``; of a module in 16 bits it is widened for the call
    """

    def __init__(self, channels: int, rate: float = 8.0, reverse: bool = False, fast: float = 0.9,
                 slow: float = 0.999):
        super().__init__()
        if int(channels) < 1:
            raise ValueError("`channels` has to be positive.")
        if not 0 < rate <= 1e6:
            raise ValueError("`rate` has to lie above 0 and not above 1e6.")
        if not 0 < fast <= slow < 1:
            raise ValueError("The initial decays have to satisfy 0 < fast <= slow < 1.")
        self.channels, self.rate, self.reverse = int(channels), float(rate), bool(reverse)
        a = fast + (slow - fast) * torch.rand(self.channels, dtype=torch.float64)
        self.decay = torch.nn.Parameter(torch.log(torch.expm1(-torch.log(a) / self.rate)).float())
        _load()

    def forward(self, x: torch.Tensor, input_gate: torch.Tensor, decay_gate: torch.Tensor,
                state: Optional[torch.Tensor] = None, reset: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Sequences ``[batch, step, channel]``; see :func:`gated_scan`."""

        return gated_scan(x, input_gate, decay_gate, _lib.widened(self.decay), state, reset=reset, lengths=lengths,
                          reverse=self.reverse, rate=self.rate)

    def step(self, x: torch.Tensor, input_gate: torch.Tensor, decay_gate: torch.Tensor,
             state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """One step ``[batch, channel]`` of a stream: its output and the state after it."""

        y, last = self(x.unsqueeze(1), input_gate.unsqueeze(1), decay_gate.unsqueeze(1), state)
        return y.squeeze(1), last

    def check_errors(self) -> int:
        """Synchronise and return the error word of the parameter's device (nonzero
        if an earlier call's copies into shared memory did not come in time)."""

        with torch.cuda.device(self.decay.device):
            return _lib.gated_scan_check(torch.cuda.current_stream().cuda_stream)

    def extra_repr(self) -> str:
        return f"channels={self.channels}, rate={self.rate}, reverse={self.reverse}"
