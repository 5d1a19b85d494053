"""``muon_step`` / ``MuonCuda``: updates of matrices orthogonalised by
Newton-Schulz products, for all matrices together (csrc/muon.cu); ``orthogonalize``
is the iteration alone::

    m = b m + (1 - b) g,  u = b m + (1 - b) g
    x = u / max(|u|, eps)
    steps times:  a = x x^T,  x = c0 x + (c1 a + c2 a a) x
    p = p (1 - lr wd) - lr adjust x

(on the shorter side of a matrix).  Every product runs on the tensor cores with
operands of two float16 terms and float32 sums: the iteration enlarges small singular values,
and rounding with them, by up to 485.  Vectors are for :class:`~triton_pesq_b200.adamw.AdamWCuda`.  The reference has no
optimiser.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _lib

__all__ = ["orthogonalize", "muon_step", "MuonCuda", "COEFFICIENTS"]

#: of the usual five steps, which bring singular values from 0.01 on to between 0.7 and 1.2
COEFFICIENTS = (3.4445, -4.775, 2.0315)
ADJUSTMENTS = ("original", "match_rms_adamw")
#: of a parameter group
HYPERPARAMETERS = frozenset(("lr", "momentum", "nesterov", "weight_decay", "coefficients", "eps", "steps", "adjust"))

_ops = None


def _load():
    global _ops
    if _ops is None:
        _lib.load_ops()
        _ops = (torch.ops.pesq_cuda.muon_step.default, torch.ops.pesq_cuda.orthogonalize.default)
    return _ops


def orthogonalize(x: torch.Tensor, *, coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7,
                  steps: int = 5) -> torch.Tensor:
    """The matrices ``[..., row, column]`` with their singular values near 1.

    Parameters
    ----------
    x
        float32, bfloat16 or float16, up to 32768 rows and columns.
    coefficients
        Of the polynomial ``c0 + c1 s^2 + c2 s^4`` of the singular values s, each between -16 and 16.  The values, the polynomial on
        them and ``c1 + c2 s^2`` have to stay below 60, the operands' range: a result of larger ones is not finite.
    eps
        Least norm that a matrix is divided by, 1.2e-38 or more.
    steps
        Between 1 and 100.

    Returns
    -------
    A dense tensor of the shape and type of ``x``, without a gradient.
    """

    if not isinstance(x, torch.Tensor):
        raise TypeError("`x` must be a torch.Tensor")
    return (_ops or _load())[1](x.detach(), *coefficients, eps, steps)


def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momenta: Sequence[torch.Tensor], *,
              copies: Optional[Sequence[torch.Tensor]] = None, lr: float = 1e-3, momentum: float = 0.95,
              nesterov: bool = True, weight_decay: float = 0.1, coefficients: Tuple[float, float, float] = COEFFICIENTS,
              eps: float = 1e-7, steps: int = 5, adjust: str = "original",
              grad_scale: Optional[torch.Tensor] = None) -> None:
    """One Muon step in place.

    Parameters
    ----------
    params
        Float32 matrices on one GPU, dense in the order of their dimensions, each given once: what is written must not
        share memory.
    grads
        Their gradients, all float32, bfloat16 or float16 (dense, or they are
        copied).  An empty tensor leaves its matrix and momentum as they are.
    momenta
        Float32 tensors of the matrices' shapes, zeros before the first step.
    copies
        The matrices in the gradients' 16-bit type, written along.
    lr, momentum, nesterov, weight_decay
        As in ``torch.optim.Muon``.
    coefficients, eps, steps
        As in :func:`orthogonalize`.
    adjust
        ``"original"``: the rate times ``sqrt(max(1, rows / columns))``;
        ``"match_rms_adamw"``: times ``0.2 sqrt(max(rows, columns))``.
    grad_scale
        One float32 value on the GPU that multiplies every gradient (an unscaling
        factor).  Where it is not finite the step is skipped whole.
    """

    if adjust not in ADJUSTMENTS:
        raise ValueError(f"Unknown adjustment `{adjust}`, pick one of {ADJUSTMENTS}.")
    if not params and not grads and not momenta and not copies:
        return
    (_ops or _load())[0](params, grads, momenta, [] if copies is None else copies, lr, momentum, nesterov, weight_decay,
                         *coefficients, eps, steps, ADJUSTMENTS.index(adjust), grad_scale)


class MuonCuda(torch.optim.Optimizer):
    """Muon whose step takes all matrices of a parameter group (and type) together.

    Parameters
    ----------
    params
        Matrices or parameter groups of them, on GPUs, dense in the order of their dimensions, up to 32768 rows and columns:
        float32, or bfloat16 / float16, which are then the rounded copies of float32 masters in the state.
    lr, momentum, nesterov, weight_decay, coefficients, eps, steps, adjust
        As in :func:`muon_step`; each may differ between groups.

    A captured step keeps the hyperparameters it was captured with; the first step makes the state and is refused
    in a capture.  16-bit parameters are written from their masters by every step: what else writes to them after the first step
    is lost, unless it writes to ``state[p]["master"]`` too.
    """

    def __init__(self, params, lr: float = 1e-3, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.1,
                 coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7, steps: int = 5,
                 adjust: str = "original"):
        if not lr >= 0 or not weight_decay >= 0:
            raise ValueError("`lr` and `weight_decay` must not be negative.")
        if not 0 <= momentum < 1:
            raise ValueError("`momentum` has to lie in [0, 1).")
        if len(coefficients) != 3 or not all(abs(c) <= 16 for c in coefficients):
            raise ValueError("`coefficients` have to be three values between -16 and 16.")
        if not torch.finfo(torch.float32).tiny <= eps < float("inf"):
            raise ValueError("`eps` has to be positive, finite and no subnormal.")
        if not 1 <= int(steps) <= 100:
            raise ValueError("`steps` has to lie between 1 and 100.")
        if adjust not in ADJUSTMENTS:
            raise ValueError(f"Unknown adjustment `{adjust}`, pick one of {ADJUSTMENTS}.")
        _load()
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=bool(nesterov), weight_decay=weight_decay,
                                      coefficients=tuple(coefficients), eps=eps, steps=int(steps), adjust=adjust))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            why = None
            if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                why = f"MuonCuda supports float32, bfloat16 and float16 parameters, not {p.dtype}."
            elif p.dim() != 2 or not all(1 <= n <= 32768 for n in p.shape):
                why = f"MuonCuda needs matrices of up to 32768 rows and columns, got shape {tuple(p.shape)}."
            elif not p.is_contiguous():
                why = (f"MuonCuda needs dense parameters in the order of their dimensions, got shape {tuple(p.shape)} "
                       f"with strides {p.stride()}.")
            if why:
                self.param_groups.pop()
                raise RuntimeError(why)

    def _state(self, p: torch.Tensor) -> dict:
        state = self.state[p]
        if not state:
            if torch.cuda.is_current_stream_capturing():
                # (a graph would take the state's making along, and every replay would begin anew)
                del self.state[p]
                raise RuntimeError("The first step of a MuonCuda makes its state and cannot be captured: take one before.")
            state["momentum"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            if p.dtype != torch.float32:
                state["master"] = p.detach().float()
        return state

    def load_state_dict(self, state_dict) -> None:
        """Takes the state of a ``MuonCuda`` on parameters of the same types and sizes; anything else is refused with a
        ``ValueError`` and changes nothing."""

        for g in state_dict["param_groups"]:
            missing = sorted(HYPERPARAMETERS - set(g))
            if missing:
                raise ValueError(f"These are not the parameter groups of a MuonCuda: {missing} are missing.")
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        kept = {}
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                state = state_dict["state"][i]
                want = {"momentum"} | ({"master"} if p.dtype != torch.float32 else set())
                if set(state) != want or any(not isinstance(v, torch.Tensor) or v.dtype != torch.float32 or v.shape != p.shape
                                             for v in state.values()):
                    raise ValueError(f"This is not the state of a parameter of MuonCuda: needs {sorted(want)} in float32 of shape "
                                     f"{tuple(p.shape)}.")
                kept[p] = {k: v.detach().to(p.device, copy=True).contiguous() for k, v in state.items()}
        # (the base class would cast float32 state to the parameters' type)
        super().load_state_dict({**state_dict, "state": {}})
        self.state.update(kept)

    def __setstate__(self, state: dict) -> None:
        _load()
        super().__setstate__(state)

    @torch.no_grad()
    def step(self, closure=None, grad_scale: Optional[torch.Tensor] = None):
        """One step; ``grad_scale`` as in :func:`muon_step`."""

        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            kinds = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not p.is_cuda:
                    raise RuntimeError("MuonCuda needs its parameters to live on a GPU.")
                kinds.setdefault((p.device, p.dtype, p.grad.dtype), []).append(p)
            for (_, dtype, _), params in kinds.items():
                states = [self._state(p) for p in params]
                masters = dtype != torch.float32
                muon_step([s["master"] for s in states] if masters else params, [p.grad for p in params],
                          [s["momentum"] for s in states], copies=params if masters else None,
                          **{k: group[k] for k in HYPERPARAMETERS}, grad_scale=grad_scale)
        return loss

    def check_errors(self) -> int:
        """Synchronise and return the error word of the first parameter's device (nonzero
        if a bounded wait of an earlier step ran out)."""

        with torch.cuda.device(self.param_groups[0]["params"][0].device):
            return _lib.muon_check(torch.cuda.current_stream().cuda_stream)
