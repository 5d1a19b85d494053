"""``adamw_step`` / ``AdamWCuda``: one AdamW step over many tensors in one
launch (csrc/adamw.cu), with moments in 32 or in 8 bits::

    m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g**2
    p = p (1 - lr wd) - lr / (1 - b1**t) m / (sqrt(v / (1 - b2**t)) + eps)

The moments of all tensors lie in two flat buffers, a tensor's part beginning at
a multiple of 256 values.  With 8 bits they are ``float8_e4m3fn`` in units of one
float32 scale per 256 values (``scales[0]`` and ``scales[1]``), the second moment
as its root.  Nearest rounding would hold what moves by less than half a rounding
step at a time for good: that root, which changes by 1 / 2000 of itself a step, and the
first moment where it is small (or ``b1`` above 15/16) and moves that little are rounded
stochastically (a hash of position, step and ``seed``).  The step count is on the device, so a
step can be captured in a CUDA graph.  The reference has no optimiser.
"""

from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib

__all__ = ["adamw_step", "AdamWCuda", "BLOCK"]

#: values that share a scale, and the unit that a tensor's part of the moments is a multiple of
BLOCK = 256

_op = None


def _load():
    global _op
    if _op is None:
        _lib.load_ops()
        _op = torch.ops.pesq_cuda.adamw_step.default
    return _op


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], moment1: torch.Tensor,
               moment2: torch.Tensor, step: torch.Tensor, *, scales: Optional[torch.Tensor] = None,
               copies: Optional[Sequence[torch.Tensor]] = None, lr: float = 1e-3,
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               grad_scale: Optional[torch.Tensor] = None, seed: int = 0) -> None:
    """One AdamW step in place.

    Parameters
    ----------
    params
        Float32 tensors on one GPU, dense in the order of their dimensions.
    grads
        Their gradients, all float32, bfloat16 or float16 (dense, or they are
        copied).  An empty tensor leaves its parameter and moments as they are.
    moment1, moment2
        Flat buffers of at least the sum of the parameters' sizes, each rounded up
        to 256 values: float32, or float8_e4m3fn with ``scales``.
    step
        int64 ``[2]``: the steps taken, counted on by the call, and 0.
    scales
        float32 ``[2, moment1.numel() // 256]``, for 8-bit moments.
    copies
        The parameters in the gradients' 16-bit type, written along.
    grad_scale
        One float32 value on the GPU that multiplies every gradient (an unscaling
        or clipping factor).  Where it is not finite the step is skipped whole.
    seed
        Of the 8-bit moments' stochastic rounding.
    """

    (_op or _load())(params, grads, moment1, moment2, step, scales, [] if copies is None else copies, lr, betas[0],
                     betas[1], eps, weight_decay, grad_scale, seed)


class _Flat:
    """The parameters of a group that step together, and their state."""

    def __init__(self, params: List[torch.Tensor], bits: int):
        first = params[0]
        sizes = [-(-p.numel() // BLOCK) * BLOCK for p in params]
        self.params, self.total = params, sum(sizes)
        self.starts = [sum(sizes[:i]) for i in range(len(sizes))]
        dtype = torch.float32 if bits == 32 else torch.float8_e4m3fn
        make = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=first.device)  # noqa: E731
        self.moment1, self.moment2 = make(self.total, dtype=dtype), make(self.total, dtype=dtype)
        self.scales = make(2, self.total // BLOCK) if bits == 8 else None
        self.step = make(2, dtype=torch.int64)
        self.masters = None
        if first.dtype != torch.float32:
            flat = make(self.total)
            self.masters = [flat[o:o + p.numel()].view(p.shape) for o, p in zip(self.starts, params)]
            for m, p in zip(self.masters, params):
                m.copy_(p)

    def state(self, i: int) -> dict:
        """Views of parameter i's state, as the optimiser's ``state`` shows them."""

        lo, n = self.starts[i], self.params[i].numel()
        hi = lo + -(-n // BLOCK) * BLOCK
        out = {"step": self.step, "moment1": self.moment1[lo:hi], "moment2": self.moment2[lo:hi]}
        if self.scales is not None:
            out["scales"] = self.scales[:, lo // BLOCK:hi // BLOCK]
        if self.masters is not None:
            out["master"] = self.masters[i]
        return out


class AdamWCuda(torch.optim.Optimizer):
    """AdamW whose step is one launch a parameter group (and type).

    Parameters
    ----------
    params
        Parameters or parameter groups, on GPUs, dense in the order of their
        dimensions (channels-last weights are not): float32, or bfloat16 / float16,
        which are then the rounded copies of float32 masters in the state.
    lr, betas, eps, weight_decay
        As in ``torch.optim.AdamW``; each may differ between groups.
    state_bits : int
        32, or 8 for float8 moments with a scale per 256 values
    seed : int
        Of the 8-bit moments' stochastic rounding

    The step count is one for all parameters of a group and type, so a parameter
    that had no gradient at first is corrected as if it had been zero.  A captured
    step keeps the hyperparameters it was captured with; the first step, and the first after
    ``load_state_dict``, make the state's buffers and are refused in a capture.  16-bit parameters are written from
    their masters by every step: what else writes to them after the first step is lost, unless
    it writes to ``state[p]["master"]`` too.
    """

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError("`state_bits` has to be 8 or 32.")
        if not lr >= 0 or not eps >= 0 or not weight_decay >= 0:
            raise ValueError("`lr`, `eps` and `weight_decay` must not be negative.")
        if not all(0 <= b < 1 for b in betas):
            raise ValueError("`betas` have to lie in [0, 1).")
        self.state_bits, self.seed = int(state_bits), int(seed)
        self._flats: Dict[int, List[_Flat]] = {}
        _load()
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            why = None
            if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                why = f"AdamWCuda supports float32, bfloat16 and float16 parameters, not {p.dtype}."
            elif not p.is_contiguous():
                why = (f"AdamWCuda needs dense parameters in the order of their dimensions, got shape {tuple(p.shape)} "
                       f"with strides {p.stride()}.")
            if why:
                self.param_groups.pop()
                raise RuntimeError(why)

    def _flat(self, index: int) -> List[_Flat]:
        flats = self._flats.get(index)
        if flats is None:
            kinds: Dict[tuple, List[torch.Tensor]] = {}
            for p in self.param_groups[index]["params"]:
                if not p.is_cuda:
                    raise RuntimeError("AdamWCuda needs its parameters to live on a GPU.")
                kinds.setdefault((p.device, p.dtype), []).append(p)
            if kinds and torch.cuda.is_current_stream_capturing():
                # (a graph would take the state's making along, and every replay would begin anew)
                raise RuntimeError("The first step of an AdamWCuda makes its state and cannot be captured: take one before.")
            flats = self._flats[index] = [_Flat(ps, self.state_bits) for ps in kinds.values()]
            for f in flats:
                for i, p in enumerate(f.params):
                    loaded, views = self.state.get(p), f.state(i)
                    if loaded:  # (a state that was loaded moves into the buffers)
                        for k, v in views.items():
                            v.copy_(loaded[k])
                    self.state[p] = views
        return flats

    def _check_state(self, p: torch.Tensor, state: dict) -> None:
        units = -(-p.numel() // BLOCK)
        moment = torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
        want = {"step": (torch.int64, (2,)), "moment1": (moment, (BLOCK * units,)), "moment2": (moment, (BLOCK * units,))}
        if self.state_bits == 8:
            want["scales"] = (torch.float32, (2, units))
        if p.dtype != torch.float32:
            want["master"] = (torch.float32, tuple(p.shape))
        got = {k: (v.dtype, tuple(v.shape)) if isinstance(v, torch.Tensor) else type(v) for k, v in state.items()}
        if got != want:
            raise ValueError(f"This is not the state of a parameter of AdamWCuda with state_bits={self.state_bits}: needs "
                             f"{want}, got {got}.")

    def load_state_dict(self, state_dict) -> None:
        """Takes the state of an ``AdamWCuda`` of the same ``state_bits`` on parameters of the same types and sizes;
        anything else is refused with a ``ValueError`` and changes nothing."""

        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        kept = {}
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                state = state_dict["state"][i]
                self._check_state(p, state)
                kept[p] = {k: v.detach().to(p.device, copy=True) for k, v in state.items()}
        # (the base class would cast float8 and int64 state to the parameters' type)
        super().load_state_dict({**state_dict, "state": {}})
        self.state.update(kept)

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "state_bits": self.state_bits, "seed": self.seed}

    def __setstate__(self, state: dict) -> None:
        _load()
        self._flats = {}  # (made from the state by the next step)
        super().__setstate__(state)

    @torch.no_grad()
    def step(self, closure=None, grad_scale: Optional[torch.Tensor] = None):
        """One step; ``grad_scale`` as in :func:`adamw_step`."""

        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for index, group in enumerate(self.param_groups):
            for f in self._flat(index):
                grads = [p.grad if p.grad is not None else p.new_empty(0) for p in f.params]
                if all(p.grad is None for p in f.params):
                    continue
                adamw_step(f.params if f.masters is None else f.masters, grads, f.moment1, f.moment2, f.step,
                           scales=f.scales, copies=None if f.masters is None else f.params, lr=group["lr"],
                           betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                           grad_scale=grad_scale, seed=self.seed)
        return loss
