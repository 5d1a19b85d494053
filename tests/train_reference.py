"""Definitions of the training operators in 64 bits (torch on the CPU, one
step or row at a time; gradients by autograd), and how far an output may be
from them."""

import torch

#: unit roundoff of an output's type: one rounding at the end, relative
ROUND = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def close(got, want, tol, what="", terms=None):
    """|got - want| is at most one rounding to got's type, with a quarter to
    spare, plus ``tol`` of the largest value: what the 32-bit arithmetic before
    that rounding may be off by.  Where the value is a difference of larger
    ``terms``, that arithmetic is off by a share of those.  Non-finite values have to
    agree."""

    assert tuple(got.shape) == tuple(want.shape), f"{what}: {tuple(got.shape)} against {tuple(want.shape)}"
    g, w = got.detach().cpu().double(), want.detach().cpu().double()
    finite = torch.isfinite(w)
    assert torch.equal(finite, torch.isfinite(g)), f"{what}: non-finite values differ"
    g, w = g[finite], w[finite]
    if g.numel() == 0:
        return
    tiny = 2.0**-24 if got.dtype == torch.float16 else 0.0  # spacing of float16 below its normal range
    size = w.abs().max() if terms is None else torch.maximum(w.abs().max(), terms.abs().max())
    allowed = 1.25 * ROUND[got.dtype] * w.abs() + tol * size + tiny
    worst = float(((g - w).abs() - allowed).max())
    assert worst <= 0, f"{what}: over the bound by {worst:.3e}, peak {float(w.abs().max()):.3e}"


def gated_scan(x, ig, rg, decay, state=None, reset=None, lengths=None, reverse=False, rate=8.0):
    """h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(ig) x, step by step."""

    batch, steps, width = x.shape
    h = torch.zeros(batch, width, dtype=torch.float64) if state is None else state
    soft = torch.nn.functional.softplus(decay, threshold=1e4)
    ys = [None] * steps
    for t in range(steps - 1, -1, -1) if reverse else range(steps):
        la = -rate * soft * torch.sigmoid(rg[:, t])
        a, beta = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
        if reset is not None:
            cut = reset[:, t, None]
            a, beta = torch.where(cut, 0.0, a), torch.where(cut, 1.0, beta)
            new = a * torch.where(cut, 0.0, h)
        else:
            new = a * h
        new = new + beta * torch.sigmoid(ig[:, t]) * x[:, t]
        if lengths is not None:
            live = (t < lengths)[:, None]
            ys[t] = torch.where(live, new, 0.0)
            h = torch.where(live, new, h)
        else:
            ys[t] = h = new
    return (torch.stack(ys, dim=1) if steps else x.clone()), h


def norm_join(stream, block, post, pre, gate=None, scale=None, eps=1e-6, activation="sigmoid", fixed=False):
    """The two norms, the gate and the residual, operation by operation.
    ``fixed``: the norms' statistics count as constants, so that autograd gives
    the terms that a norm's gradient subtracts its mean from."""

    def rms(v):
        root = torch.sqrt((v * v).mean(dim=-1, keepdim=True) + eps)
        return v / (root.detach() if fixed else root)

    if block is not None:
        branch = rms(block) * post
        if gate is not None:
            branch = branch * (torch.nn.functional.silu(gate) if activation == "silu" else torch.sigmoid(gate))
        if scale is not None:
            branch = branch * scale
        stream = stream + branch
    return stream, rms(stream) * pre


def adamw(p, g, m, v, t, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, decay=1e-2):
    """New (p, m, v) of step t (the first is 1)."""

    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    p = p - lr * decay * p - lr * (m / (1 - betas[0] ** t)) / (torch.sqrt(v / (1 - betas[1] ** t)) + eps)
    return p, m, v
