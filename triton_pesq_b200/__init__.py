"""B200-native PESQ loss engine.

``PesqLossCuda`` is a drop-in for the reference's ``PesqLossTriton``
(torch_pesq/triton_ops/loss.py) evaluated by hand-written sm_100a kernels
through the C ABI of ``libpesq_cuda.so`` (``include/pesq_cuda.h``);
``ResampleCuda`` is the reference's ``TritonResample`` (its polyphase sinc
resampler as a standalone op) and ``IIRCuda`` its ``TritonIIR`` (the causal
IIR filter as a standalone op) on the same library.

Beside them, the operators of the networks that are trained on the loss:
``gated_scan`` / ``GatedScanCuda`` (a gated linear recurrence),
``norm_join`` / ``pre_norm`` / ``NormJoinCuda`` (the norms before and after a
block with its gate and residual) and ``adamw_step`` / ``AdamWCuda`` (the
optimiser over all parameters at once).
"""

from .adamw import AdamWCuda, adamw_step
from .gated_scan import GatedScanCuda, gated_scan
from .iir import IIRCuda
from .loss import PesqLossCuda
from .norm_join import NormJoinCuda, norm_join, pre_norm
from .resample import ResampleCuda

__all__ = ["PesqLossCuda", "ResampleCuda", "IIRCuda", "GatedScanCuda", "gated_scan", "NormJoinCuda",
           "norm_join", "pre_norm", "AdamWCuda", "adamw_step"]
