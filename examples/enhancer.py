"""A causal speech enhancer trained on the PESQ loss, and run frame by frame.

    python examples/enhancer.py [--steps 200] [--state-bits 8] [--mixer attention] [--muon]

The network estimates a mask on the magnitude spectrum (512-sample frames, hop
256) with blocks of a gated linear recurrence, or of linear attention whose heads are normed.  It is trained with
``PesqLossCuda`` and ``AdamWCuda``, or ``MuonCuda`` for its matrices, on synthetic speech in noise; afterwards the same
weights run one frame at a time with the recurrences' states carried along, as
a live stream would, and give the same masks.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from triton_pesq_b200 import (AdamWCuda, GatedScanCuda, LayerNormCuda, LinearAttentionCuda, MuonCuda, NormJoinCuda,  # noqa: E402
                              PesqLossCuda, pre_norm)
from triton_pesq_b200.signals import add_noise, speech_like  # noqa: E402

N_FFT, HOP = 512, 256


class Block(torch.nn.Module):
    """Projection to the recurrence's input and gates, the recurrence, and the
    projection back; the join with the stream norms and gates its output."""

    def __init__(self, width: int):
        super().__init__()
        self.inner = torch.nn.Linear(width, 4 * width)
        self.scan = GatedScanCuda(width)
        self.outer = torch.nn.Linear(width, width)
        self.join = NormJoinCuda(width, activation="silu", scale=0.5)

    def forward(self, stream, normed, state=None):
        x, input_gate, decay_gate, gate = self.inner(normed).chunk(4, dim=2)
        y, state = self.scan(x, input_gate, decay_gate, state)
        stream, normed = self.join(stream, self.outer(y), gate)
        return stream, normed, state


class AttentionBlock(torch.nn.Module):
    """The same with linear attention: every head remembers for another time, and its output is normed by itself."""

    def __init__(self, width: int, heads: int = 4):
        super().__init__()
        self.heads, self.channels = heads, width // heads
        self.inner = torch.nn.Linear(width, 4 * width)
        self.attention = LinearAttentionCuda(heads, self.channels)
        self.norm = LayerNormCuda(self.channels, heads=heads)
        self.outer = torch.nn.Linear(width, width)
        self.join = NormJoinCuda(width, activation="silu", scale=0.5)

    def forward(self, stream, normed, state=None):
        *qkv, gate = self.inner(normed).chunk(4, dim=2)
        y, state = self.attention(*(t.unflatten(2, (self.heads, self.channels)) for t in qkv), state)
        stream, normed = self.join(stream, self.outer(self.norm(y).flatten(2)), gate)
        return stream, normed, state


class Enhancer(torch.nn.Module):
    def __init__(self, width: int = 96, blocks: int = 3, mixer: str = "scan"):
        super().__init__()
        bins = N_FFT // 2 + 1
        self.embed = torch.nn.Linear(bins, width)
        self.weight = torch.nn.Parameter(torch.ones(width))
        block = {"scan": Block, "attention": AttentionBlock}[mixer]
        self.blocks = torch.nn.ModuleList(block(width) for _ in range(blocks))
        self.head = torch.nn.Linear(width, bins)
        self.register_buffer("window", torch.hann_window(N_FFT))

    def masks(self, magnitude, states=None):
        """``[batch, frame, bin]`` magnitudes -> masks and the states after the last frame."""

        stream = self.embed(torch.log1p(magnitude))
        normed = pre_norm(stream, self.weight)
        after = []
        for i, block in enumerate(self.blocks):
            stream, normed, state = block(stream, normed, None if states is None else states[i])
            after.append(state)
        return torch.sigmoid(self.head(normed) + 2.0), after

    def spectrum(self, wave):
        return torch.stft(wave, N_FFT, HOP, window=self.window, return_complex=True).transpose(1, 2)

    def forward(self, wave):
        """Noisy waves ``[batch, sample]`` -> enhanced waves."""

        spec = self.spectrum(wave)
        mask, _ = self.masks(spec.abs())
        return torch.istft((spec * mask).transpose(1, 2), N_FFT, HOP, window=self.window, length=wave.shape[1])

    @torch.no_grad()
    def stream_masks(self, magnitude):
        """The masks of ``[batch, frame, bin]``, one frame after the other."""

        states, out = None, []
        for t in range(magnitude.shape[1]):
            mask, states = self.masks(magnitude[:, t:t + 1], states)
            out.append(mask)
        return torch.cat(out, dim=1)


def train(model, steps: int, batch: int = 8, seconds: float = 2.0, state_bits: int = 32, lr: float = 3e-3, seed: int = 0,
          muon: bool = False):
    """Trains on synthetic speech at 0 to 10 dB; returns the losses."""

    device = next(model.parameters()).device
    loss_fn = PesqLossCuda(0.5, sample_rate=16000).to(device)
    # (a norm's weights [head, channel] are a vector for each head, no matrix)
    matrices = [m.weight for m in model.blocks.modules() if isinstance(m, torch.nn.Linear) and muon]
    rest = [p for p in model.parameters() if not any(p is m for m in matrices)]
    optimisers = [AdamWCuda(rest, lr=lr, state_bits=state_bits, seed=seed)]
    if matrices:
        optimisers.append(MuonCuda(matrices, lr=lr, weight_decay=1e-2, adjust="match_rms_adamw"))
    samples, losses = int(16000 * seconds), []
    for step in range(steps):
        clean = speech_like(batch, samples, 16000, seed=seed + step % 16)
        noisy = add_noise(clean, float(step % 11), seed=1000 + seed + step % 16).to(device)
        clean = clean.to(device)
        model.zero_grad()
        enhanced = model(noisy)
        loss = loss_fn(clean, enhanced).mean()
        loss.backward()
        for optimiser in optimisers:
            optimiser.step()
        losses.append(loss.detach())
    return torch.stack(losses).cpu()


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    parser.add_argument("--mixer", default="scan", choices=("scan", "attention"))
    parser.add_argument("--muon", action="store_true", help="step the blocks' matrices by orthogonalised updates")
    args = parser.parse_args()
    torch.manual_seed(0)
    model = Enhancer(mixer=args.mixer).cuda()
    losses = train(model, args.steps, state_bits=args.state_bits, muon=args.muon)
    print(f"loss of the first ten steps {losses[:10].mean():.3f}, of the last ten {losses[-10:].mean():.3f}")
    noisy = add_noise(speech_like(1, 32000, 16000, seed=99), 5.0, seed=98).cuda()
    magnitude = model.spectrum(noisy).abs()
    with torch.no_grad():
        whole, _ = model.masks(magnitude)
    print(f"frame by frame: masks within {float((model.stream_masks(magnitude) - whole).abs().max()):.1e}")


if __name__ == "__main__":
    main()
