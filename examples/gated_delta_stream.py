"""Train a gated-delta sequence classifier on waveforms, then run it on streams.

    python examples/gated_delta_stream.py [--steps 30] [--time 640] [--width 64]

The pieces as a program uses them together: gated_delta_scan over padded
batches of unlike lengths in training (its gradients through autograd),
clip_grads_ between the backward and the optimiser, gated_delta_scan over a
stream's first part and gated_delta_step from there on, on states in a pool of
slots.  The stream's logits are compared with those of the whole sequence.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import prospective_rqf_b200 as rqf  # noqa: E402
from prospective_rqf_b200.train import waveform_batch  # noqa: E402


class GatedDeltaLayer(nn.Module):
    """x + W_o o(x), with o from the gated delta rule on projections of x."""

    def __init__(self, width: int, heads: int = 2, key_dim: int = 32):
        super().__init__()
        self.heads, self.key_dim, self.value_dim = heads, key_dim, width // heads
        self.sizes = [heads * key_dim, heads * key_dim, heads * self.value_dim]
        self.norm = nn.RMSNorm(width)
        self.qkv = nn.Linear(width, sum(self.sizes), bias=False)
        self.gates = nn.Linear(width, 2 * heads)
        nn.init.constant_(self.gates.bias[:heads], -4.0)  # slow decay at first
        self.out = nn.Linear(heads * self.value_dim, width, bias=False)

    def _inputs(self, x):
        x = self.norm(x)
        # parts of one projection: the operators take these views as they are
        q, k, v = (t.unflatten(-1, (self.heads, -1)) for t in self.qkv(x).split(self.sizes, -1))
        decay, beta = self.gates(x).chunk(2, -1)
        unit = lambda t: nn.functional.normalize(t.float(), dim=-1).to(v.dtype)  # noqa: E731
        return unit(q), unit(k), v, -nn.functional.softplus(decay), torch.sigmoid(beta)

    def forward(self, x, lengths=None):
        """x (batch, time, width); returns the same and the states after each row's end."""
        o, state = rqf.gated_delta_scan(*self._inputs(x), lengths=lengths, return_state=True)
        return x + self.out(o.flatten(-2)), state

    def step(self, x, pool, slots):
        """One token of each row, x (batch, width), on the states pool[slots]."""
        o = rqf.gated_delta_step(*self._inputs(x), pool, slots=slots)
        return x + self.out(o.flatten(-2))


class Classifier(nn.Module):
    """Waveform to class logits at every step."""

    def __init__(self, width: int, classes: int, layers: int = 2, frame: int = 16):
        super().__init__()
        self.frame = frame
        self.embed = nn.Linear(frame, width)
        self.layers = nn.ModuleList(GatedDeltaLayer(width) for _ in range(layers))
        self.head = nn.Linear(width, classes)

    def forward(self, frames, lengths=None):
        x, states = self.embed(frames), []
        for layer in self.layers:
            x, state = layer(x, lengths)
            states.append(state)
        return self.head(x), states

    def step(self, frame, pools, slots):
        x = self.embed(frame)
        for layer, pool in zip(self.layers, pools):
            x = layer.step(x, pool, slots)
        return self.head(x)


def train(model, steps: int, time: int, classes: int, batch: int = 16, seed: int = 0):
    """A few optimisation steps; returns the losses and the gradients' norms."""
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    g = torch.Generator().manual_seed(seed)
    x, y = waveform_batch(batch, time, 16000.0, classes, g, "cuda")
    frames = x.view(batch, -1, model.frame)
    lengths = torch.randint(frames.shape[1] // 2, frames.shape[1] + 1, (batch,), generator=g).cuda()
    last = (lengths - 1)[:, None, None].expand(-1, 1, classes)
    losses, norms = [], []
    for _ in range(steps):
        logits, _ = model(frames, lengths)
        loss = nn.functional.cross_entropy(logits.gather(1, last)[:, 0], y)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        norms.append(rqf.clip_grads_([p.grad for p in model.parameters()], 1.0))
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses), torch.stack(norms)


@torch.no_grad()
def stream(model, frames, prompt: int, slots):
    """Logits of streams whose first `prompt` frames come at once and the others one by one, on
    the states `slots` of a pool that is larger than the batch."""
    logits, states = model(frames[:, :prompt])
    pools = [s.new_zeros(int(slots.max()) + 3, *s.shape[1:]).index_copy_(0, slots.long(), s) for s in states]
    out = [logits]
    for t in range(prompt, frames.shape[1]):
        out.append(model.step(frames[:, t], pools, slots)[:, None])
    return torch.cat(out, 1)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--time", type=int, default=640 * 16, help="samples of a waveform, whole frames of 16")
    ap.add_argument("--width", type=int, default=64)
    args = ap.parse_args(argv)
    torch.manual_seed(0)
    classes = 8
    model = Classifier(args.width, classes).cuda()
    losses, norms = train(model, args.steps, args.time, classes)
    print(f"loss {float(losses[0]):.4f} -> {float(losses[-1]):.4f}, gradient norm {float(norms[0]):.3f} -> "
          f"{float(norms[-1]):.3f}")
    frames = waveform_batch(4, args.time, 16000.0, classes, torch.Generator().manual_seed(1), "cuda")[0]
    frames = frames.view(4, -1, model.frame)
    slots = torch.tensor([5, 0, 3, 1], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        whole, _ = model(frames)
    apart = stream(model, frames, frames.shape[1] - 20, slots)
    difference = float((apart - whole).abs().max() / whole.abs().max())
    rqf.check_device_errors()
    print(f"streamed logits differ from the whole sequence's by {difference:.1e} of their largest")
    return losses, norms, difference


if __name__ == "__main__":
    main()
