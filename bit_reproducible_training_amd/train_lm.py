"""Trains a small language model with every operation of a step from this package, and prints the losses
and a hash of the trained parameters: the same on every run, on a GPU and on the CPU.

    python -m bit_reproducible_training_amd.train_lm --steps 20
    python -m bit_reproducible_training_amd.train_lm --steps 20 --device cpu --state-bits 8

The model predicts the next symbol from the last `context` ones (a feed-forward language model): a Linear
over their one-hot vectors, blocks of Linear, ReLU, Linear whose outputs go through ResidualNorm into the
residual stream (gated, normalised before and after with --sandwich), and LinearCrossEntropy as the
head; AdamW takes the steps. The text is made up: symbols that mostly follow from the one before.
"""
import argparse

import torch

from . import AdamW, Linear, LinearCrossEntropy, Norm, ResidualNorm, guard, name_layers
from ._lib import _backend

__all__ = ["Model", "parameter_hash", "text", "train"]


def text(length, vocab, seed=1):
    """A list of symbols below vocab: mostly a fixed function of the one before, else arbitrary."""
    out, state = [0], seed
    while len(out) < length:
        state = (state * 6364136223846793005 + 1442695040888963407) % 2 ** 64
        draw = state >> 33
        out.append((5 * out[-1] + 1) % vocab if draw % 8 else draw // 8 % vocab)
    return out[:length]


class Block(torch.nn.Module):
    def __init__(self, width, hidden, kind, sandwich):
        super().__init__()
        self.up, self.down = Linear(width, hidden), Linear(hidden, width)
        self.norm = ResidualNorm(width, kind=kind, post_norm=sandwich, scale=0.5 if sandwich else 1.0)
        self.gate = torch.nn.Parameter(torch.ones(width)) if sandwich else None

    def forward(self, r, y):
        return self.norm(r, self.down(torch.relu(self.up(y))), self.gate)


class Model(torch.nn.Module):
    def __init__(self, vocab, context, width, blocks, kind="layer", sandwich=False):
        super().__init__()
        self.vocab = vocab
        self.embed = Linear(vocab * context, width)
        self.first = Norm(width, kind=kind)
        self.blocks = torch.nn.ModuleList(Block(width, 4 * width, kind, sandwich) for _ in range(blocks))
        self.head = LinearCrossEntropy(width, vocab)

    def forward(self, context, target):
        """The mean loss of target [n] after context [n, symbols]."""
        hot = torch.nn.functional.one_hot(context, self.vocab).to(torch.float32).flatten(1)
        r = self.embed(hot)
        y = self.first(r)
        for block in self.blocks:
            r, y = block(r, y)
        return self.head(y, target)


def parameter_hash(model):
    h = 0xcbf29ce484222325
    for p in model.parameters():
        h = _backend.fnv1a64(p.detach().cpu().contiguous(), h)
    return h


def train(device, steps, vocab=64, context=4, width=64, blocks=2, batch=512, state_bits=32, kind="layer",
          sandwich=False, report=None):
    """(losses, hash of the trained parameters)"""
    torch.manual_seed(0)
    model = name_layers(Model(vocab, context, width, blocks, kind, sandwich)).to(device)
    decayed = [p for p in model.parameters() if p.dim() > 1]
    others = [p for p in model.parameters() if p.dim() < 2]
    optimizer = AdamW([{"params": decayed}, {"params": others, "weight_decay": 0.0}], lr=3e-3, betas=(0.9, 0.95),
                      weight_decay=0.1, state_bits=state_bits)
    symbols = torch.tensor(text(batch * steps + context + 1, vocab))
    windows = symbols.unfold(0, context + 1, 1)
    losses = []
    for step in range(steps):
        rows = windows[step * batch:(step + 1) * batch].to(device)
        loss = model(rows[:, :-1], rows[:, -1].contiguous())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if report is not None:
            report(step, losses[-1])
    guard().check()
    return [x.item() for x in losses], parameter_hash(model)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--vocab", type=int, default=64)
    ap.add_argument("--context", type=int, default=4)
    ap.add_argument("--width", type=int, default=64)
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--batch", type=int, default=512)
    ap.add_argument("--state-bits", type=int, choices=(8, 32), default=32)
    ap.add_argument("--kind", choices=("layer", "rms"), default="layer")
    ap.add_argument("--sandwich", action="store_true", help="norms before and after each block, and a gate")
    a = ap.parse_args(argv)
    losses, h = train(a.device, a.steps, a.vocab, a.context, a.width, a.blocks, a.batch, a.state_bits, a.kind, a.sandwich)
    for step, loss in enumerate(losses):
        print("step %3d  loss %.6f" % (step, loss))
    print("parameters %016x" % h)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
