"""Framewise training on an alignment, with every operator of the package in its place:

    python -m i6_native_ops_b200.framewise.example [--workload monophone] [--steps 20] [--dtype bf16] [--state-bits 8]

A batch of automata and scores (``workloads``) is aligned (``align_viterbi``); a small network with the left label
context (``label_embedding``) learns the aligned class of every frame (``linear_cross_entropy``, ``AdamW``); its
output layer then scores the alignment, and one frame alone.  Prints the loss per frame along the way.
"""
from __future__ import annotations

import argparse
import math

import torch

from .. import workloads as wl
from ..fast_viterbi import align_viterbi
from . import AdamW, label_embedding, linear_cross_entropy

IGNORE = -100


class ContextModel(torch.nn.Module):
    """Features and the embedding of the frame's left label, one hidden layer; the output layer is the loss's."""

    def __init__(self, features: int, width: int, classes: int, dtype: torch.dtype, device):
        super().__init__()
        kw = {"dtype": dtype, "device": device}
        self.inner = torch.nn.Linear(features, width, **kw)
        self.context = torch.nn.Parameter(torch.randn(classes, width, **kw) / math.sqrt(width))
        self.out = torch.nn.Linear(width, classes, **kw)

    def hidden(self, x, left, seq_lens):
        context = label_embedding(left, self.context, scale=math.sqrt(self.context.shape[1]), seq_lens=seq_lens,
                                  ignore_index=IGNORE)
        return torch.tanh(self.inner(x) + context)

    def loss(self, x, left, targets, seq_lens):
        """(B, T) losses of the frames."""
        return linear_cross_entropy(self.hidden(x, left, seq_lens), self.out.weight, targets, bias=self.out.bias,
                                    seq_lens=seq_lens, ignore_index=IGNORE)


def left_labels(labels: torch.Tensor) -> torch.Tensor:
    """The label of the frame before; a sequence's first frame has none."""
    return torch.nn.functional.pad(labels[:, :-1], (1, 0), value=IGNORE)


def train(workload="monophone", steps=20, dtype=torch.bfloat16, state_bits=8, width=256, seqs=None, scale=1.0):
    """Losses per frame before each step and after the last, and the loss of the first frame scored by itself."""
    torch.manual_seed(0)
    device = torch.device("cuda:0")
    batch = wl.make_batch(workload, B=seqs, scale=scale)  # scale: shorter sequences
    scores = -wl.make_scores(batch, device)  # (T, B, F) log probabilities
    fsa, seq_lens = wl.to_torch(batch, device)
    log_probs = scores.transpose(0, 1).contiguous()
    targets, _ = align_viterbi(log_probs, fsa, seq_lens)
    # what the network sees: a random projection of the scores that the alignment went by
    x = (log_probs @ torch.randn(batch.F, width, device=device) / math.sqrt(batch.F)).to(dtype)
    left, count = left_labels(targets), seq_lens.sum()
    model = ContextModel(width, width, batch.F, dtype, device)
    optimizer = AdamW(model.parameters(), lr=2e-3, betas=(0.9, 0.98), state_bits=state_bits)
    losses = []
    for _ in range(steps):
        loss = model.loss(x, left, targets, seq_lens).sum() / count
        losses.append(loss.detach())
        loss.backward()
        optimizer.step()
        optimizer.zero_grad()
    with torch.no_grad():
        scored = model.loss(x, left, targets, seq_lens)
        losses.append(scored.sum() / count)
        one = slice(0, 1)
        alone = model.loss(x[one, one], left[one, one], targets[one, one].contiguous(), None)
    return [float(v) for v in losses], (float(scored[0, 0]), float(alone[0, 0]))


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--workload", default="monophone")
    ap.add_argument("--seqs", type=int, default=None)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--dtype", default="bf16", choices=["f32", "bf16"])
    ap.add_argument("--state-bits", type=int, default=8, choices=[8, 32])
    args = ap.parse_args()
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[args.dtype]
    losses, (within, alone) = train(args.workload, args.steps, dtype, args.state_bits, seqs=args.seqs)
    for i, v in enumerate(losses):
        print(f"step {i:3d}  loss per frame {v:.4f}")
    print(f"first frame: {within:.4f} in its batch, {alone:.4f} by itself")


if __name__ == "__main__":
    main()
