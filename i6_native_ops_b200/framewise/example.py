"""Framewise training on an alignment, with every operator of the package in its place:

    python -m i6_native_ops_b200.framewise.example [--workload monophone] [--steps 20] [--dtype bf16] [--state-bits 8] [--muon]

A batch of automata and scores (``workloads``) is aligned (``align_viterbi``); a small network with the left label
context (``label_embedding``) learns the aligned class of every frame (``linear_cross_entropy``, ``AdamW``); its
output layer then scores the alignment, and one frame alone.  With ``--muon`` the hidden layer's matrix is updated by ``Muon``, the
rest by ``AdamW``, and a share of the distributions' entropy is added to the objective (``label_scores``).  Prints the loss
per frame along the way, and how sure the network is of the alignment in the end.
"""
from __future__ import annotations

import argparse
import math

import torch

from .. import workloads as wl
from ..fast_viterbi import align_viterbi
from . import AdamW, LabelScores, Muon, label_embedding, label_scores, linear_cross_entropy

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

    def scores(self, x, left, targets, seq_lens, top=0) -> LabelScores:
        """Log probabilities of the targets, entropies and the best classes, from logits in memory."""
        logits = torch.nn.functional.linear(self.hidden(x, left, seq_lens), self.out.weight, self.out.bias)
        return label_scores(logits, targets, top=top, seq_lens=seq_lens, ignore_index=IGNORE)

    def optimizers(self, muon: bool, state_bits: int):
        """``AdamW`` for all, or ``Muon`` for the hidden layer's matrix and ``AdamW`` for the rest."""
        matrices = [self.inner.weight] if muon else []
        rest = [p for p in self.parameters() if all(p is not m for m in matrices)]
        adamw = AdamW(rest, lr=2e-3, betas=(0.9, 0.98), state_bits=state_bits)
        return [adamw, Muon(matrices, lr=2e-3, adjust_lr="match_rms_adamw", weight_decay=0.01)] if muon else [adamw]


def left_labels(labels: torch.Tensor) -> torch.Tensor:
    """The label of the frame before; a sequence's first frame has none."""
    return torch.nn.functional.pad(labels[:, :-1], (1, 0), value=IGNORE)


def train(workload="monophone", steps=20, dtype=torch.bfloat16, state_bits=8, width=256, seqs=None, scale=1.0, muon=False, report=None):
    """Losses per frame before each step and after the last, and the loss of the first frame scored by itself.  ``report``: is
    given the model's scores of the alignment in the end (``LabelScores`` with three alternatives)."""
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
    optimizers = model.optimizers(muon, state_bits)
    losses = []
    for _ in range(steps):
        if muon:
            got = model.scores(x, left, targets, seq_lens)
            loss = -got.log_probs.sum() / count
            objective = loss - 0.01 * got.entropy.sum() / count
        else:
            objective = loss = model.loss(x, left, targets, seq_lens).sum() / count
        losses.append(loss.detach())
        objective.backward()
        for optimizer in optimizers:
            optimizer.step()
            optimizer.zero_grad()
    with torch.no_grad():
        if report is not None:
            report(model.scores(x, left, targets, seq_lens, top=min(3, batch.F)))
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
    ap.add_argument("--muon", action="store_true", help="Muon for the hidden layer, an entropy bonus in the objective")
    args = ap.parse_args()
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[args.dtype]
    sure = []
    losses, (within, alone) = train(args.workload, args.steps, dtype, args.state_bits, seqs=args.seqs, muon=args.muon, report=sure.append)
    for i, v in enumerate(losses):
        print(f"step {i:3d}  loss per frame {v:.4f}")
    print(f"first frame: {within:.4f} in its batch, {alone:.4f} by itself")
    got, inside = sure[0], sure[0].top_labels[..., 0] != IGNORE
    print(f"entropy per frame {float(got.entropy[inside].mean()):.4f}; the first frame's best classes: "
          + ", ".join(f"{c} ({p:.3f})" for c, p in zip(got.top_labels[0, 0].tolist(), got.top_log_probs[0, 0].exp().tolist())))


if __name__ == "__main__":
    main()
