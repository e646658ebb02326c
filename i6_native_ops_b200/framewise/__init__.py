"""Framewise training: the operators that follow an alignment or a label sequence.

``align_viterbi`` gives a class per frame, ``topology`` and ``fbw`` take label sequences; a network is trained on
them with an output layer over thousands of classes, an embedding of label contexts and an optimizer step:

  :func:`linear_cross_entropy`  output layer and softmax cross entropy in one, without logits in memory
  :func:`label_embedding`       scaled embedding of labels (and its gradient)
  :func:`label_scores`          log probabilities of given labels, entropies and the best classes, off logits in memory
  :class:`AdamW`                AdamW over all parameters at once, states in 32 or 8 bits; :func:`adamw_step`,
                                :func:`adamw_values`, the step itself and what 8-bit states stand for
  :class:`Muon`                 Muon for hidden layers' matrices, all of them in a launch per product; :func:`muon_step`,
                                :func:`orthogonalize`, the step itself and its Newton-Schulz products

No counterpart in the reference, which ends at losses on log probabilities.  The native extension is required:
importing this module fails if it is not built (``python -m i6_native_ops_b200.build``); there is no CPU or
eager fallback.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
from typing import List, NamedTuple, Optional, Sequence, Tuple, Union

import torch

_PKG = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_LIB = os.path.join(_PKG, "libframewise_b200.so")
_EXT = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_build", "framewise_core.so")


def _load_core():
    if not (os.path.isfile(_LIB) and os.path.isfile(_EXT)):
        raise ImportError(
            "i6_native_ops_b200: native extension not built "
            f"(missing {_LIB if not os.path.isfile(_LIB) else _EXT}); "
            "run `python -m i6_native_ops_b200.build`"
        )
    # the extension links against libframewise_b200.so by soname; load it first so the loader finds it
    ctypes.CDLL(_LIB, mode=ctypes.RTLD_GLOBAL)
    spec = importlib.util.spec_from_file_location("framewise_core", _EXT)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


core = _load_core()


def _lengths(seq_lens: Optional[torch.Tensor], labels: torch.Tensor) -> Optional[torch.Tensor]:
    """``seq_lens`` as the ops want it, (B,) int32; also a (T, B) index mask, as ``fbw_loss`` takes it."""
    if seq_lens is not None and seq_lens.dim() == 2:
        if labels.dim() != 2 or tuple(seq_lens.shape) != (labels.shape[1], labels.shape[0]):
            raise RuntimeError(f"index mask must have shape (T, B), got {tuple(seq_lens.shape)}")
        return (seq_lens != 0).sum(0).to(torch.int32).contiguous()
    return seq_lens


def linear_cross_entropy(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    targets: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    seq_lens: Optional[torch.Tensor] = None,
    ignore_index: int = -100,
) -> torch.Tensor:
    """Negative log likelihood of a class per position under ``softmax(hidden @ weight.T + bias)``.

    :param hidden: (B, T, D) or (N, D) float32 or bfloat16 activations (CUDA); any strides, read in place where the
        last dimension is dense
    :param weight: (V, D) of the output layer, same dtype
    :param targets: (B, T) or (N,) int32 or int64 classes, such as the alignment of ``align_viterbi``
    :param bias: (V,), same dtype; a class with bias -inf has probability 0
    :param seq_lens: (B,) int32 lengths, or a (T, B) index mask
    :param ignore_index: targets of positions that are left out
    :return: float32 losses in the shape of ``targets``, 0 at positions past their length or left out.  Their
        gradients (unlike ``fbw_loss``) are scaled by the incoming gradient, per position; those of ``hidden`` are 0 at
        positions that do not count, whose values are never read.  A target outside 0..V-1 at a position that
        counts gives NaN.

    The (N, V) logits are never in memory: forward they stay on the SM, backward they are formed again and the
    gradients' left factor is held for some thousand rows at a time.  Sums are formed in 32 bits in a fixed order
    (logits by 1024 of the width at most, then added up); the products of float32 inputs keep 24 bits.  bfloat16: the
    left factor is held in 8 bits (16 for up to 256 positions), so gradients are some 1.4 times as far from exact ones as
    their own rounding alone, those of ``hidden`` twice where the rows of ``weight`` have most in common.

    Backward needs ``weight`` unchanged.  Derivatives are those of backward passes and of the first order; others are
    refused.  What backward needs (the rows that count, for float32 in three parts of 16 bits, and then the weight
    likewise) is saved as one tensor of bytes that saved-tensor hooks see."""
    return core.linear_cross_entropy(hidden, weight, targets, bias, _lengths(seq_lens, targets), int(ignore_index))


def label_embedding(
    labels: torch.Tensor,
    weight: torch.Tensor,
    scale: float = 1.0,
    seq_lens: Optional[torch.Tensor] = None,
    ignore_index: int = -100,
) -> torch.Tensor:
    """``scale * weight[labels]``, zeros at positions past their length or with the ignored label.

    :param labels: (B, T) or (N,) int32 or int64 (CUDA)
    :param weight: (V, D) float32 or bfloat16
    :param seq_lens: (B,) int32 lengths, or a (T, B) index mask
    :return: (*labels.shape, D) in the dtype of ``weight``.  The gradient of ``weight`` adds up the positions of a label
        in 32 bits, in a fixed order (equal calls give equal bits).  A label outside 0..V-1 at a position that counts
        gives NaN, in its row and in the whole gradient."""
    return core.label_embedding(labels, weight, float(scale), _lengths(seq_lens, labels), int(ignore_index))


class LabelScores(NamedTuple):
    """What :func:`label_scores` returns."""

    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: torch.Tensor
    top_labels: torch.Tensor


def label_scores(
    logits: torch.Tensor,
    labels: torch.Tensor,
    top: int = 0,
    seq_lens: Optional[torch.Tensor] = None,
    ignore_index: int = -100,
) -> LabelScores:
    """Log probabilities of given labels under ``softmax(logits)``, its entropy and its best classes, position by
    position.

    :param logits: (B, T, V) or (N, V) float32 or bfloat16 (CUDA), such as the ``log_probs`` that ``fbw_loss`` and
        ``align_viterbi`` take; any strides, read in place where the last dimension is dense.  A class of -inf has
        probability 0.
    :param labels: (B, T) or (N,) int32 or int64, such as an alignment
    :param top: how many of the best classes are returned, at most 32
    :param seq_lens: (B,) int32 lengths, or a (T, B) index mask
    :param ignore_index: labels of positions that are left out
    :return: ``log_probs`` and ``entropy``, float32 in the shape of ``labels``; ``top_log_probs`` and ``top_labels``, (..., top):
        the largest logits in falling order, equal ones by their class (NaN is the largest), so that fewer are the first of
        more; labels in the dtype of ``labels``.  Positions past their length or left out have 0 and the ignored label, and their logits are never read.

    A position whose logits are all -inf has log probabilities of -inf, entropy 0 and a gradient of 0; one with NaN or +inf
    has NaN.  A label outside 0..V-1 at a position that counts gives NaN, there and in that position's gradient.
    Everything is formed in 32 bits.  ``logits`` get gradients from the three float results, each position's in one pass,
    rounded once; they must not change before the backward pass.  Derivatives are of the first order, by backward passes."""
    return LabelScores(*core.label_scores(logits, labels, int(top), _lengths(seq_lens, labels), int(ignore_index)))


State = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def _split(states: Sequence[State]) -> Tuple[List[torch.Tensor], List[torch.Tensor]]:
    """Codes (or values) and steps of a list of states."""
    if any(isinstance(s, torch.Tensor) for s in states):
        return list(states), []
    return [s[0] for s in states], [s[1] for s in states]


def adamw_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    exp_avg: Sequence[State],
    exp_avg_sq: Sequence[State],
    step: int,
    master: Optional[Sequence[torch.Tensor]] = None,
    lr: float = 1e-3,
    betas: Tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 0.01,
    follow: bool = False,
) -> None:
    """One step of AdamW over a list of parameters, in place, in as few launches as there are 48 tensors.  As after any
    operation in place, graphs that saved a parameter before refuse their backward pass.

    :param params: contiguous CUDA tensors, all float32 or all bfloat16
    :param exp_avg, exp_avg_sq: per parameter a float32 tensor of its shape, or (8-bit states) ``(codes, steps)``: int8
        (first moment) or uint8 (root of the second) codes in the parameter's shape and a float32 step for each 256
        values in a row, which stand for ``code * |code| * step``.  They are rounded to the nearest codes where both
        betas are 0.98 at most, else up or down by offsets that change with ``step``, so that moments which shrink slower
        than codes are apart do so on average (roots of the second moment are then within about ``1 / sqrt(2 code)``)
    :param step: of this call, counted from 1; has to grow from step to step
    :param master: float32 copies that are updated in place of the parameters, which then get their rounded values
    :param follow: a copy of which its parameter is not the rounded value starts from the parameter, which has been changed
        since the last step; without, what the parameter holds makes no difference"""
    m, m_steps = _split(exp_avg)
    v, v_steps = _split(exp_avg_sq)
    core.adamw_step(list(params), list(grads), [] if master is None else list(master), m, v, m_steps, v_steps, float(lr),
                    float(betas[0]), float(betas[1]), float(eps), float(weight_decay), int(step), bool(follow))


def adamw_values(exp_avg: Sequence[State], exp_avg_sq: Sequence[State]) -> Tuple[List[torch.Tensor], List[torch.Tensor]]:
    """The float32 moments that 8-bit states stand for."""
    m, m_steps = _split(exp_avg)
    v, v_steps = _split(exp_avg_sq)
    return core.adamw_values(m, m_steps, v, v_steps)


class _Optimizer(torch.optim.Optimizer):
    """States keep their own types when they are loaded."""

    @staticmethod
    def _copy(p: torch.Tensor) -> torch.Tensor:
        return p.detach().to(torch.float32, memory_format=torch.contiguous_format)

    def load_state_dict(self, state_dict):
        """As torch's, but codes, moments and copies keep their own types (torch would turn them into the parameters').
        bfloat16 parameters whose states come from float32 ones start a copy of their own."""
        seen = {}  # what earlier hooks have made of the states; later ones see them with their types
        hooks = (self.register_load_state_dict_pre_hook(lambda _, given: seen.update(given)),
                 self.register_load_state_dict_post_hook(lambda _: self._take_states(seen), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _take_states(self, state_dict: dict) -> None:
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                state = {k: v.to(p.device, copy=True) if isinstance(v, torch.Tensor) else v
                         for k, v in state_dict["state"][i].items()}
                if state and p.dtype != torch.float32 and "master" not in state:
                    state["master"] = self._copy(p)
                self.state[p] = state


class AdamW(_Optimizer):
    """AdamW whose step takes all parameters of a group in one launch or a few.

    ``state_bits=8`` holds the moments in 8 bits (2 bytes a parameter instead of 8): per 256 values a step and quadratic
    codes, 16 thousand to one (first moment) and 65 thousand to one (root of the second) between largest and smallest
    (:func:`adamw_step` says how they are rounded: on average right at any betas, a root of the second moment that is a
    hundredth of its block's largest to some 15 %).
    bfloat16 parameters get a float32 copy that the steps accumulate in (``state["master"]``); values that the program
    changes between steps (a model loaded, weights clipped) are taken over from the parameter.  Parameters without a
    gradient are passed over.  The learning rate may be changed between steps, as for any torch optimizer."""

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def _fresh(self, p: torch.Tensor, bits: int) -> dict:
        state = {"step": 0}
        if bits == 8:
            steps = -(-p.numel() // core.state_block)
            for name, kind in (("exp_avg", torch.int8), ("exp_avg_sq", torch.uint8)):
                state[name] = torch.zeros(p.shape, dtype=kind, device=p.device)
                state[name + "_steps"] = torch.zeros(steps, dtype=torch.float32, device=p.device)
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if p.dtype != torch.float32:
            state["master"] = self._copy(p)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            calls = {}  # parameters of one device, dtype and step count go together
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state.update(self._fresh(p, group["state_bits"]))
                calls.setdefault((p.device, p.dtype, state["step"] + 1), []).append(p)
            for (_, dtype, step), params in calls.items():
                states = [self.state[p] for p in params]
                pick = lambda name: [s[name] for s in states]  # noqa: E731
                eight = group["state_bits"] == 8
                core.adamw_step(params, [p.grad for p in params], [] if dtype == torch.float32 else pick("master"),
                                pick("exp_avg"), pick("exp_avg_sq"), pick("exp_avg_steps") if eight else [],
                                pick("exp_avg_sq_steps") if eight else [], float(group["lr"]), float(group["betas"][0]),
                                float(group["betas"][1]), float(group["eps"]), float(group["weight_decay"]), int(step), True)
                for s in states:  # a call that was refused has not taken place
                    s["step"] = step
        return loss


Triple = Tuple[float, float, float]
COEFFICIENTS: Triple = (3.4445, -4.7750, 2.0315)


def _flat(coefficients: Union[Triple, Sequence[Triple]], steps: int) -> List[float]:
    """Three numbers per step, from those of one step or of all."""
    try:
        given = list(coefficients)
        rows = [tuple(c) for c in given] if given and isinstance(given[0], (tuple, list)) else [tuple(float(c) for c in given)] * int(steps)
    except TypeError:
        rows = []
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise RuntimeError("steps must be in 1..100, and coefficients three numbers, or three for each of the steps")
    return [float(c) for r in rows for c in r]


def _match_rms(adjust_lr: Optional[str]) -> bool:
    if adjust_lr not in (None, "original", "match_rms_adamw"):
        raise ValueError('adjust_lr must be "original" or "match_rms_adamw"')
    return adjust_lr == "match_rms_adamw"


def orthogonalize(
    x: torch.Tensor,
    steps: int = 5,
    coefficients: Union[Triple, Sequence[Triple]] = COEFFICIENTS,
    eps: float = 1e-7,
) -> torch.Tensor:
    """Matrices with singular values near one and the singular vectors of ``x``, by Newton-Schulz products: ``X = x /
    max(|x|, eps)`` (Frobenius norm), then ``steps`` times ``A = X X^T; X = a X + (b A + c A A) X``, matrices with more
    rows than columns the other way round.

    :param x: (..., rows, cols) float32 or bfloat16 (CUDA)
    :param coefficients: (a, b, c) of every step, or one such triple per step.  Those that let singular values grow past
        10^6 are refused
    :return: the same shape and dtype; there is no gradient.  X is held in 32 bits; the operands of the products have 11
        bits for bfloat16 matrices (A 22 where the shorter side is at most 128) and 22 for float32 ones, sums are formed in
        32 bits in a fixed order.  A matrix with NaN or an infinity becomes NaN, one of zeros stays as it is."""
    return core.orthogonalize(x, _flat(coefficients, steps), float(eps))


def muon_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    momentum: Sequence[torch.Tensor],
    lr: float = 1e-3,
    beta: float = 0.95,
    nesterov: bool = True,
    weight_decay: float = 0.1,
    steps: int = 5,
    coefficients: Union[Triple, Sequence[Triple]] = COEFFICIENTS,
    eps: float = 1e-7,
    adjust_lr: Optional[str] = None,
    master: Optional[Sequence[torch.Tensor]] = None,
    follow: bool = False,
) -> None:
    """One step of Muon over a list of matrices, in place: ``v += (1 - beta) (g - v)``, ``u = g + beta (v - g)`` (without
    ``nesterov``: ``v``), ``p = p (1 - lr weight_decay) - lr s orthogonalize(u)``.  Matrices of up to 128 x 256 take a
    launch for every 24 of them, the others, of whatever shapes, go through each product in one launch (256 of them, as far as
    two gigabytes of scratch hold them).  Copies too get what :func:`orthogonalize` makes of the parameters' type: for
    bfloat16 parameters the update is off by some 0.6e-3 to 1e-3 of its norm (up to 2e-3 where a matrix has a few rows), whether
    or not there is a copy in 32 bits.  As after any operation in place, graphs that saved a parameter before refuse their backward pass.

    :param params: contiguous CUDA matrices, all float32 or all bfloat16.  Parameters, momentum and copies overlap neither each
        other nor a gradient; gradients may be shared
    :param momentum: per parameter a float32 tensor of its shape
    :param adjust_lr: ``"original"`` (or None): ``s = sqrt(max(1, rows / cols))``; ``"match_rms_adamw"``: ``s = 0.2
        sqrt(max(rows, cols))``
    :param master: float32 copies of bfloat16 parameters, updated in place of them; they then get their rounded values
    :param follow: a copy of which its parameter is not the rounded value starts from the parameter, as for
        :func:`adamw_step`"""
    core.muon_step(list(params), list(grads), list(momentum), [] if master is None else list(master), float(lr), float(beta), bool(nesterov),
                   float(weight_decay), _match_rms(adjust_lr), _flat(coefficients, steps), float(eps), bool(follow))


class Muon(_Optimizer):
    """Muon for the matrices of a model's hidden layers: momentum, made orthogonal, as the update.  (Embeddings, output
    layers and vectors are for :class:`AdamW`.)

    Parameters have to be matrices.  bfloat16 parameters get a float32 copy that the steps accumulate in
    (``state["master"]``); values that the program changes between steps are taken over from the parameter.  Parameters
    without a gradient are passed over.  The arguments are those of :func:`muon_step`."""

    def __init__(self, params, lr: float = 1e-3, beta: float = 0.95, nesterov: bool = True, weight_decay: float = 0.1, steps: int = 5,
                 coefficients: Union[Triple, Sequence[Triple]] = COEFFICIENTS, eps: float = 1e-7, adjust_lr: Optional[str] = None):
        _flat(coefficients, steps)
        _match_rms(adjust_lr)
        super().__init__(params, dict(lr=lr, beta=beta, nesterov=nesterov, weight_decay=weight_decay, steps=steps, coefficients=coefficients,
                                      eps=eps, adjust_lr=adjust_lr))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2:
                self.param_groups.pop()
                raise ValueError(f"Muon takes matrices, got a parameter of shape {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            calls = {}  # parameters of one device and dtype go together
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state["momentum"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                    if p.dtype != torch.float32:
                        state["master"] = self._copy(p)
                calls.setdefault((p.device, p.dtype), []).append(p)
            for (_, dtype), params in calls.items():
                states = [self.state[p] for p in params]
                muon_step(params, [p.grad for p in params], [s["momentum"] for s in states], lr=group["lr"], beta=group["beta"],
                          nesterov=group["nesterov"], weight_decay=group["weight_decay"], steps=group["steps"],
                          coefficients=group["coefficients"], eps=group["eps"], adjust_lr=group["adjust_lr"],
                          master=None if dtype == torch.float32 else [s["master"] for s in states], follow=True)
        return loss


__all__ = ["core", "linear_cross_entropy", "label_embedding", "LabelScores", "label_scores", "adamw_step", "adamw_values", "AdamW",
           "orthogonalize", "muon_step", "Muon"]
