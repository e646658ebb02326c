"""Framewise training: the operators that follow an alignment or a label sequence.

``align_viterbi`` gives a class per frame, ``topology`` and ``fbw`` take label sequences; a network is trained on
them with an output layer over thousands of classes, an embedding of label contexts and an optimizer step:

  :func:`linear_cross_entropy`  output layer and softmax cross entropy in one, without logits in memory
  :func:`label_embedding`       scaled embedding of labels (and its gradient)
  :class:`AdamW`                AdamW over all parameters at once, states in 32 or 8 bits; :func:`adamw_step`,
                                :func:`adamw_values`, the step itself and what 8-bit states stand for

No counterpart in the reference, which ends at losses on log probabilities.  The native extension is required:
importing this module fails if it is not built (``python -m i6_native_ops_b200.build``); there is no CPU or
eager fallback.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
from typing import List, Optional, Sequence, Tuple, Union

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


class AdamW(torch.optim.Optimizer):
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


__all__ = ["core", "linear_cross_entropy", "label_embedding", "adamw_step", "adamw_values", "AdamW"]
