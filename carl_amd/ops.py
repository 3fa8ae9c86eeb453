"""Operators of a policy with memory, as kernels for the MI355X.

  linear_attention       linear attention with a decay for each head over
                         rollouts and replays, with gradients
  linear_attention_step  its recurrent form: one step of every agent
  gated_ffn              a gated feed-forward block, with gradients
  rms_norm               root-mean-square norm with the addition before it,
                         with gradients
  action_log_prob        log-probability and entropy of actions over several
                         heads, with gradients
  top_actions            the best actions of each head, or a sample

and, for acting with weights in 8 bits:

  quantize_int8          rows as 8-bit codes with a scale for each
  rms_norm_int8          rms_norm with such an output
  int8_linear            a projection of codes by codes
  int8_gated_linear      the gate and up projections of a gated block

Formulas are those of include/carl_amd_ops.h.  Tensors must be on cuda:0; work
is queued on torch's current stream.  Unfitting arguments raise ValueError or
TypeError before anything is queued.
"""
from __future__ import annotations

from collections.abc import Sequence

import torch

import carl_amd  # noqa: F401  (the engine's library, and its error where it is not built)

from . import _ops


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                     starts: torch.Tensor | None = None, initial_state: torch.Tensor | None = None,
                     scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Outputs of every step and the memory after the last one.

        S_t = [starts_t ? 0 : exp(log_decay) S_{t-1}] + k_t v_t^T
        out_t = scale S_t^T q_t

    q               [batch, steps, heads, key width], float32, bfloat16 or float16
    k, v            [batch, steps, key heads, key or value width]; query head h
                    reads key head h // (heads / key heads)
    log_decay       float32 [heads], at most 0; it has no gradient, and may ask
                    for one only where gradients are off
    starts          bool [batch, steps]: steps that begin an episode and see
                    nothing before them (the `done` of the step before)
    initial_state   float32 [batch, heads, key width, value width], contiguous;
                    zero without
    scale           key width ** -0.5 without

    Widths are at most 128, batch times heads 4,194,304.  Batch, step and head
    strides are free (a rollout kept as [steps, batch, ...] is passed
    transposed, and its outputs and gradients come in the same order); the last
    dimension is contiguous.  Gradients reach q, k, v and initial_state, once.
    """
    return _ops.linear_attention(q, k, v, log_decay, starts, initial_state, scale)


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: torch.Tensor, *, starts: torch.Tensor | None = None,
                          scale: float | None = None) -> torch.Tensor:
    """One step of `linear_attention` for every agent: q, k and v without the
    steps' dimension, starts [batch], and the contiguous memory `state` updated
    in place.  For acting; it has no gradient."""
    return _ops.linear_attention_step(q, k, v, log_decay, state, starts, scale)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *,
              activation: str = "silu") -> torch.Tensor:
    """(act(x w_gate^T) * (x w_up^T)) w_down^T

    x               [..., width], float32, bfloat16 or float16
    w_gate, w_up    [inner, width], as torch.nn.Linear keeps them
    w_down          [width, inner]
    activation      "silu", or "gelu" in its tanh form

    All of one type; products are summed in float32.  Widths are at most
    65,536, rows 2^28, and rows times the larger width about 2^36.  Gradients
    reach x and the weights, once; the backward pass computes both projections
    again instead of keeping them.
    """
    return _ops.gated_ffn(x, w_gate, w_up, w_down, activation)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None,
             eps: float = 1e-6) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """s / sqrt(mean(s^2) + eps) * weight with s = x + residual; with a
    residual (result, s).

    x, residual     [..., width], float32, bfloat16 or float16
    weight          [width]
    eps             at least 1e-30

    All of one type; s is rounded to it once and the norm is that of the
    rounded s.  Widths are at most 16,384.  Gradients reach x, residual and
    weight, once, from both results.
    """
    return _ops.rms_norm(x, weight, residual, eps)


def action_log_prob(logits: torch.Tensor, actions: torch.Tensor, heads: Sequence[int], *,
                    mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(log-probability, entropy) of the actions of all heads, float32 [...].

    logits          [..., sum of heads], float32, bfloat16 or float16: the
                    heads' logits next to each other
    actions         [..., len(heads)], int32 or int64
    heads           the heads' sizes (carl.ACTION_NVECS): 1 to 64 of them,
                    16,384 logits in all at most
    mask            bool, of the logits' shape: True where an action can be taken

    A masked logit, or one of -infinity, weighs nothing whatever it holds and
    gets the gradient 0; its action's log-probability is -infinity.  A head
    with nothing to take has entropy 0.  An action below 0 is none: its head
    adds nothing to the log-probability; an action past its head's last makes
    it NaN, and its head's gradients by it.  Gradients of both results reach
    logits, once.
    """
    return _ops.action_log_prob(logits, actions, list(heads), mask)


def top_actions(logits: torch.Tensor, heads: Sequence[int], k: int = 1, *, mask: torch.Tensor | None = None,
                noise: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The k best actions of each head, int32 [..., len(heads), k], and their
    log-probabilities, float32.

    noise           float32, of the logits' shape, added to them before they
                    are compared (not to the log-probabilities): with
                    -log(-log(u)), u uniform in (0, 1), the best action is a
                    sample of the policy

    Logits, heads and mask are those of `action_log_prob`.  Equal ones go by
    their index.  Where fewer than k can be taken the rest are -1, with the
    log-probability -infinity; k is at most 64.  For acting; it has no gradient.
    """
    return _ops.top_actions(logits, list(heads), k, mask, noise)


def quantize_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (int8 [..., width]) and scales (float32 [...]) of rows: a code c of
    a row stands for c times the row's scale, its largest magnitude / 127.

    Codes lie in rows that begin every 16 bytes, as `int8_linear` reads them
    best.  Widths are at most 16,384.  A row with a NaN or an infinity has the
    scale NaN.  For weights, and for rows that no norm has made; it has no
    gradient.
    """
    return _ops.quantize_int8(x)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None,
                  eps: float = 1e-6) -> tuple[torch.Tensor, ...]:
    """`rms_norm` with its result as codes and scales, as `quantize_int8` gives
    them: (codes, scales), and with a residual (codes, scales, s)."""
    return _ops.rms_norm_int8(x, weight, residual, eps)


def int8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """(x weight^T) x_scale weight_scale + bias

    x               int8 [..., width], x_scale float32 [...]
    weight          int8 [columns, width], weight_scale float32 [columns]
    bias            [columns], of the result's type
    dtype           of the result: float32, bfloat16 or float16

    The sum of products is exact; it is scaled in float32 and rounded once.
    Widths and columns are at most 65,536.  It has no gradient.
    """
    return _ops.int8_linear(x, x_scale, weight, weight_scale, bias, dtype)


def int8_gated_linear(x: torch.Tensor, x_scale: torch.Tensor, w_gate: torch.Tensor, gate_scale: torch.Tensor, w_up: torch.Tensor,
                      up_scale: torch.Tensor, *, activation: str = "silu", dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """act(gate) * up of two products as `int8_linear` makes them: the inner
    values of `gated_ffn`, in one pass over x."""
    return _ops.int8_gated_linear(x, x_scale, w_gate, gate_scale, w_up, up_scale, activation, dtype)


__all__ = ["action_log_prob", "gated_ffn", "int8_gated_linear", "int8_linear", "linear_attention", "linear_attention_step",
           "quantize_int8", "rms_norm", "rms_norm_int8", "top_actions"]
