"""Operators of a policy with memory, as kernels for the MI355X.

  linear_attention       linear attention with a decay for each head over
                         rollouts and replays, with gradients
  linear_attention_step  its recurrent form: one step of every agent
  gated_ffn              a gated feed-forward block, with gradients

Formulas are those of include/carl_amd_ops.h.  Tensors must be on cuda:0; work
is queued on torch's current stream.  Unfitting arguments raise ValueError or
TypeError before anything is queued.
"""
from __future__ import annotations

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


__all__ = ["gated_ffn", "linear_attention", "linear_attention_step"]
