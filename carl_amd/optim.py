"""AdamW for the learner: one fused step over all of a policy's tensors.

    optimizer = carl_amd.optim.AdamW(policy.parameters(), lr=3e-4, bits=8)
    loss.backward()
    optimizer.step()

`AdamW` is a `torch.optim.Optimizer`; `adamw_step` is the step itself on lists
of tensors, and `decode_moments` / `encode_moments` convert between 8-bit
moments and float32.  Formulas, codes and orders of rounding are those of
include/carl_amd_ops.h.  Tensors must be on cuda:0; work is queued on torch's
current stream.
"""
from __future__ import annotations

from collections.abc import Sequence

import torch

import carl_amd  # noqa: F401  (the engine's library, and its error where it is not built)

from . import _ops

BLOCK = 256          # elements that share a scale


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avg: Sequence[torch.Tensor],
               exp_avg_sq: Sequence[torch.Tensor], *, step: int, lr: float, betas: tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 0.01, exp_avg_scale: Sequence[torch.Tensor] | None = None,
               exp_avg_sq_scale: Sequence[torch.Tensor] | None = None, grad_scale: torch.Tensor | None = None) -> None:
    """One AdamW step of every tensor in place, in one launch for 60 tensors.
    No two of them may overlap.

    params, grads   float32, bfloat16 or float16, contiguous, each of its own type
    exp_avg, exp_avg_sq   both float32; or int8 and uint8 codes with their
                    scales, one float32 for each 256 elements of a tensor
    step            the number of this update, 1 for the first; a captured call
                    keeps this and the other numbers in every replay
    grad_scale      a float32 tensor of one value on the GPU, multiplied onto
                    every gradient (a clipping factor that never reaches the host)
    """
    _ops.adamw_step(params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, step, lr, betas[0], betas[1], eps,
                    weight_decay, grad_scale)


def decode_moments(exp_avg: torch.Tensor, exp_avg_scale: torch.Tensor, exp_avg_sq: torch.Tensor,
                   exp_avg_sq_scale: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The float32 values of 8-bit moments."""
    return _ops.decode_moments(exp_avg, exp_avg_scale, exp_avg_sq, exp_avg_sq_scale)


def encode_moments(exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor) -> tuple[torch.Tensor, ...]:
    """(exp_avg, exp_avg_scale, exp_avg_sq, exp_avg_sq_scale) in 8 bits of float32 moments."""
    return _ops.encode_moments(exp_avg, exp_avg_sq)


class AdamW(torch.optim.Optimizer):
    """AdamW with the fused step; bits=8 keeps both moments in 8 bits.

    `step(grad_scale=...)` takes a clipping factor as `adamw_step` does.
    Parameters must be contiguous and their gradients dense; parameters without
    a gradient are passed over.  Steps are counted on the host, so `step` is
    refused while a graph is captured.
    """

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, *, bits: int = 32):
        if bits not in (8, 32):
            raise ValueError("bits must be 8 or 32")
        if not 0.0 <= lr:
            raise ValueError("lr must be non-negative")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("betas must be in [0, 1)")
        if not 0.0 <= eps:
            raise ValueError("eps must be non-negative")
        if not 0.0 <= weight_decay:
            raise ValueError("weight_decay must be non-negative")
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay, "bits": bits})

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        twice = len(set(group["params"])) != len(group["params"])     # one launch would step it by two threads at once
        if twice or group["bits"] not in (8, 32):
            self.param_groups.pop()
            raise ValueError("a parameter is in the group twice" if twice else "bits must be 8 or 32")

    def _moments(self, p: torch.Tensor, bits: int) -> dict:
        state = self.state[p]
        if not state:
            state["step"] = 0
            if bits == 8:
                blocks = -(-p.numel() // BLOCK)
                state["exp_avg"] = torch.zeros(p.shape, dtype=torch.int8, device=p.device)
                state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
                state["exp_avg_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
                state["exp_avg_sq_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
            else:
                state["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return state

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but the moments keep their own types (torch's would cast them to the parameters')."""
        saved = {i: dict(s) for i, s in state_dict["state"].items()}
        super().load_state_dict(state_dict)
        order = [i for g in state_dict["param_groups"] for i in g["params"]]
        for p, i in zip((p for g in self.param_groups for p in g["params"]), order):
            for name, value in saved.get(i, {}).items():
                if torch.is_tensor(value):
                    self.state[p][name] = value.detach().to(device=p.device, copy=True)

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: torch.Tensor | None = None):
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step counts its steps on the host: a graph would repeat one step's bias correction")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_step: dict[int, list] = {}
            for p in group["params"]:
                if p.grad is not None:
                    if p.grad.is_sparse:
                        raise ValueError("AdamW takes dense gradients")
                    state = self._moments(p, group["bits"])
                    by_step.setdefault(state["step"], []).append((p, p.grad.contiguous(), state))
            for last, rows in by_step.items():
                def column(name, rows=rows):
                    return [s[name] for _, _, s in rows]

                scales = {n: column(n) for n in ("exp_avg_scale", "exp_avg_sq_scale")} if group["bits"] == 8 else {}
                adamw_step([p for p, _, _ in rows], [g for _, g, _ in rows], column("exp_avg"), column("exp_avg_sq"),
                           step=last + 1, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"], grad_scale=grad_scale, **scales)
                for _, _, state in rows:
                    state["step"] = last + 1
        return loss


__all__ = ["AdamW", "adamw_step", "decode_moments", "encode_moments"]
