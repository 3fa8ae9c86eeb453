"""A policy with memory for every car, trained on the vector environment's rollouts.

    python examples/recurrent_policy.py --n-sim 256 --updates 20

The policy acts one step at a time with `linear_attention_step` (the memories
of all agents stay on the GPU), and is trained on whole rollouts with
`linear_attention`: the rollout's buffers are [steps, agents, ...], the memory
it began with is its initial state, and an episode that ended restarts the
memory at the next step.  Around the two lie `rms_norm`, which adds to the
residual stream as it norms it, and `gated_ffn`; `top_actions` samples and
`action_log_prob` scores all action heads at once; `AdamW` takes all tensors in
one step, its clipping factor computed and applied on the GPU.  With
`--act-bits 8` the policy acts on 8-bit codes of its weights, made anew for each
rollout.  The loss is a plain policy gradient with a learned baseline: an
example of the operators together, not a training recipe.
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import carl  # noqa: E402
from carl.gymnasium import ACTION_NVECS, CARLActionCodec  # noqa: E402
from carl.gymnasium.torch import CARLTorchVectorEnv  # noqa: E402
from carl.ops import (action_log_prob, gated_ffn, int8_gated_linear, int8_linear, linear_attention, linear_attention_step,  # noqa: E402
                      quantize_int8, rms_norm, rms_norm_int8, top_actions)
from carl.optim import AdamW  # noqa: E402


EPS = torch.finfo(torch.float32).eps


class Block(nn.Module):
    """Linear attention and a gated feed-forward block, each on normalised input."""

    def __init__(self, width: int, heads: int, inner: int):
        super().__init__()
        self.heads = heads
        self.norms = nn.ParameterList(nn.Parameter(torch.ones(width)) for _ in range(2))
        self.qkv = nn.Linear(width, 3 * width, bias=False)
        self.out = nn.Linear(width, width, bias=False)
        self.gate, self.up = nn.Linear(width, inner, bias=False), nn.Linear(width, inner, bias=False)
        self.down = nn.Linear(inner, width, bias=False)
        # memories of 8 to 512 steps
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(-torch.linspace(3.0, 9.0, heads))))

    def quantized(self) -> dict:
        """Codes and scales of the weights, to act with."""
        return {name: quantize_int8(getattr(self, name).weight.detach()) for name in ("qkv", "out", "gate", "up", "down")}

    def _split(self, qkv: torch.Tensor) -> list[torch.Tensor]:
        return [t.unflatten(-1, (self.heads, -1)) for t in qkv.chunk(3, dim=-1)]

    def forward(self, x: torch.Tensor, stream: torch.Tensor, memory: torch.Tensor,
                starts: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """x is added to the stream first, and what comes back is yet to be added to the stream that comes with it:
        [agents, width] and the memory in place, or [steps, agents, width] and a new memory."""
        y, stream = rms_norm(x, self.norms[0], residual=stream, eps=EPS)
        q, k, v = self._split(self.qkv(y))
        if x.dim() == 2:
            mixed = linear_attention_step(q, k, v, self.log_decay, memory, starts=starts)
        else:
            mixed, memory = linear_attention(q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1), self.log_decay,
                                             starts=None if starts is None else starts.t(), initial_state=memory)
            mixed = mixed.transpose(0, 1)
        y, stream = rms_norm(self.out(mixed.flatten(-2)), self.norms[1], residual=stream, eps=EPS)
        return gated_ffn(y, self.gate.weight, self.up.weight, self.down.weight), stream, memory

    def act(self, x: torch.Tensor, stream: torch.Tensor, memory: torch.Tensor, starts: torch.Tensor | None,
            codes: dict) -> tuple[torch.Tensor, torch.Tensor]:
        """A step of `forward` with the weights' codes."""
        dtype = x.dtype
        y, scale, stream = rms_norm_int8(x, self.norms[0], residual=stream, eps=EPS)
        q, k, v = self._split(int8_linear(y, scale, *codes["qkv"], dtype=dtype))
        mixed = linear_attention_step(q, k, v, self.log_decay, memory, starts=starts)
        x = int8_linear(*quantize_int8(mixed.flatten(-2)), *codes["out"], dtype=dtype)
        y, scale, stream = rms_norm_int8(x, self.norms[1], residual=stream, eps=EPS)
        inner = int8_gated_linear(y, scale, *codes["gate"], *codes["up"], dtype=dtype)
        return int8_linear(*quantize_int8(inner), *codes["down"], dtype=dtype), stream


class RecurrentPolicy(nn.Module):
    """Action logits (one row of all heads, unavailable ones at -infinity) and a value for each agent and step."""

    def __init__(self, obs_dim: int, width: int = 128, heads: int = 4, inner: int = 344, layers: int = 2):
        super().__init__()
        self.width, self.heads = width, heads
        self.encode = nn.Linear(obs_dim, width)
        self.blocks = nn.ModuleList(Block(width, heads, inner) for _ in range(layers))
        self.act, self.value = nn.Linear(width, carl.ACTION_LOGITS), nn.Linear(width, 1)
        self.codec = CARLActionCodec()

    def memories(self, agents: int, device="cuda") -> list[torch.Tensor]:
        width = self.width // self.heads
        return [torch.zeros(agents, self.heads, width, width, device=device) for _ in self.blocks]

    def forward(self, obs: torch.Tensor, memories: list[torch.Tensor], starts: torch.Tensor | None = None):
        """obs [agents, obs_dim] (memories are updated in place) or [steps, agents, obs_dim] (new ones are returned)."""
        x = self.encode(obs)
        stream = torch.zeros_like(x)
        after = []
        for block, memory in zip(self.blocks, memories):
            x, stream, memory = block(x, stream, memory, starts)
            after.append(memory)
        return *self._heads(x + stream, obs), after

    def quantized(self) -> list[dict]:
        return [block.quantized() for block in self.blocks]

    def step(self, obs: torch.Tensor, memories: list[torch.Tensor], starts: torch.Tensor, codes: list[dict]):
        """Logits and values of one step of every agent, the blocks' products in 8 bits."""
        x = self.encode(obs)
        stream = torch.zeros_like(x)
        for block, memory, weights in zip(self.blocks, memories, codes):
            x, stream = block.act(x, stream, memory, starts, weights)
        return self._heads(x + stream, obs)

    def _heads(self, x: torch.Tensor, obs: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return self.act(x).masked_fill(~self.codec.mask(obs), -math.inf), self.value(x).squeeze(-1)


def sample(logits: torch.Tensor) -> torch.Tensor:
    noise = torch.empty(logits.shape, device=logits.device).exponential_().log_().neg_()
    return top_actions(logits, ACTION_NVECS, noise=noise)[0].squeeze(-1)


def log_prob(logits: torch.Tensor, actions: torch.Tensor) -> torch.Tensor:
    return action_log_prob(logits, actions, ACTION_NVECS)[0]


class Rollout:
    """Steps of every agent, [steps, agents, ...], and the memories they began with."""

    def __init__(self, policy: RecurrentPolicy, env: CARLTorchVectorEnv, steps: int, act_bits: int = 32):
        n = env.n_envs
        self.policy, self.env, self.steps, self.act_bits = policy, env, steps, act_bits
        self.memories = policy.memories(n)
        self.next_obs = env.reset().as_subclass(torch.Tensor).clone()
        self.next_start = torch.ones(n, dtype=torch.bool, device="cuda")

    @torch.no_grad()
    def collect(self) -> dict:
        first = [m.clone() for m in self.memories]
        rows = {name: [] for name in ("obs", "starts", "actions", "logits", "rewards")}
        codes = self.policy.quantized() if self.act_bits == 8 else None
        for _ in range(self.steps):
            if codes is None:
                logits, _, _ = self.policy(self.next_obs, self.memories, self.next_start)
            else:
                logits, _ = self.policy.step(self.next_obs, self.memories, self.next_start, codes)
            actions = sample(logits)
            rows["obs"].append(self.next_obs)
            rows["starts"].append(self.next_start)
            rows["actions"].append(actions)
            rows["logits"].append(logits)
            obs, reward, terminated, truncated, _ = self.env.step(actions)
            rows["rewards"].append(reward.float())
            self.next_obs = obs.as_subclass(torch.Tensor).clone()
            self.next_start = terminated | truncated
        batch = {name: torch.stack(x) for name, x in rows.items()}
        batch["ends"] = torch.cat((batch["starts"][1:], self.next_start[None]))
        # what the episodes that go on are worth after the last step
        _, batch["next_values"], _ = self.policy(self.next_obs, [m.clone() for m in self.memories], self.next_start)
        return batch | {"memories": first}


def returns(rewards: torch.Tensor, ends: torch.Tensor, last: torch.Tensor, discount: float) -> torch.Tensor:
    out = torch.empty_like(rewards)
    for t in reversed(range(len(rewards))):
        last = rewards[t] + discount * torch.where(ends[t], 0.0, last)
        out[t] = last
    return out


def update(policy: RecurrentPolicy, optimizer: AdamW, batch: dict, discount: float = 0.99, clip: float = 1.0) -> float:
    logits, values, _ = policy(batch["obs"], batch["memories"], batch["starts"])
    target = returns(batch["rewards"], batch["ends"], batch["next_values"], discount)
    advantage = target - values.detach()
    loss = -(log_prob(logits, batch["actions"]) * advantage).mean() + 0.5 * (values - target).square().mean()
    optimizer.zero_grad()
    loss.backward()
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(p.grad.float()) for p in policy.parameters()]))
    optimizer.step(grad_scale=(clip / norm.clamp(min=clip)).reshape(1))
    return loss.item()


def main() -> None:
    args = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    args.add_argument("--n-sim", type=int, default=256)
    args.add_argument("--steps", type=int, default=32)
    args.add_argument("--updates", type=int, default=20)
    args.add_argument("--bits", type=int, default=8, choices=(8, 32), help="of the optimizer's moments")
    args.add_argument("--act-bits", type=int, default=32, choices=(8, 32), help="of the weights while acting")
    a = args.parse_args()
    torch.manual_seed(0)
    env = CARLTorchVectorEnv(a.n_sim, 1, 1, normalize=True, discrete_actions=True)
    policy = RecurrentPolicy(env.single_observation_space.shape[0]).cuda()
    optimizer = AdamW(policy.parameters(), lr=3e-4, bits=a.bits)
    rollout = Rollout(policy, env, a.steps, a.act_bits)
    for i in range(a.updates):
        print(f"update {i}: loss {update(policy, optimizer, rollout.collect()):.5f}", flush=True)
    env.close()


if __name__ == "__main__":
    main()
