"""The operators around a policy's layers as the example policy uses them: a
rollout acted in 8 bits, and the gradients of its loss against torch's own
operations; and while another device than their tensors' is the current one."""
from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "recurrent_policy.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("recurrent_policy", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _setting(example, steps, **rollout):
    torch.manual_seed(0)
    env = example.CARLTorchVectorEnv(12, 1, 1, normalize=True, discrete_actions=True)
    policy = example.RecurrentPolicy(env.single_observation_space.shape[0]).cuda()
    return env, policy, example.Rollout(policy, env, steps, **rollout)


def test_acting_in_8_bits_runs(example):
    """Actions that can be taken, and an update on the rollout that they made."""
    env, policy, rollout = _setting(example, 16, act_bits=8)
    optimizer = example.AdamW(policy.parameters(), lr=3e-4)
    for _ in range(2):
        batch = rollout.collect()
        log_prob, entropy = example.action_log_prob(batch["logits"], batch["actions"], example.ACTION_NVECS)
        assert bool(torch.isfinite(log_prob).all()) and bool((entropy > 0).all())
        assert bool((batch["actions"] >= 0).all())
        assert math.isfinite(example.update(policy, optimizer, batch))
    assert all(bool(torch.isfinite(p).all()) for p in policy.parameters())
    env.close()


def test_the_policys_gradients_are_those_of_torchs_operations(example):
    """The loss of a rollout through the operators, and through torch's norm, additions, softmax and indexing."""
    env, policy, rollout = _setting(example, 12)
    batch = rollout.collect()

    def gradients(rms_norm, action_log_prob):
        kept = example.rms_norm, example.action_log_prob
        example.rms_norm, example.action_log_prob = rms_norm, action_log_prob
        try:
            logits, values, _ = policy(batch["obs"], batch["memories"], batch["starts"])
            loss = -example.log_prob(logits, batch["actions"]).mean() + 0.5 * (values - batch["rewards"]).square().mean()
            return loss.detach(), torch.autograd.grad(loss, list(policy.parameters()))
        finally:
            example.rms_norm, example.action_log_prob = kept

    def plain_norm(x, weight, *, residual, eps):
        s = x + residual
        return torch.nn.functional.rms_norm(s, s.shape[-1:], weight, eps), s

    def plain_log_prob(logits, actions, heads):
        picked = [h.log_softmax(-1).gather(-1, actions[..., i:i + 1].long()) for i, h in enumerate(logits.split(heads, -1))]
        return torch.cat(picked, -1).sum(-1), None

    loss, ours = gradients(example.rms_norm, example.action_log_prob)
    want, theirs = gradients(plain_norm, plain_log_prob)
    assert loss.item() == pytest.approx(want.item(), rel=1e-5)
    for a, b in zip(ours, theirs):
        # float32 sums over 288 steps of agents in another order, through two layers
        assert torch.allclose(a, b, rtol=0, atol=2e-5 * float(b.abs().max()) + 1e-9)
    env.close()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_stay_on_their_device():
    from carl_amd import ops

    gen = torch.Generator().manual_seed(0)
    x, residual, weight, logits = (torch.randn(s, generator=gen).cuda(0) for s in ((200, 48), (200, 48), (48,), (200, 18)))
    actions = torch.zeros(200, 7, dtype=torch.int32).cuda(0)
    heads = (3, 3, 3, 2, 2, 3, 2)

    def program():
        leaves = [t.clone().requires_grad_() for t in (x, weight, logits)]
        y, total = ops.rms_norm(leaves[0], leaves[1], residual=residual)
        log_prob, entropy = ops.action_log_prob(leaves[2], actions, heads)
        grads = torch.autograd.grad([y, total, log_prob, entropy], leaves, [x, x, x[:, 0], x[:, 1]])
        codes, scale, _ = ops.rms_norm_int8(x, weight, residual=residual)
        inner = ops.int8_gated_linear(codes, scale, codes, scale, codes, scale)
        return (y.detach(), total.detach(), log_prob.detach(), entropy.detach(), *grads, codes, scale, inner,
                ops.int8_linear(*ops.quantize_int8(inner), *ops.quantize_int8(inner)), *ops.top_actions(logits, heads, 2))

    want = program()
    torch.cuda.synchronize(0)
    with torch.cuda.device(1):
        got = program()
        torch.cuda.synchronize(0)
        assert torch.cuda.current_device() == 1
    for a, b in zip(got, want):
        assert a.device == b.device and torch.equal(a, b)
