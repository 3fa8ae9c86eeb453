"""The example policy on the vector environment: acting step by step and the
chunked pass over the rollout agree, and training moves the policy."""
from __future__ import annotations

import importlib.util
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


def _setting(example, steps, **env):
    torch.manual_seed(0)
    env = example.CARLTorchVectorEnv(12, 1, 1, normalize=True, discrete_actions=True, **env)
    policy = example.RecurrentPolicy(env.single_observation_space.shape[0]).cuda()
    return env, policy, example.Rollout(policy, env, steps)


def test_steps_and_rollouts_agree(example):
    """Over two rollouts, with memories carried and episodes that end on the way."""
    env, policy, rollout = _setting(example, 40, no_touch_timeout_ticks=8 * 15)
    for _ in range(2):
        batch = rollout.collect()
        assert bool(batch["starts"][1:].any())
        with torch.no_grad():
            logits, _, memories = policy(batch["obs"], batch["memories"], batch["starts"])
        seen = torch.isfinite(batch["logits"])
        assert torch.equal(seen, torch.isfinite(logits))
        # float32 sums in another order, through two layers
        assert torch.allclose(logits[seen], batch["logits"][seen], rtol=0, atol=1e-4)
        for a, b in zip(memories, rollout.memories):
            assert torch.allclose(a, b, rtol=0, atol=1e-4 * float(b.abs().max()))
    env.close()


def _imitation(example, make, steps):
    """The losses of a policy that learns another one's likeliest actions on a rollout: a function of what it sees."""
    env, policy, rollout = _setting(example, 16)
    batch = rollout.collect()
    with torch.no_grad():
        teacher = example.RecurrentPolicy(batch["obs"].shape[-1]).cuda()
        teacher.act.weight.mul_(20.0)
        logits, _, _ = teacher(batch["obs"], batch["memories"], batch["starts"])
        actions = torch.stack([h.argmax(-1) for h in logits.split(example.ACTION_NVECS, dim=-1)], dim=-1)
    optimizer = make([p for n, p in policy.named_parameters() if not n.startswith("value")])
    losses = []
    for _ in range(steps):
        optimizer.zero_grad()
        logits, _, _ = policy(batch["obs"], batch["memories"], batch["starts"])
        loss = -example.log_prob(logits, actions).mean()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    assert all(bool(torch.isfinite(p.grad).all()) for n, p in policy.named_parameters() if not n.startswith("value"))
    env.close()
    return losses


def test_training_follows_torchs_adamw(example):
    """The same start, rollout and steps: float32 roundings apart, the same losses."""
    ours = _imitation(example, lambda ps: example.AdamW(ps, lr=1e-3, weight_decay=0.01), 20)
    theirs = _imitation(example, lambda ps: torch.optim.AdamW(ps, lr=1e-3, weight_decay=0.01, fused=False), 20)
    assert ours == pytest.approx(theirs, rel=1e-3)
    assert ours[-1] < ours[0]


def test_eight_bit_moments_train_as_well(example):
    eight = _imitation(example, lambda ps: example.AdamW(ps, lr=1e-3, bits=8), 60)
    full = _imitation(example, lambda ps: example.AdamW(ps, lr=1e-3), 60)
    assert eight[-1] < 0.5 * eight[0] and eight[-1] < 1.25 * full[-1]


def test_policy_gradient_updates_run(example):
    env, policy, rollout = _setting(example, 16)
    optimizer = example.AdamW(policy.parameters(), lr=3e-4, bits=8)
    before = [p.detach().clone() for p in policy.parameters()]
    for _ in range(3):
        assert example.update(policy, optimizer, rollout.collect()) == pytest.approx(0.0, abs=100.0)
    assert all(bool(torch.isfinite(p).all()) for p in policy.parameters())
    assert any(not torch.equal(a, b) for a, b in zip(before, policy.parameters()))
    env.close()


def test_the_loss_is_that_of_the_returns(example):
    """Returns by hand, in 64 bits: rewards to the episode's end, or to the rollout's and then the value of the
    observation after it, which a pass over one step more gives."""
    env, policy, rollout = _setting(example, 24, no_touch_timeout_ticks=8 * 15)
    with torch.no_grad():
        policy.value.weight.mul_(30.0)
    batch = rollout.collect()
    assert bool(batch["ends"].any()) and not bool(batch["ends"][-1].all())
    obs = torch.cat((batch["obs"], rollout.next_obs[None]))
    starts = torch.cat((batch["starts"], rollout.next_start[None]))
    with torch.no_grad():
        logits, values, _ = policy(obs, batch["memories"], starts)
    rewards, ends, values = batch["rewards"].double().cpu(), batch["ends"].cpu(), values.double().cpu()
    log_probs = example.log_prob(logits[:-1], batch["actions"]).double().cpu()

    def loss(after):
        total = 0.0
        for agent in range(rewards.shape[1]):
            for t in range(24):
                target, weight = 0.0, 1.0
                for s in range(t, 24):
                    target += weight * float(rewards[s, agent])
                    weight *= 0.99
                    if ends[s, agent]:
                        break
                else:
                    target += weight * float(after[agent])
                advantage = target - float(values[t, agent])
                total += -float(log_probs[t, agent]) * advantage + 0.5 * advantage ** 2
        return total / rewards.numel()

    # float32 values and log-probabilities of order 1 to 30, good to 1e-4 as the passes agree
    want, last = loss(values[24]), loss(values[23])
    assert abs(want - last) > 2e-2 * abs(want)
    assert example.update(policy, example.AdamW(policy.parameters(), lr=0.0), batch) == pytest.approx(want, rel=2e-3)
    env.close()
