"""The operators while another device than their tensors' is the current one."""
from __future__ import annotations

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")]


def test_tensors_stay_on_their_device():
    from carl_amd import ops, optim

    gen = torch.Generator().manual_seed(0)
    x, w, w_down = (torch.randn(s, generator=gen).cuda(0) for s in ((40, 32), (48, 32), (32, 48)))
    q, k, v, state = (torch.randn(s, generator=gen).cuda(0) for s in ((2, 30, 2, 16), (2, 30, 2, 16), (2, 30, 2, 24), (2, 2, 16, 24)))
    decay = torch.tensor([-0.1, -0.01]).cuda(0)

    def program():
        leaves = [t.clone().requires_grad_() for t in (q, k, v, x)]
        memory, p, m, s = state.clone(), w.clone(), torch.zeros_like(w), torch.zeros_like(w)
        out, final = ops.linear_attention(*leaves[:3], decay, initial_state=state)
        y = ops.gated_ffn(leaves[3], w, w, w_down)
        grads = torch.autograd.grad([out, y], leaves, [v.expand_as(out), x])
        step = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, memory)
        optim.adamw_step([p], [w], [m], [s], step=1, lr=1e-3)
        return (out.detach(), final.detach(), y.detach(), *grads, step, memory, p, m, s, *optim.encode_moments(m, s))

    want = program()
    torch.cuda.synchronize(0)
    with torch.cuda.device(1):
        got = program()
        torch.cuda.synchronize(0)
        assert torch.cuda.current_device() == 1
    for a, b in zip(got, want):
        assert a.device == b.device and torch.equal(a, b)
