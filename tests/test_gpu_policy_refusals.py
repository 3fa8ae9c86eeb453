"""Refused calls of the operators around a policy's layers, on tensors of the GPU: nothing is queued for them."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ops():
    from carl_amd import ops

    return ops


def _refused(call, error, message):
    """The error, and no tensor made: copies of inputs that do not lie in rows come after all checks."""
    def allocations():
        return torch.cuda.memory_stats()["allocation.all.allocated"]

    before = allocations()
    with pytest.raises(error, match=message):
        call()
    assert allocations() == before


def _turned(*shape, dtype=torch.float32):
    """Rows whose elements do not lie next to each other."""
    return torch.zeros(*shape, dtype=dtype, device="cuda").mT.contiguous().mT


def test_actions_are_checked_before_logits_are_copied():
    ops = _ops()
    logits, mask = _turned(6, 8), _turned(6, 8, dtype=torch.bool)
    for actions, error, message in ((torch.zeros(6, 2, device="cuda"), TypeError, "actions must have dtype int32 or int64"),
                                    (torch.zeros(6, 3, device="cuda", dtype=torch.int32), ValueError, "actions must have shape"),
                                    (torch.zeros(5, 2, device="cuda", dtype=torch.int32), ValueError, "actions must have shape"),
                                    (torch.zeros(6, 2, dtype=torch.int32), ValueError, "actions must be on cuda:0")):
        for leaf in (logits, logits.detach().requires_grad_()):
            _refused(lambda: ops.action_log_prob(leaf, actions, (5, 3), mask=mask), error, message)


@pytest.mark.parametrize("eps", [0.0, 9e-31, -1.0, math.inf, math.nan, 1e39])
def test_eps_is_checked_before_rows_are_copied(eps):
    ops = _ops()
    x, residual, weight = _turned(6, 8), _turned(6, 8), torch.ones(16, device="cuda")[::2]
    for call in (ops.rms_norm, ops.rms_norm_int8):
        for r in (None, residual):
            _refused(lambda: call(x, weight, residual=r, eps=eps), ValueError, "eps must be finite and at least 1e-30")
    leaf = x.detach().requires_grad_()
    _refused(lambda: ops.rms_norm(leaf, weight, eps=eps), ValueError, "eps must be finite and at least 1e-30")


def test_biases_and_rows_are_checked_before_codes_are_copied():
    ops = _ops()
    x, w, up = (_turned(n, 32, dtype=torch.int8) for n in (6, 12, 12))
    x_scale, w_scale = torch.ones(12, device="cuda")[::2], torch.ones(24, device="cuda")[::2]
    for bias, error, message in ((torch.zeros(12, device="cuda"), TypeError, "bias must have the result's dtype"),
                                 (torch.zeros(13, device="cuda", dtype=torch.bfloat16), ValueError, "bias must have shape"),
                                 (torch.zeros(12, dtype=torch.bfloat16), ValueError, "bias must be on cuda:0")):
        _refused(lambda: ops.int8_linear(x, x_scale, w, w_scale, bias=bias), error, message)
    rows, scales = x[:1].expand((1 << 28) + 1, 32), x_scale[:1].expand((1 << 28) + 1)
    _refused(lambda: ops.int8_linear(rows, scales, w, w_scale), ValueError, "rows are out of range")
    _refused(lambda: ops.int8_gated_linear(rows, scales, w, w_scale, up, w_scale), ValueError, "rows are out of range")
    wide, wide_scale = w[:1].expand(65_536, 32), w_scale[:1].expand(65_536)
    rows, scales = x[:1].expand((1 << 20) + 1, 32), x_scale[:1].expand((1 << 20) + 1)
    _refused(lambda: ops.int8_linear(rows, scales, wide, wide_scale), ValueError, "rows are out of range")
