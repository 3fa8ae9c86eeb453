"""Refused calls of the operators around a policy's layers, on tensors of the GPU: every check of types and shapes, and
that nothing is queued for them."""
from __future__ import annotations

import math

import pytest
import torch

import policy_refusals as refusals

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


@pytest.mark.parametrize("group", refusals.GROUPS)
def test_types_and_shapes(group):
    calls = refusals.calls("cuda")
    for name, changes, error, message in refusals.GROUPS[group]:
        a = refusals.made(changes, "cuda")
        with pytest.raises(error, match=message):
            calls[name](**a)


def test_calls_that_fit_are_taken():
    for call in refusals.calls("cuda").values():
        call()


@pytest.mark.parametrize("name,tensors", [("action_log_prob", ("logits", "mask", "actions")), ("top_actions", ("logits", "mask", "noise")),
                                          ("rms_norm", ("x", "weight", "residual")), ("rms_norm_int8", ("x", "weight", "residual")),
                                          ("quantize_int8", ("x",)), ("int8_linear", ("x", "x_scale", "weight", "weight_scale", "bias")),
                                          ("int8_gated_linear", ("x", "x_scale", "w_gate", "gate_scale", "w_up", "up_scale"))])
def test_each_tensor_has_to_be_on_the_gpu(name, tensors):
    shapes = {"logits": (4, 6, 8), "mask": (4, 6, 8), "noise": (4, 6, 8), "actions": (4, 6, 2), "residual": (4, 6, 16), "x_scale": (4, 6),
              "bias": (12,)}
    for tensor in tensors:
        codes = "linear" in name and tensor in ("x", "weight", "w_gate", "w_up")
        shape = (4, 6, 32) if codes and tensor == "x" else (12, 32) if codes else (4, 6, 16) if tensor == "x" \
            else (16,) if tensor == "weight" else shapes.get(tensor, (12,))
        dtype = torch.int8 if codes else {"mask": torch.bool, "actions": torch.int32, "bias": torch.bfloat16}.get(
            tensor, torch.bfloat16 if "norm" in name else torch.float32)
        with pytest.raises(ValueError, match=f"{tensor} must be on cuda:0"):
            refusals.calls("cuda")[name](**{tensor: torch.zeros(*shape, dtype=dtype)})


def test_second_derivatives_are_refused():
    ops = _ops()
    logits = torch.randn(4, 8, device="cuda", requires_grad=True)
    actions = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    x, weight = torch.randn(4, 16, device="cuda", requires_grad=True), torch.ones(16, device="cuda", requires_grad=True)
    for name, out, leaf in (("action_log_prob", ops.action_log_prob(logits, actions, (5, 3))[0], logits), ("rms_norm", ops.rms_norm(x, weight), x),
                            ("rms_norm", ops.rms_norm(x, weight, residual=x)[0], weight)):
        with pytest.raises(RuntimeError, match=f"{name} has no second derivative"):
            torch.autograd.grad(out.sum(), [leaf], create_graph=True)


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
