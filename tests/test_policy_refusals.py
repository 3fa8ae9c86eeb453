"""What the torch layer of the operators around a policy's layers refuses, on host tensors: types and shapes are looked
at before the device."""
from __future__ import annotations

import pytest

import policy_refusals as refusals


def test_calls_that_fit_reach_the_check_of_the_device():
    for call in refusals.calls("cpu").values():
        with pytest.raises(ValueError, match="must be on cuda:0"):
            call()


@pytest.mark.parametrize("group", refusals.GROUPS)
def test_types_and_shapes(group):
    for name, changes, error, message in refusals.GROUPS[group]:
        with pytest.raises(error, match=message):
            refusals.calls("cpu")[name](**refusals.made(changes, "cpu"))


def test_every_argument_is_looked_at():
    """Of each operator every tensor has a wrong type and a wrong shape among the cases."""
    for name, tensors in (("action_log_prob", ("logits", "mask", "actions")), ("top_actions", ("logits", "mask", "noise")),
                          ("rms_norm", ("x", "weight", "residual")), ("rms_norm_int8", ("x", "weight", "residual")), ("quantize_int8", ("x",)),
                          ("int8_linear", ("x", "x_scale", "weight", "weight_scale", "bias")),
                          ("int8_gated_linear", ("x", "x_scale", "w_gate", "gate_scale", "w_up", "up_scale"))):
        for tensor in tensors:
            errors = {case[2] for case in refusals.GROUPS[f"{name}-{tensor}"]}
            assert errors == {TypeError, ValueError}, (name, tensor)
