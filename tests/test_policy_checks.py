"""What the operators around a policy's layers refuse, on the host (the C-ABI's
checks, which come before anything is queued, and the torch layer's), and their
64-bit references against autograd."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

import ops_reference as ref
import policy_reference as policy
from carl_amd import build, ops

OK, VALUE, TYPE = 0, -1, -2
P, I32, I64, F32 = C.c_void_p, C.c_int32, C.c_int64, C.c_float


class Actions(C.Structure):
    _fields_ = [("rows", I64), ("type", I32), ("heads", I32), ("sizes", C.POINTER(I32)), ("logits", P), ("logits_row", I64), ("mask", P),
                ("mask_row", I64), ("actions", P), ("actions_row", I64), ("actions_wide", I32), ("log_prob", P), ("entropy", P),
                ("d_log_prob", P), ("d_entropy", P), ("d_log_prob_step", I64), ("d_entropy_step", I64), ("d_logits", P), ("noise", P),
                ("noise_row", I64), ("k", I32), ("best", P)]


class Norm(C.Structure):
    _fields_ = [("rows", I64), ("width", I32), ("type", I32), ("eps", F32), ("x", P), ("x_row", I64), ("residual", P), ("residual_row", I64),
                ("weight", P), ("sum", P), ("y", P), ("codes", P), ("codes_row", I64), ("scale", P), ("sum_row", I64), ("dy", P),
                ("dy_row", I64), ("d_sum", P), ("d_sum_row", I64), ("d_x", P), ("d_weight", P), ("workspace", P)]


class Linear(C.Structure):
    _fields_ = [("rows", I64), ("width", I32), ("columns", I32), ("type", I32), ("activation", I32), ("x", P), ("x_row", I64), ("x_scale", P),
                ("w", P), ("w_row", I64), ("w_scale", P), ("w_up", P), ("w_up_row", I64), ("w_up_scale", P), ("bias", P), ("y", P)]


SOME = 4096        # an address that no call of these tests reads


@pytest.fixture(scope="module")
def lib():
    L = C.CDLL(str(build.engine_path()))
    L.carl_last_error.restype = C.c_char_p
    return L


def _with(struct, changes):
    for name, value in changes.items():
        setattr(struct, name, value)
    return struct


def _sizes(*sizes):
    return (I32 * max(1, len(sizes)))(*sizes)


def _actions(**changes):
    a = Actions(rows=4, heads=2, sizes=_sizes(3, 2), logits=SOME, logits_row=5, actions=SOME, actions_row=2, log_prob=SOME, entropy=SOME,
                d_logits=SOME, k=1, best=SOME)
    return _with(a, changes)


def _norm(**changes):
    return _with(Norm(rows=4, width=16, eps=1e-6, x=SOME, x_row=16, weight=SOME, sum=SOME, y=SOME, codes=SOME, codes_row=16, scale=SOME,
                      sum_row=16, dy=SOME, dy_row=16, d_x=SOME, d_weight=SOME, workspace=SOME), changes)


def _linear(**changes):
    return _with(Linear(rows=4, width=16, columns=8, x=SOME, x_row=16, x_scale=SOME, w=SOME, w_row=16, w_scale=SOME, y=SOME), changes)


BAD_HEADS = b"head sizes must be at least 1, and 16,384 in all at most"


@pytest.mark.parametrize("changes,code,message", [
    ({"type": 3}, TYPE, b"unknown element type"),
    ({"rows": -1}, VALUE, b"rows are out of range"),
    ({"rows": (1 << 40) + 1}, VALUE, b"rows are out of range"),
    ({"heads": 0}, VALUE, b"heads must be in [1, 64]"),
    ({"heads": 65, "sizes": _sizes(*[1] * 65)}, VALUE, b"heads must be in [1, 64]"),
    ({"sizes": None}, VALUE, b"null head sizes"),
    ({"sizes": _sizes(3, 0)}, VALUE, BAD_HEADS),
    ({"sizes": _sizes(-1, 3)}, VALUE, BAD_HEADS),
    ({"sizes": _sizes(16384, 1)}, VALUE, BAD_HEADS),
    ({"sizes": _sizes(1, 2 ** 31 - 1)}, VALUE, BAD_HEADS),
    ({"logits": None}, VALUE, b"null action tensor"),
])
def test_actions_refuse(lib, changes, code, message):
    for call in (lib.carl_action_log_prob, lib.carl_action_log_prob_backward, lib.carl_top_actions):
        assert call(C.byref(_actions(**changes)), None) == code
        assert lib.carl_last_error() == message
        assert call(None, None) == VALUE


def test_actions_refuse_what_a_call_needs(lib):
    for call, names in ((lib.carl_action_log_prob, ("actions", "log_prob", "entropy")),
                        (lib.carl_action_log_prob_backward, ("actions", "d_logits")), (lib.carl_top_actions, ("best", "log_prob"))):
        for name in names:
            assert call(C.byref(_actions(**{name: None})), None) == VALUE
            assert lib.carl_last_error() == b"null action tensor"
        # no rows need nothing
        assert call(C.byref(_actions(rows=0, **{n: None for n in names})), None) == OK
    for k in (0, 65):
        assert lib.carl_top_actions(C.byref(_actions(k=k)), None) == VALUE
        assert lib.carl_last_error() == b"k must be in [1, 64]"


@pytest.mark.parametrize("changes,code,message", [
    ({"type": 3}, TYPE, b"unknown element type"),
    ({"rows": -1}, VALUE, b"rows are out of range"),
    ({"rows": (1 << 40) + 1}, VALUE, b"rows are out of range"),
    ({"width": 0}, VALUE, b"width must be in [1, 16384]"),
    ({"width": 16385}, VALUE, b"width must be in [1, 16384]"),
    ({"eps": 0.0}, VALUE, b"eps must be finite and at least 1e-30"),
    ({"eps": 9e-31}, VALUE, b"eps must be finite and at least 1e-30"),
    ({"eps": -1.0}, VALUE, b"eps must be finite and at least 1e-30"),
    ({"eps": math.inf}, VALUE, b"eps must be finite and at least 1e-30"),
    ({"eps": math.nan}, VALUE, b"eps must be finite and at least 1e-30"),
    ({"weight": None}, VALUE, b"null weight"),
    ({"x": None, "sum": None}, VALUE, b"null norm tensor"),
])
def test_norm_refuses(lib, changes, code, message):
    for call in (lib.carl_rms_norm, lib.carl_rms_norm_int8, lib.carl_rms_norm_backward):
        assert call(C.byref(_norm(**changes)), None) == code
        assert lib.carl_last_error() == message
        assert call(None, None) == VALUE


def test_norm_refuses_what_a_call_needs(lib):
    for changes in ({"y": None}, {"residual": SOME, "sum": None}):
        assert lib.carl_rms_norm(C.byref(_norm(**changes)), None) == VALUE
    for changes in ({"codes": None}, {"scale": None}, {"residual": SOME, "sum": None}, {"codes_row": 15}):
        assert lib.carl_rms_norm_int8(C.byref(_norm(**changes)), None) == VALUE
    for changes in ({"x": None}, {"codes": None}, {"scale": None}, {"codes_row": 15}, {"width": 16385}, {"rows": -1}):
        assert lib.carl_quantize_int8(C.byref(_norm(**changes)), None) == VALUE
    assert lib.carl_rms_norm_backward(C.byref(_norm(dy=None)), None) == VALUE
    size = I64(-1)
    assert lib.carl_rms_norm_workspace(C.byref(_norm(rows=100_000)), C.byref(size)) == OK and size.value > 0 and size.value % (16 * 4) == 0
    assert lib.carl_rms_norm_backward(C.byref(_norm(rows=100_000, workspace=None)), None) == VALUE
    assert lib.carl_last_error() == b"null workspace"
    assert lib.carl_rms_norm_workspace(C.byref(_norm(rows=0)), C.byref(size)) == OK and size.value == 0
    assert lib.carl_rms_norm_workspace(C.byref(_norm()), None) == VALUE
    assert lib.carl_rms_norm_workspace(None, C.byref(size)) == VALUE
    # nothing to do is no error, and queues nothing
    assert lib.carl_rms_norm(C.byref(_norm(rows=0, x=None, y=None)), None) == OK
    assert lib.carl_rms_norm_backward(C.byref(_norm(d_x=None, d_weight=None)), None) == OK


@pytest.mark.parametrize("changes,code,message", [
    ({"type": -1}, TYPE, b"unknown element type"),
    ({"width": 0}, VALUE, b"width must be in [1, 65536]"),
    ({"width": 65537}, VALUE, b"width must be in [1, 65536]"),
    ({"columns": 0}, VALUE, b"columns must be in [1, 65536]"),
    ({"columns": 65537}, VALUE, b"columns must be in [1, 65536]"),
    ({"rows": -1}, VALUE, b"rows are out of range"),
    ({"rows": (1 << 28) + 1}, VALUE, b"rows are out of range"),
    ({"rows": (1 << 20) + 1, "columns": 65536}, VALUE, b"rows are out of range"),
    ({"w_up": SOME, "w_up_scale": SOME, "activation": 2}, VALUE, b"unknown activation"),
    ({"w_up": SOME, "w_up_scale": SOME, "bias": SOME}, VALUE, b"the gated product has no bias"),
    ({"w_up": SOME}, VALUE, b"null product tensor"),
    ({"x": None}, VALUE, b"null product tensor"),
    ({"x_scale": None}, VALUE, b"null product tensor"),
    ({"w": None}, VALUE, b"null product tensor"),
    ({"w_scale": None}, VALUE, b"null product tensor"),
    ({"y": None}, VALUE, b"null product tensor"),
])
def test_products_refuse(lib, changes, code, message):
    assert lib.carl_int8_linear_forward(C.byref(_linear(**changes)), None) == code
    assert lib.carl_last_error() == message
    assert lib.carl_int8_linear_forward(None, None) == VALUE
    assert lib.carl_int8_linear_forward(C.byref(_linear(rows=0, x=None, y=None)), None) == OK


# ------------------------------------------------------------------ torch layer

def _calls():
    x, w, c = torch.zeros(2, 8), torch.ones(8), torch.zeros(2, 8, dtype=torch.int8)
    s, a = torch.ones(2), torch.zeros(2, 2, dtype=torch.int32)
    return [(lambda t: ops.rms_norm(t, w), x), (lambda t: ops.rms_norm_int8(t, w), x), (lambda t: ops.quantize_int8(t), x),
            (lambda t: ops.action_log_prob(t, a, (5, 3)), x), (lambda t: ops.top_actions(t, (5, 3)), x),
            (lambda t: ops.int8_linear(c, s, c, t), s), (lambda t: ops.int8_gated_linear(c, t, c, s, c, s), s)]


def test_host_tensors_are_refused():
    for call, t in _calls():
        with pytest.raises(ValueError, match="must be on cuda:0"):
            call(t)


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        for call, t in _calls()[:5]:
            with pytest.raises(ValueError, match="has a forward-mode tangent"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))


def test_operators_without_a_gradient_say_so():
    for i, name in ((1, "rms_norm_int8"), (2, "quantize_int8"), (4, "top_actions"), (5, "int8_linear"), (6, "int8_gated_linear")):
        call, t = _calls()[i]
        with pytest.raises(ValueError, match=f"{name} has no gradient"):
            call(t.requires_grad_())


def test_arguments_that_fit_nothing_are_refused():
    x = torch.zeros(2, 8)
    a = torch.zeros(2, 2, dtype=torch.int32)
    for heads in ((), (1,) * 65, (8, 0), (-1, 9), (2 ** 40,), (9000, 9000)):
        with pytest.raises(ValueError):
            ops.action_log_prob(x, a, heads)
    for k in (0, 65, -1):
        with pytest.raises(ValueError, match="k must be in"):
            ops.top_actions(x, (8,), k)
    with pytest.raises(TypeError):
        ops.action_log_prob(x, a, "heads")
    c, s = torch.zeros(2, 8, dtype=torch.int8), torch.ones(2)
    for dtype in (torch.int8, torch.float64, None, "float32"):
        with pytest.raises(TypeError, match="dtype must be"):
            ops.int8_linear(c, s, c, s, dtype=dtype)
    with pytest.raises(ValueError, match="activation must be"):
        ops.int8_gated_linear(c, s, c, s, c, s, activation="relu")


def test_aliases():
    import carl.ops

    for name in ("rms_norm", "rms_norm_int8", "quantize_int8", "int8_linear", "int8_gated_linear", "action_log_prob", "top_actions"):
        assert getattr(carl.ops, name) is getattr(ops, name) and name in ops.__all__


# ---------------------------------------------------------- the 64-bit references

def test_reference_log_probabilities_are_autograds():
    gen = torch.Generator().manual_seed(0)
    heads = (4, 3, 9)
    x = torch.randn(6, 16, generator=gen)
    mask = torch.rand(6, 16, generator=gen) < 0.7
    mask[:, [0, 4, 7]] = True
    actions = torch.zeros(6, 3, dtype=torch.int32)
    d = torch.randn(2, 6, generator=gen)
    leaf = x.double().requires_grad_()
    total = entropy = 0.0
    for i, h in enumerate(leaf.masked_fill(~mask, -math.inf).split(heads, -1)):
        logs = h.log_softmax(-1)
        total = total + logs.gather(-1, actions[:, i:i + 1].long()).squeeze(-1)
        entropy = entropy - (logs.exp() * logs.masked_fill(torch.isinf(h), 0.0)).sum(-1)
    (grad,) = torch.autograd.grad([total, entropy], [leaf], [d[0].double(), d[1].double()])
    (lp, lp_off), (h, h_off) = policy.log_prob(x, actions, heads, mask)
    assert torch.allclose(lp, total, atol=1e-12) and torch.allclose(h, entropy, atol=1e-12)
    want, off = policy.log_prob_gradient(x, actions, heads, d[0], d[1], mask)
    assert torch.allclose(want, grad, atol=1e-12)
    for bound, value in ((lp_off, lp), (h_off, h), (off, want)):
        assert bool((bound >= 0).all()) and bool((bound <= 1e-4 * (1 + value.abs())).all())
    # a mistake in a mask, an action or a head's border is out of bounds
    for wrong in (policy.log_prob(x, actions, heads, None)[0][0], policy.log_prob(x, actions + 1, heads, mask)[0][0],
                  policy.log_prob(x, actions, (3, 4, 9), mask)[0][0]):
        with pytest.raises(AssertionError):
            ref.assert_within(wrong, lp, lp_off, "log-probability")
    best, logs, _ = policy.top(x, heads, 1, mask)
    assert torch.equal(best[:, 2, 0], x[:, 7:].masked_fill(~mask[:, 7:], -math.inf).argmax(-1).int())


def test_reference_norm_gradients_are_autograds():
    gen = torch.Generator().manual_seed(0)
    x, residual, dy, dsum = (torch.randn(5, 12, generator=gen) for _ in range(4))
    w = torch.randn(12, generator=gen)
    kept = policy.kept_sum(x, residual)
    s, weight = kept.double().requires_grad_(), w.double().requires_grad_()
    y = torch.nn.functional.rms_norm(s, (12,), weight, 1e-6)
    grads = torch.autograd.grad([y, s * 1.0], [s, weight], [dy.double(), dsum.double()])
    value, bound = policy.norm(x, w, residual, 1e-6, dy, dsum)
    for name, want in (("y", y), ("dx", grads[0]), ("dweight", grads[1])):
        assert torch.allclose(value[name], want, atol=1e-12), name
        assert bool((bound[name] > 0).all()) and bool((bound[name] < 1e-3).all())
    with pytest.raises(AssertionError):
        ref.assert_within(policy.norm(x, w, residual, 1e-2)[0]["y"], value["y"], bound["y"], "y")


def test_reference_codes_stand_for_their_rows():
    t = torch.randn(20, 100, generator=torch.Generator().manual_seed(0)) * torch.logspace(-35, 30, 20)[:, None]
    code, step = policy.codes(t)
    have = t.abs().amax(1) >= 2.0 ** -100
    off = (code.double() * step.double()[:, None] - t.double()).abs()
    assert bool((off[have] <= 0.50001 * step.double()[have, None]).all()) and bool((code.abs().amax(1)[have] == 127).all())
    t[3, 4] = math.nan
    code, step = policy.codes(t)
    assert torch.isnan(step[3]) and not code[3].any() and torch.isfinite(step[4:]).all()
