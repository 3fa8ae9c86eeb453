"""What the learner's operators refuse, on the host: the C-ABI's checks, which
come before anything is queued, and the torch layer's."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

import carl_amd
import ops_reference as ref
from carl_amd import build, ops, optim

OK, VALUE, TYPE = 0, -1, -2
P, I32, I64, F32, F64 = C.c_void_p, C.c_int32, C.c_int64, C.c_float, C.c_double


class Rows(C.Structure):
    _fields_ = [("data", P), ("batch", I64), ("step", I64), ("head", I64)]


class Attention(C.Structure):
    _fields_ = [("batch", I64), ("steps", I64), ("heads", I32), ("kv_heads", I32), ("key_dim", I32), ("value_dim", I32),
                ("type", I32), ("scale", F32), ("q", Rows), ("k", Rows), ("v", Rows), ("out", Rows), ("log_decay", P),
                ("starts", P), ("starts_batch", I64), ("starts_step", I64), ("initial_state", P), ("final_state", P),
                ("d_out", Rows), ("d_q", Rows), ("d_k", Rows), ("d_v", Rows), ("d_final_state", P), ("d_initial_state", P),
                ("workspace", P)]


class Ffn(C.Structure):
    _fields_ = [("rows", I64), ("width", I32), ("inner", I32), ("type", I32), ("activation", I32), ("x", P), ("x_row", I64),
                ("w_gate", P), ("w_up", P), ("w_down", P), ("y", P), ("dy", P), ("dy_row", I64), ("dx", P), ("dw_gate", P),
                ("dw_up", P), ("dw_down", P), ("workspace", P)]


class Tensor(C.Structure):
    _fields_ = [("param", P), ("grad", P), ("exp_avg", P), ("exp_avg_sq", P), ("exp_avg_scale", P), ("exp_avg_sq_scale", P),
                ("n", I64), ("param_type", I32), ("grad_type", I32)]


class Hyper(C.Structure):
    _fields_ = [("lr", F64), ("beta1", F64), ("beta2", F64), ("eps", F64), ("weight_decay", F64), ("step", I64),
                ("bits", I32), ("grad_scale", P)]


SOME = 4096        # an address that no call of these tests reads


@pytest.fixture(scope="module")
def lib():
    L = C.CDLL(str(build.engine_path()))
    L.carl_last_error.restype = C.c_char_p
    L.carl_adamw_decode.argtypes = L.carl_adamw_encode.argtypes = [P, P, P, P, I64, P, P, P]
    L.carl_adamw_encode.argtypes = [P, P, I64, P, P, P, P, P]
    return L


def _attention(**changes):
    a = Attention(batch=2, steps=3, heads=2, kv_heads=1, key_dim=16, value_dim=16, type=0, scale=1.0, log_decay=SOME, workspace=SOME)
    for name in ("q", "k", "v", "out", "d_out", "d_q", "d_k", "d_v"):
        setattr(a, name, Rows(SOME, 96, 32, 16))
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def _ffn(**changes):
    f = Ffn(rows=4, width=16, inner=32, type=0, activation=0, x=SOME, x_row=16, w_gate=SOME, w_up=SOME, w_down=SOME, y=SOME,
            dy=SOME, dy_row=16, dx=SOME, workspace=SOME)
    for name, value in changes.items():
        setattr(f, name, value)
    return f


def _hyper(**changes):
    h = Hyper(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, step=1, bits=32)
    for name, value in changes.items():
        setattr(h, name, value)
    return h


NONE = Rows(None, 0, 0, 0)


@pytest.mark.parametrize("changes,code,message", [
    ({"type": 3}, TYPE, b"unknown element type"),
    ({"batch": -1}, VALUE, b"batch and steps must be non-negative"),
    ({"steps": -1}, VALUE, b"batch and steps must be non-negative"),
    ({"heads": 0}, VALUE, b"heads must be in [1, 65535]"),
    ({"heads": 65536, "kv_heads": 65536}, VALUE, b"heads must be in [1, 65535]"),
    ({"kv_heads": 0}, VALUE, b"heads must be a multiple of kv_heads"),
    ({"heads": 3, "kv_heads": 2}, VALUE, b"heads must be a multiple of kv_heads"),
    ({"key_dim": 0}, VALUE, b"key_dim must be in [1, 128]"),
    ({"key_dim": 129}, VALUE, b"key_dim must be in [1, 128]"),
    ({"value_dim": 0}, VALUE, b"value_dim must be in [1, 128]"),
    ({"value_dim": 129}, VALUE, b"value_dim must be in [1, 128]"),
    ({"batch": (1 << 21) + 1}, VALUE, b"batch times heads must be at most 4,194,304"),
    ({"steps": (1 << 40) + 1}, VALUE, b"too many steps"),
    ({"log_decay": None}, VALUE, b"null log_decay"),
    ({"q": NONE}, VALUE, b"null attention input"),
    ({"k": NONE}, VALUE, b"null attention input"),
    ({"v": NONE}, VALUE, b"null attention input"),
])
def test_attention_refuses(lib, changes, code, message):
    a = _attention(**changes)
    for call in (lib.carl_linear_attention, lib.carl_linear_attention_backward):
        assert call(C.byref(a), None) == code
        assert lib.carl_last_error() == message
    if "steps" not in changes:
        a.steps = 1
        assert lib.carl_linear_attention_step(C.byref(a), P(SOME), None) == code


def test_attention_refuses_missing_outputs(lib):
    for call in (lib.carl_linear_attention, lib.carl_linear_attention_backward):
        assert call(None, None) == VALUE
    assert lib.carl_linear_attention(C.byref(_attention(out=NONE)), None) == VALUE
    assert lib.carl_last_error() == b"null attention output"
    for name in ("d_out", "d_q", "d_k", "d_v"):
        assert lib.carl_linear_attention_backward(C.byref(_attention(**{name: NONE})), None) == VALUE
        assert lib.carl_last_error() == b"null attention gradient"
    # shared heads need scratch memory backwards, long sequences both ways
    assert lib.carl_linear_attention_backward(C.byref(_attention(workspace=None)), None) == VALUE
    assert lib.carl_last_error() == b"null workspace"
    assert lib.carl_linear_attention(C.byref(_attention(steps=5000, workspace=None)), None) == VALUE
    assert lib.carl_last_error() == b"null workspace"
    assert lib.carl_linear_attention_step(C.byref(_attention(steps=3)), P(SOME), None) == VALUE
    assert lib.carl_last_error() == b"steps must be 1"
    assert lib.carl_linear_attention_step(C.byref(_attention(steps=1)), None, None) == VALUE
    assert lib.carl_last_error() == b"null state"


def test_attention_workspace_needs_no_tensors(lib):
    size = I64(-1)
    bare = _attention(log_decay=None, **{n: NONE for n in ("q", "k", "v", "out", "d_out", "d_q", "d_k", "d_v")})
    assert lib.carl_linear_attention_workspace(C.byref(bare), 0, C.byref(size)) == OK and size.value == 0
    assert lib.carl_linear_attention_workspace(C.byref(bare), 1, C.byref(size)) == OK
    assert size.value >= 2 * 3 * 2 * 32 * 4 and size.value % 256 == 0
    bare.steps = 0
    assert lib.carl_linear_attention_workspace(C.byref(bare), 1, C.byref(size)) == OK and size.value == 0
    assert lib.carl_linear_attention_workspace(C.byref(bare), 1, None) == VALUE
    bare.heads = 0
    assert lib.carl_linear_attention_workspace(C.byref(bare), 0, C.byref(size)) == VALUE


@pytest.mark.parametrize("changes,code,message", [
    ({"type": -1}, TYPE, b"unknown element type"),
    ({"activation": 2}, VALUE, b"unknown activation"),
    ({"width": 0}, VALUE, b"width must be in [1, 65536]"),
    ({"width": 65537}, VALUE, b"width must be in [1, 65536]"),
    ({"inner": 0}, VALUE, b"inner must be in [1, 65536]"),
    ({"inner": 65537}, VALUE, b"inner must be in [1, 65536]"),
    ({"rows": -1}, VALUE, b"rows are out of range"),
    ({"rows": 1 << 40}, VALUE, b"rows are out of range"),
    ({"w_gate": None}, VALUE, b"null weights"),
    ({"w_up": None}, VALUE, b"null weights"),
    ({"w_down": None}, VALUE, b"null weights"),
    ({"x": None}, VALUE, b"null feed-forward tensor"),
    ({"y": None, "dy": None}, VALUE, b"null feed-forward tensor"),
    ({"workspace": None}, VALUE, b"null workspace"),
])
def test_ffn_refuses(lib, changes, code, message):
    f = _ffn(**changes)
    for call in (lib.carl_gated_ffn, lib.carl_gated_ffn_backward):
        assert call(C.byref(f), None) == code
        assert lib.carl_last_error() == message
    assert lib.carl_gated_ffn(None, None) == VALUE


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_ffn_takes_what_its_tiles_reach(lib, kind, backward):
    """2^36 elements in tiles of 128 x 128 (float32: 128 x 64), 2^28 rows."""
    size = I64(-1)

    def rc(**changes):
        return lib.carl_gated_ffn_workspace(C.byref(_ffn(type=kind, **changes)), backward, C.byref(size))

    assert rc(rows=1 << 20, width=8192, x_row=8192, dy_row=8192) == OK
    assert rc(rows=1 << 20, width=65536, inner=65536, x_row=65536, dy_row=65536) == OK
    assert size.value >= (1 << 36) * (4 if kind == 0 else 2)
    assert rc(rows=1 << 28) == OK
    for changes in ({"rows": (1 << 20) + 1, "width": 65536}, {"rows": (1 << 28) + 1}, {"rows": 1 << 28, "inner": 257}):
        assert rc(**changes) == VALUE
        assert lib.carl_last_error() == b"rows are out of range"


@pytest.mark.parametrize("changes,message", [
    ({"bits": 16}, b"moments must have 8 or 32 bits"),
    ({"step": 0}, b"step must be at least 1"),
    ({"beta1": 1.0}, b"betas must be in [0, 1)"),
    ({"beta2": -0.1}, b"betas must be in [0, 1)"),
    ({"beta1": float("nan")}, b"betas must be in [0, 1)"),
    ({"lr": -1.0}, b"lr must be finite and non-negative"),
    ({"lr": float("inf")}, b"lr must be finite and non-negative"),
    ({"eps": -1.0}, b"eps must be finite and non-negative"),
    ({"weight_decay": float("nan")}, b"weight_decay must be finite and non-negative"),
])
def test_adamw_refuses_hyperparameters(lib, changes, message):
    assert lib.carl_adamw_step(None, 0, C.byref(_hyper(**changes)), None) == VALUE
    assert lib.carl_last_error() == message


def test_adamw_refuses_tensors(lib):
    def step(bits=32, **changes):
        t = Tensor(SOME, SOME, SOME, SOME, SOME, SOME, 10, 0, 0)
        for name, value in changes.items():
            setattr(t, name, value)
        return lib.carl_adamw_step(C.byref(t), 1, C.byref(_hyper(bits=bits)), None), lib.carl_last_error()

    assert step(n=-1) == (VALUE, b"a tensor's size is out of range")
    assert step(n=(1 << 33) + 1) == (VALUE, b"a tensor's size is out of range")
    assert step(param_type=3)[0] == TYPE and step(grad_type=-1)[0] == TYPE
    for name in ("param", "grad", "exp_avg", "exp_avg_sq"):
        assert step(**{name: None}) == (VALUE, b"null AdamW tensor")
    for name in ("exp_avg_scale", "exp_avg_sq_scale"):
        assert step(bits=8, **{name: None}) == (VALUE, b"8-bit moments need their scales")
    assert lib.carl_adamw_step(None, 1, C.byref(_hyper()), None) == VALUE
    assert lib.carl_adamw_step(None, 0, None, None) == VALUE
    assert lib.carl_adamw_step(None, -1, C.byref(_hyper()), None) == VALUE
    # nothing to do is no error, and queues nothing
    assert lib.carl_adamw_step(None, 0, C.byref(_hyper()), None) == OK
    assert step(n=0, param=None)[0] == OK
    assert lib.carl_adamw_decode(None, None, None, None, 0, None, None, None) == OK
    assert lib.carl_adamw_decode(None, None, None, None, 1, None, None, None) == VALUE
    assert lib.carl_adamw_encode(None, None, -1, None, None, None, None, None) == VALUE


# ------------------------------------------------------------------ torch layer

def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 3, 2, 16), torch.zeros(2, dtype=torch.float32)
    with pytest.raises(ValueError, match="q must be on cuda:0"):
        ops.linear_attention(x, x, x, w)
    with pytest.raises(ValueError, match="q must be on cuda:0"):
        ops.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], w, torch.zeros(2, 2, 16, 16))
    with pytest.raises(ValueError, match="x must be on cuda:0"):
        ops.gated_ffn(x, torch.zeros(4, 16), torch.zeros(4, 16), torch.zeros(16, 4))
    with pytest.raises(ValueError, match="activation must be 'silu' or 'gelu'"):
        ops.gated_ffn(x, torch.zeros(4, 16), torch.zeros(4, 16), torch.zeros(16, 4), activation="relu")
    one = [torch.zeros(4)]
    with pytest.raises(ValueError, match="params must be on cuda:0"):
        optim.adamw_step(one, one, one, one, step=1, lr=1e-3)
    with pytest.raises(ValueError, match="same length"):
        optim.adamw_step(one, [], one, one, step=1, lr=1e-3)
    with pytest.raises(ValueError, match="have no scales"):
        optim.adamw_step(one, one, one, one, step=1, lr=1e-3, exp_avg_scale=one)
    with pytest.raises(ValueError, match="moments must be on cuda:0"):
        optim.encode_moments(one[0], one[0])


def test_forward_mode_tangents_are_refused():
    """A dual tensor needs no gradient, so a call would run, and its result would have no tangent."""
    from torch.autograd import forward_ad

    x, w, w_down, decay, state = torch.zeros(2, 3, 2, 16), torch.zeros(4, 16), torch.zeros(16, 4), torch.zeros(2), torch.zeros(2, 2, 16, 16)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = [lambda: ops.gated_ffn(dual(x), w, w, w_down), lambda: ops.linear_attention(dual(x), x, x, decay),
                 lambda: ops.linear_attention_step(dual(x[:, 0]), x[:, 0], x[:, 0], decay, state),
                 lambda: optim.adamw_step([dual(decay)], [decay], [decay], [decay], step=1, lr=1e-3),
                 lambda: optim.encode_moments(dual(decay), decay)]
        for call in calls:
            with pytest.raises(ValueError, match="has a forward-mode tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="has a forward-mode tangent"):
                call()
        with torch.inference_mode(), pytest.raises(ValueError, match="must be on cuda:0"):
            ops.gated_ffn(x, w, w, w_down)


@pytest.mark.parametrize("changes", [{"bits": 4}, {"lr": -1.0}, {"betas": (1.0, 0.9)}, {"eps": -1.0}, {"weight_decay": -1.0}])
def test_optimizer_refuses(changes):
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(2))], **changes)


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate parameters")
def test_the_optimizer_refuses_groups():
    """A parameter that is listed twice (two threads of a launch would step it at once), and other bits in a group."""
    p, q = (torch.nn.Parameter(torch.zeros(2)) for _ in range(2))
    with pytest.raises(ValueError, match="in the group twice"):
        optim.AdamW([p, q, p])
    with pytest.raises(ValueError, match="bits must be 8 or 32"):
        optim.AdamW([{"params": [p], "bits": 16}])
    opt = optim.AdamW([p], bits=8)
    for group in ({"params": [q, q]}, {"params": [q], "bits": 4}):
        with pytest.raises(ValueError):
            opt.add_param_group(group)
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [q], "bits": 32})
    assert [g["bits"] for g in opt.param_groups] == [8, 32]


def test_the_optimizer_refuses_to_be_captured(monkeypatch):
    """Before anything is done: no state is made, the closure is not called."""
    p = torch.nn.Parameter(torch.zeros(2))
    p.grad = torch.ones(2)
    opt = optim.AdamW([p])
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="counts its steps on the host"):
        opt.step(lambda: pytest.fail("called"))
    assert not opt.state


def test_aliases():
    import carl.ops
    import carl.optim

    assert carl.ops.linear_attention is ops.linear_attention and carl.optim.AdamW is optim.AdamW
    assert carl_amd.Env is not None


# ---------------------------------------------------------- the 64-bit references

def _attention_inputs():
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    starts = torch.tensor([[False, False, True, False, False], [True, False, False, False, True]])
    return r(2, 5, 4, 3), r(2, 5, 2, 3), r(2, 5, 2, 6), torch.tensor([-0.1, -0.5, 0.0, -2.0]), starts, r(2, 4, 3, 6), r(2, 5, 4, 6), r(2, 4, 3, 6)


def test_reference_attention_gradients_are_autograds():
    q, k, v, log_decay, starts, memory, dout, dfinal = _attention_inputs()
    leaves = [x.requires_grad_() for x in (q, k, v, memory)]

    def program(q, k, v, memory):          # the same sums as a masked product of all pairs of steps
        T, group = q.shape[1], q.shape[2] // k.shape[2]
        k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
        t = torch.arange(T)
        episode = starts.long().cumsum(1)
        gap = (t[:, None] - t[None]).clamp(min=0)
        w = torch.exp(log_decay.double()[:, None, None] * gap) * (t[:, None] >= t[None])
        w = w[None] * (episode[:, :, None] == episode[:, None])[:, None]
        into = torch.exp(log_decay.double()[None, :, None] * (t + 1)) * (episode == 0)[:, None]
        out = torch.einsum("bthd,bshd,bhts,bshe->bthe", q, k, w, v) + torch.einsum("bthd,bhde,bht->bthe", q, memory, into)
        last = w[:, :, -1]
        final = torch.einsum("bhs,bshd,bshe->bhde", last, k, v) + memory * into[:, :, -1, None, None]
        return out * 3 ** -0.5, final

    out, final = program(*leaves)
    want, last = ref.attention(q, k, v, log_decay, starts, memory)
    assert torch.allclose(out, want, rtol=1e-12, atol=1e-12) and torch.allclose(final, last, rtol=1e-12, atol=1e-12)
    grads = torch.autograd.grad([out, final], leaves, [dout, dfinal])
    for a, b in zip(grads, ref.attention_gradients(q, k, v, log_decay, dout, starts, memory, dfinal)):
        assert torch.allclose(a, b, rtol=1e-11, atol=1e-11)


def test_reference_ffn_gradients_are_autograds():
    gen = torch.Generator().manual_seed(0)
    leaves = [torch.randn(*s, generator=gen, dtype=torch.float32).double() for s in ((5, 4), (7, 4), (7, 4), (4, 7))]
    dy = torch.randn(5, 4, generator=gen).double()
    for name, act in (("silu", torch.nn.functional.silu), ("gelu", lambda g: torch.nn.functional.gelu(g, approximate="tanh"))):
        x, wg, wu, wd = (t.clone().requires_grad_() for t in leaves)
        y = (act(x @ wg.t()) * (x @ wu.t())) @ wd.t()
        grads = torch.autograd.grad(y, (x, wg, wu, wd), dy)
        value, bound = ref.ffn(*(t.float() for t in leaves), name, dy)
        for n, want in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), (y, *grads)):
            assert torch.allclose(value[n], want, rtol=1e-9, atol=1e-9), n
            assert bool((bound[n] > 0).all())


def test_a_planted_mistake_is_out_of_bounds():
    """The bounds catch a wrong decay, a missed start and a transposed memory (planted in the 64-bit reference)."""
    q, k, v, log_decay, starts, memory, _, _ = _attention_inputs()
    want, _ = ref.attention(q, k, v, log_decay, starts, memory)
    size, _ = ref.magnitudes(ref.attention, q, k, v, log_decay, starts, memory)
    bound = ref.attention_bound(torch.bfloat16, want, size, 5, 3)
    wrong = [ref.attention(q, k, v, log_decay - 0.05, starts, memory)[0], ref.attention(q, k, v, log_decay, None, memory)[0],
             ref.attention(q, k, v, log_decay, starts, memory.flip(2))[0]]
    for w in wrong:
        with pytest.raises(AssertionError):
            ref.assert_within(w, want, bound, "out")


def test_eight_bit_codes_keep_what_the_header_says():
    rng = np.random.default_rng(0)
    m = (rng.normal(size=4096) * 10.0 ** rng.uniform(-4, 0, 4096)).astype(np.float32)
    code, scale = ref.encode(m, False)
    top = np.abs(m) > 0.5 * np.repeat(scale, 256)
    assert (np.abs(ref.decode(code, scale, False) - m)[top] <= 0.016 * np.abs(m)[top]).all()
    v = (m * m).astype(np.float32)
    code, scale = ref.encode(v, True)
    assert (code[v > 0] >= 1).all()
    back = ref.decode(code, scale, True)
    top = v > 0.5 * np.repeat(scale, 256)
    assert (np.abs(np.sqrt(back) - np.sqrt(v))[top] <= 0.006 * np.sqrt(v)[top]).all()
