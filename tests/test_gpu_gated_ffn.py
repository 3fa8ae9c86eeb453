"""The gated feed-forward block on the GPU against its definition in 64 bits:
outputs and gradients over sizes, types, activations, strides and alignments."""
from __future__ import annotations

import math

import pytest
import torch

import ops_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
GRADS = ("dx", "dw_gate", "dw_up", "dw_down")


def _ops():
    from carl_amd import ops

    return ops


def _inputs(N, D, F, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    shapes = ((N, D), (F, D), (F, D), (D, F), (N, D))
    scales = (1.0, D ** -0.5, D ** -0.5, F ** -0.5, 1.0)
    return [(torch.randn(s, generator=gen) * c).to(dtype).cuda() for s, c in zip(shapes, scales)]


def _check(x, w_gate, w_up, w_down, dy, activation="silu"):
    leaves = [t.detach().requires_grad_() for t in (x, w_gate, w_up, w_down)]
    y = _ops().gated_ffn(*leaves, activation=activation)
    assert y.shape == x.shape and y.dtype == x.dtype
    grads = torch.autograd.grad(y, leaves, dy)
    value, bound = ref.ffn(x, w_gate, w_up, w_down, activation, dy)
    ref.assert_within(y, value["y"], bound["y"], "y")
    for name, got, leaf in zip(GRADS, grads, leaves):
        assert got.shape == leaf.shape and got.dtype == leaf.dtype
        ref.assert_within(got, value[name], bound[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("N", [1, 2, 16, 17, 33, 34, 63, 65, 128, 129, 257, 1000])
def test_rows(N, activation, dtype):
    _check(*_inputs(N, 64, 136, dtype, seed=N), activation)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D,F", [(1, 1), (1, 300), (300, 1), (7, 13), (31, 33), (64, 683), (333, 201), (129, 130), (264, 520)])
def test_widths(D, F, dtype):
    _check(*_inputs(70, D, F, dtype, seed=D * 1000 + F))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N,D,F", [(4100, 64, 96), (5003, 136, 264), (8192, 256, 320), (4097, 33, 65)])
def test_many_rows(N, D, F, dtype):
    """Large tiles, and sums over rows split over workgroups."""
    _check(*_inputs(N, D, F, dtype, seed=N), "gelu")


@pytest.mark.parametrize("dtype,N,D,F", [
    (torch.bfloat16, 33_000, 512, 70), (torch.bfloat16, 8_192, 1024, 600), (torch.float16, 2_000, 1024, 2049),
    (torch.float32, 25_000, 300, 520), (torch.float32, 8_000, 200, 300), (torch.float32, 9_001, 256, 96)])
def test_every_tile(dtype, N, D, F):
    """Sizes on both sides of each rule that chooses a product's tiles."""
    _check(*_inputs(N, D, F, dtype, seed=N))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_large_activations(dtype):
    """Gates far into both tails: no overflow on the way, and the block stays finite."""
    x, w_gate, w_up, w_down, dy = _inputs(40, 32, 48, dtype)
    for activation in ("silu", "gelu"):
        _check(x, w_gate * 40, w_up, w_down, dy, activation)


@pytest.mark.parametrize("what,factors", [
    ("inner values of 100,000 and more", (1.0, 400.0, 400.0, 0.01, 0.001)),
    ("inner values below float16's normal numbers", (1.0, 0.002, 0.002, 64.0, 0.01)),
    ("gradients of outputs below them", (1.0, 30.0, 1.0, 1.0, 2.0 ** -18)),
    ("gradients of projections past its largest", (0.002, 0.002, 640.0, 256.0, 512.0))])
@pytest.mark.parametrize("N", [20, 100, 200, 5000])
def test_float16_keeps_what_its_range_does_not_hold(N, what, factors, monkeypatch):
    """Inputs and results are within float16's range, values on the way are not: each is off by one rounding all the same."""
    tensors = [t * f for t, f in zip(_inputs(N, 40, 56, torch.float16), factors)]
    if "below float16's normal" in what:
        tensors[0][N // 2] *= 32.0        # a row that stands out
    x, w_gate, w_up, w_down, dy = tensors
    leaves = [t.detach().requires_grad_() for t in tensors[:4]]
    y = _ops().gated_ffn(*leaves)
    got = dict(zip(("y", *GRADS), (y, *torch.autograd.grad(y, leaves, dy))))
    monkeypatch.setitem(ref.TINY, torch.float16, 0.0)
    value, bound = ref.ffn(*tensors[:4], "silu", dy)
    # 2^-25 of values that are written times what takes the product of the largest norms to at least 2^14
    xs, gs, us, ds, ys = (ref.wide(t).abs() for t in tensors)
    norm = [t.square().sum(d).sqrt().max() for t, d in ((xs, 1), (gs, 1), (us, 1), (ds, 0), (ys, 1))]
    h = 2.0 ** -39 * norm[0] ** 2 * norm[1] * norm[2]
    d = 2.0 ** -39 * norm[4] * norm[3] * norm[0] * torch.maximum(norm[1], norm[2])
    more = {"y": h * ds.sum(1), "dx": d * (gs.sum(0) + us.sum(0)), "dw_gate": d * xs.sum(0), "dw_up": d * xs.sum(0),
            "dw_down": h * ys.sum(0)[:, None]}
    for name, result in got.items():
        assert float(value[name].abs().max()) < 65504
        ref.assert_within(result, value[name], bound[name] + more[name] + 2.0 ** -24, name)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_gates_whose_square_is_past_float32(dtype, activation):
    """Gates about 10^20: flat tails, whose slopes are 0 and 1."""
    x, w_gate, w_up, w_down, dy = _inputs(40, 32, 48, dtype)
    _check(x, w_gate * 1e20, w_up, w_down * 1e-20, dy, activation)


def test_leading_dimensions_strides_and_odd_addresses():
    ops = _ops()
    x, w_gate, w_up, w_down, dy = _inputs(60, 32, 48, torch.bfloat16)
    want = ops.gated_ffn(x, w_gate, w_up, w_down)
    assert torch.equal(ops.gated_ffn(x.view(3, 4, 5, 32), w_gate, w_up, w_down), want.view(3, 4, 5, 32))
    cut = torch.zeros(60, 71, device="cuda", dtype=torch.bfloat16)
    cut[:, 5:37] = x
    assert torch.equal(ops.gated_ffn(cut[:, 5:37], w_gate, w_up, w_down), want)
    turned = x.t().contiguous().t()
    assert torch.equal(ops.gated_ffn(turned, w_gate.t().contiguous().t(), w_up, w_down.t().contiguous().t()), want)

    def odd(t):
        return torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)[1:].view(t.shape).copy_(t)

    assert torch.equal(ops.gated_ffn(*(odd(t) for t in (x, w_gate, w_up, w_down))), want)
    _check(odd(x), odd(w_gate), odd(w_up), odd(w_down), odd(dy))
    _check(cut[:, 5:37], w_gate, w_up, w_down, dy.t().contiguous().t())


def test_broadcast_rows_and_gradient():
    ops = _ops()
    x, w_gate, w_up, w_down, _ = _inputs(50, 32, 48, torch.float32)
    leaf = x[:1].detach().requires_grad_()
    y = ops.gated_ffn(leaf.expand(50, 32), w_gate, w_up, w_down)
    (got,) = torch.autograd.grad(y.sum(), [leaf])
    value, bound = ref.ffn(x[:1].expand(50, 32), w_gate, w_up, w_down, "silu", torch.ones(50, 32))
    ref.assert_within(got, value["dx"].sum(0, keepdim=True), (bound["dx"] + 50 * ref.EPS * value["dx"].abs()).sum(0, keepdim=True), "dx")


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (3,), (0, 2), (1, 3)])
def test_some_gradients(wanted):
    x, w_gate, w_up, w_down, dy = _inputs(300, 40, 56, torch.bfloat16)
    every = [t.detach().requires_grad_() for t in (x, w_gate, w_up, w_down)]
    full = torch.autograd.grad(_ops().gated_ffn(*every), every, dy)
    some = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((x, w_gate, w_up, w_down))]
    got = torch.autograd.grad(_ops().gated_ffn(*some), [some[i] for i in wanted], dy)
    for i, g in zip(wanted, got):
        assert torch.equal(g, full[i])


@pytest.mark.parametrize("which", range(4))
def test_forward_mode_tangents_are_refused(which):
    from torch.autograd import forward_ad

    tensors = _inputs(8, 40, 24, torch.float32)[:4]
    with forward_ad.dual_level():
        tensors[which] = forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
        with pytest.raises(ValueError, match="has a forward-mode tangent"):
            _ops().gated_ffn(*tensors)


def test_no_rows():
    x, w_gate, w_up, w_down, dy = _inputs(0, 32, 48, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w_gate, w_up, w_down)]
    y = _ops().gated_ffn(*leaves)
    assert y.shape == (0, 32)
    grads = torch.autograd.grad(y, leaves, dy)
    assert all(bool((g == 0).all()) for g in grads)


def test_a_non_finite_row_stays_its_own():
    ops = _ops()
    x, w_gate, w_up, w_down, _ = _inputs(80, 40, 56, torch.bfloat16)
    want = ops.gated_ffn(x, w_gate, w_up, w_down)
    x[33, 39], x[34, 0] = math.nan, math.inf
    got = ops.gated_ffn(x, w_gate, w_up, w_down)
    rest = [i for i in range(80) if i not in (33, 34)]
    assert torch.equal(got[rest], want[rest])
    assert torch.isnan(got[33]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("N", [1, 16])
def test_inner_values_of_few_rows_past_the_types_range(N, dtype):
    """h of up to 16 rows is not rounded to the elements' type: 90,000 of it meet weights of 0.01."""
    gen = torch.Generator().manual_seed(N)

    def around(middle, off, *shape):
        return (middle + off * torch.randn(*shape, generator=gen)).to(dtype).cuda()

    x, w_gate, w_up, w_down = around(1, 0.1, N, 8), around(37.5, 3.75, 24, 8), around(37.5, 3.75, 24, 8), around(0, 0.01, 8, 24)
    value, bound = ref.ffn(x, w_gate, w_up, w_down, "silu")
    ref.assert_within(_ops().gated_ffn(x, w_gate, w_up, w_down), value["y"], bound["y"], "y")


def test_an_inner_value_between_bfloat16s_and_float32s_largest():
    """gate = 2^64 (1 - 2^-10), up = 2^64 (1 - 2^-11): h is finite in float32 and would be infinite in bfloat16."""
    x, w_down = torch.ones(1, 2), torch.full((2, 1), 2.0 ** -10)
    w_gate, w_up = torch.tensor([[2.0 ** 64, -2.0 ** 54]]), torch.tensor([[2.0 ** 64, -2.0 ** 53]])
    y = _ops().gated_ffn(*(t.bfloat16().cuda() for t in (x, w_gate, w_up, w_down)))
    # 2^118 (1 - 2^-10) (1 - 2^-11), rounded to 8 bits
    assert torch.equal(y.float().cpu(), torch.full((1, 2), 2.0 ** 118))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N,F", [(1, 24), (16, 24), (16, 683), (40, 24), (40, 683), (200, 24), (200, 683), (9000, 681)])
def test_an_infinity_is_no_nan(N, F, dtype):
    """With weights above zero an infinite input makes its row's outputs infinite, and no other's."""
    x, w_gate, w_up, w_down, _ = _inputs(N, 40, F, dtype)
    x[N - 1, 3] = math.inf
    y = _ops().gated_ffn(x, w_gate.abs(), w_up.abs(), w_down.abs())
    assert torch.isposinf(y[N - 1]).all() and torch.isfinite(y[: N - 1]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N,F", [(16, 24), (16, 683), (200, 683), (9000, 681)])
def test_an_infinite_gradient_is_no_nan(N, F, dtype):
    """With weights and rows above zero: infinite gradients of its row and of every weight of both projections."""
    *tensors, dy = _inputs(N, 40, F, dtype)
    dy[N - 1, 3] = math.inf
    leaves = [t.abs().requires_grad_() for t in tensors]
    dx, dg, du, dd = torch.autograd.grad(_ops().gated_ffn(*leaves), leaves, dy)
    assert torch.isposinf(dx[N - 1]).all() and torch.isfinite(dx[: N - 1]).all()
    assert torch.isposinf(dg).all() and torch.isposinf(du).all()
    rest = [i for i in range(40) if i != 3]
    assert torch.isposinf(dd[3]).all() and torch.isfinite(dd[rest]).all()


def test_gradients_against_differences():
    x, w_gate, w_up, w_down, dy = _inputs(20, 24, 40, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w_gate, w_up, w_down)]
    gen = torch.Generator().manual_seed(1)
    for activation in ("silu", "gelu"):
        grads = torch.autograd.grad(_ops().gated_ffn(*leaves, activation=activation), leaves, dy)
        for i, grad in enumerate(grads):
            way = torch.randn(leaves[i].shape, generator=gen).double()

            def loss(step):
                tensors = [ref.wide(t) for t in leaves]
                tensors[i] = tensors[i] + step * way
                act, _ = ref.activation(activation, tensors[0] @ tensors[1].t())
                return ((act * (tensors[0] @ tensors[2].t())) @ tensors[3].t() * ref.wide(dy)).sum()

            along, size = (ref.wide(grad) * way).sum(), (ref.wide(grad) * way).abs().sum()
            # the difference's own error is of the order of step^2 = 1e-8, the gradient's of 2^-17
            assert abs((loss(1e-4) - loss(-1e-4)) / 2e-4 - along) <= 1e-4 * size


def test_rows_past_two_to_the_31():
    """More than 2^31 elements of x and y: the last rows are what they are by themselves."""
    ops = _ops()
    N, D, F = (1 << 21) + 77, 1032, 64
    _, w_gate, w_up, w_down, _ = _inputs(1, D, F, torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(N, D, generator=gen, device="cuda", dtype=torch.bfloat16)
    y = ops.gated_ffn(x, w_gate, w_up, w_down)
    tail = x[-100:].clone()
    value, bound = ref.ffn(tail, w_gate, w_up, w_down, "silu")
    ref.assert_within(y[-100:], value["y"], bound["y"], "y")


def test_more_elements_than_small_tiles_reach():
    """2^33 elements of x and of y, more than 2^22 small tiles of 64 x 32: the last rows are what they are by themselves."""
    N, D, F = 1 << 20, 8192, 16
    _, w_gate, w_up, w_down, _ = _inputs(1, D, F, torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(N, D, generator=gen, device="cuda", dtype=torch.bfloat16)
    y = _ops().gated_ffn(x, w_gate, w_up, w_down)
    value, bound = ref.ffn(x[-100:].clone(), w_gate, w_up, w_down, "silu")
    ref.assert_within(y[-100:], value["y"], bound["y"], "y")


def test_another_stream_and_a_graph():
    x, w_gate, w_up, w_down, dy = _inputs(5000, 64, 105, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w_gate, w_up, w_down)]

    def program():
        y = _ops().gated_ffn(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in program()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = program()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        torch.randn(1000, device="cuda").sum()
