"""The root-mean-square norm, its gradients and its 8-bit form on the GPU against
their definition: in 64 bits, and rounding for rounding where codes are made."""
from __future__ import annotations

import math

import pytest
import torch

import ops_reference as ref
import policy_reference as policy

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# every number of lanes and pieces a row takes, at its borders in both element sizes
WIDTHS = [1, 2, 7, 8, 9, 16, 31, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 511, 512, 513, 683, 1000, 1024, 1025, 2047, 2048, 2049,
          4095, 4096, 4097, 8191, 8192, 8193, 16383, 16384, 32, 33, 192, 193, 384, 385, 768, 769, 1408, 1536, 1537, 2373, 3100, 5000, 6144, 6145,
          12288, 12289]


def _ops():
    from carl_amd import ops

    return ops


def _rows(N, D, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x, residual, dy, dsum = (torch.randn(N, D, generator=gen).to(dtype).cuda() for _ in range(4))
    weight = (1 + 0.3 * torch.randn(D, generator=gen)).to(dtype).cuda()
    return x, weight, residual, dy, dsum


def _check(x, weight, residual, dy, dsum, eps=1e-6):
    """All results and gradients, with the residual and without."""
    leaves = [t.detach().requires_grad_() for t in (x, weight, residual)]
    y, total = _ops().rms_norm(leaves[0], leaves[1], residual=leaves[2], eps=eps)
    assert y.shape == total.shape == x.shape and y.dtype == total.dtype == x.dtype
    assert torch.equal(total.cpu(), policy.kept_sum(x, residual))
    grads = torch.autograd.grad([y, total], leaves, [dy, dsum])
    value, bound = policy.norm(x, weight, residual, eps, dy, dsum)
    ref.assert_within(y, value["y"], bound["y"], "y")
    assert torch.equal(grads[0], grads[2])
    ref.assert_within(grads[0], value["dx"], bound["dx"], "dx")
    ref.assert_within(grads[1], value["dweight"], bound["dweight"], "dweight")

    leaves = leaves[:2]
    y = _ops().rms_norm(*leaves, eps=eps)
    grads = torch.autograd.grad(y, leaves, dy)
    value, bound = policy.norm(x, weight, None, eps, dy)
    ref.assert_within(y, value["y"], bound["y"], "y alone")
    ref.assert_within(grads[0], value["dx"], bound["dx"], "dx alone")
    ref.assert_within(grads[1], value["dweight"], bound["dweight"], "dweight alone")


def _check_codes(x, weight, residual, eps=1e-6):
    ops = _ops()

    def same(codes, scale, t, r):
        want, step = policy.codes(t)
        rows = codes.reshape(-1, codes.shape[-1])
        assert codes.dtype == torch.int8 and codes.shape == x.shape and (codes.dim() < 2 or codes.stride(-2) % 16 == 0)
        assert torch.equal(rows.cpu(), want)
        step = step.double() * r
        assert torch.equal(torch.isnan(scale).cpu().reshape(-1), torch.isnan(step))
        got = scale.cpu().reshape(-1).double()
        have = ~torch.isnan(step)
        assert bool(((got - step)[have].abs() <= 2 * policy.ROW * step[have]).all())

    w = weight.cpu().float()
    codes, scale, total = ops.rms_norm_int8(x, weight, residual=residual, eps=eps)
    kept = policy.kept_sum(x, residual)
    assert torch.equal(total.cpu(), kept)

    def factor(s):
        return (s.reshape(-1, s.shape[-1]).double().square().mean(1) + eps).rsqrt()

    same(codes, scale, kept.float() * w, factor(kept))
    codes, scale = ops.rms_norm_int8(x, weight, eps=eps)
    same(codes, scale, x.cpu().float() * w, factor(x.cpu()))
    codes, scale = ops.quantize_int8(x)
    same(codes, scale, x.cpu().float(), 1.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(D, dtype):
    tensors = _rows(21, D, dtype, seed=D)
    _check(*tensors)
    _check_codes(*tensors[:3])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 15, 16, 17, 64, 1000, 20_001])
def test_rows(N, dtype):
    for D in (40, 256) if N > 5000 else (40, 256, 700, 5000):
        tensors = _rows(N, D, dtype, seed=N)
        _check(*tensors)
        _check_codes(*tensors[:3])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_more_rows_than_a_launch_takes_at_once(dtype):
    tensors = _rows(70_000, 33, dtype)
    _check(*tensors)
    _check_codes(*tensors[:3])


@pytest.mark.parametrize("dtype,power", [(torch.float32, 60), (torch.float32, 100), (torch.bfloat16, 62), (torch.bfloat16, 120),
                                         (torch.float32, -60), (torch.bfloat16, -100), (torch.float16, 13), (torch.float16, -12)])
@pytest.mark.parametrize("D", [40, 300, 9000])
def test_large_and_small_rows(D, dtype, power):
    """Squares past float32's range, and below it, where eps is all that is left."""
    x, weight, residual, dy, dsum = _rows(12, D, dtype)
    big = [(t.double() * 2.0 ** power).to(dtype) for t in (x, residual)]
    # rows of ordinary size beside them
    big[0][::3], big[1][::3] = x[::3], residual[::3]
    _check(big[0], weight, big[1], dy, dsum)
    # codes do not change with a power of two that is taken out of large rows first
    _check_codes(big[0], weight, big[1])


@pytest.mark.parametrize("eps", [1e-30, 1e-12, 1e-3, 10.0])
def test_eps(eps):
    x, weight, residual, dy, dsum = _rows(30, 100, torch.float32)
    x[3], residual[3] = 0.0, 0.0
    x[4] *= 1e-5
    _check(x, weight, residual, dy, dsum, eps=eps)
    _check_codes(x, weight, residual, eps=eps)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D", [24, 700, 5000])
def test_non_finite_rows_stay_their_own(D, dtype):
    ops = _ops()
    x, weight, _, dy, _ = _rows(40, D, dtype)
    weight[5] = 0.0
    want, (want_codes, want_scale) = ops.rms_norm(x, weight), ops.rms_norm_int8(x, weight)
    x[7, D - 1], x[8, 0], x[9, 5] = math.nan, math.inf, -math.inf
    rest = [i for i in range(40) if i not in (7, 8, 9)]
    leaf, w = x.clone().requires_grad_(), weight.clone().requires_grad_()
    y = ops.rms_norm(leaf, w)
    assert torch.equal(y[rest], want[rest]) and torch.isnan(y[7]).all() and torch.isnan(y[8, 0]) and torch.isnan(y[9, 5])
    dx, dw = torch.autograd.grad(y, [leaf, w], dy)
    assert torch.isfinite(dx[rest]).all() and torch.isnan(dx[7]).all() and torch.isnan(dw).all()
    for codes, scale, kept in (ops.rms_norm_int8(x, weight) + (want_scale,), ops.quantize_int8(x) + (ops.quantize_int8(x[rest])[1],)):
        assert torch.isnan(scale[7:10]).all() and (codes[7:10] == 0).all()
        assert torch.equal(scale[rest], kept if kept.shape[0] == len(rest) else kept[rest])
    codes, _ = ops.rms_norm_int8(x, weight)
    assert torch.equal(codes[rest], want_codes[rest])


def test_rows_of_zeros():
    x = torch.zeros(5, 48, device="cuda", dtype=torch.bfloat16)
    weight = torch.ones(48, device="cuda", dtype=torch.bfloat16)
    assert (_ops().rms_norm(x, weight) == 0).all()
    for codes, scale in (_ops().rms_norm_int8(x, weight), _ops().quantize_int8(x)):
        assert (codes == 0).all() and torch.isfinite(scale).all()
    codes, scale = _ops().rms_norm_int8(x + 1, weight * 0)
    assert (codes == 0).all() and torch.isfinite(scale).all()


def test_leading_dimensions_strides_and_odd_addresses():
    ops = _ops()
    x, weight, residual, dy, dsum = _rows(60, 40, torch.bfloat16)
    y, total = ops.rms_norm(x, weight, residual=residual)
    codes, scale, _ = ops.rms_norm_int8(x, weight, residual=residual)

    def cut(t):
        rows = torch.full((60, 47), math.nan, device="cuda", dtype=t.dtype)
        rows[:, 3:43] = t
        return rows[:, 3:43]

    def odd(t):
        return torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)[1:].view(t.shape).copy_(t)

    def turned(t):
        return t.t().contiguous().t()

    for change in (lambda t: t.view(3, 4, 5, 40), cut, odd, turned):
        a, b = ops.rms_norm(change(x), odd(weight), residual=change(residual))
        assert a.shape == change(x).shape and torch.equal(a.reshape(60, 40), y) and torch.equal(b.reshape(60, 40), total)
        c, s, b = ops.rms_norm_int8(change(x), weight, residual=change(residual))
        assert torch.equal(c.reshape(60, 40), codes) and torch.equal(s.reshape(60), scale) and torch.equal(b.reshape(60, 40), total)
        if change(x).dim() == 2:
            _check(change(x), odd(weight), change(residual), change(dy), change(dsum))
    one = ops.rms_norm(x[0], weight)
    assert one.shape == (40,) and torch.equal(one, ops.rms_norm(x, weight)[0])
    c, s = ops.quantize_int8(x[0])
    assert c.shape == (40,) and s.shape == ()


def test_broadcast_rows_and_gradients():
    x, weight, residual, dy, _ = _rows(50, 72, torch.float32)
    leaf, w = x[:1].detach().requires_grad_(), weight.detach().requires_grad_()
    y, total = _ops().rms_norm(leaf.expand(50, 72), w, residual=residual)
    got = torch.autograd.grad(y.sum(), [leaf, w])
    value, bound = policy.norm(x[:1].expand(50, 72), weight, residual, 1e-6, torch.ones(1))
    ref.assert_within(got[0], value["dx"].sum(0, keepdim=True), (bound["dx"] + 50 * ref.EPS * value["dx"].abs()).sum(0, keepdim=True), "dx")
    ref.assert_within(got[1], value["dweight"], bound["dweight"], "dweight")


def test_some_gradients():
    x, weight, residual, dy, dsum = _rows(300, 72, torch.bfloat16)

    def run(wanted, outputs=(0, 1)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((x, weight, residual))]
        out = _ops().rms_norm(leaves[0], leaves[1], residual=leaves[2])
        return torch.autograd.grad([out[i] for i in outputs], [leaves[i] for i in wanted], [(dy, dsum)[i] for i in outputs], allow_unused=True)

    full = run((0, 1, 2))
    for wanted in ((0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
        for i, g in zip(wanted, run(wanted)):
            assert torch.equal(g, full[i])
    # the sum alone was used: its gradient goes through, the weight has none
    dx, dw, dres = run((0, 1, 2), (1,))
    assert torch.equal(dx, dsum) and torch.equal(dres, dsum) and (dw is None or not dw.any())
    # the norm alone
    value, bound = policy.norm(x, weight, residual, 1e-6, dy)
    dx, dw, dres = run((0, 1, 2), (0,))
    ref.assert_within(dx, value["dx"], bound["dx"], "dx")
    ref.assert_within(dw, value["dweight"], bound["dweight"], "dweight")
    assert torch.equal(dx, dres)


def test_one_tensor_as_input_and_residual():
    x, weight, _, dy, dsum = _rows(300, 72, torch.float32)
    leaf, w = x.detach().requires_grad_(), weight.detach().requires_grad_()
    y, total = _ops().rms_norm(leaf, w, residual=leaf)
    torch.autograd.backward([y, total], [dy, dsum])
    value, bound = policy.norm(x, weight, x, 1e-6, dy, dsum)
    ref.assert_within(leaf.grad, 2 * value["dx"], 2 * bound["dx"], "dx")        # doubling rounds nothing
    ref.assert_within(w.grad, value["dweight"], bound["dweight"], "dweight")


def test_gradients_add_up_over_a_stream():
    """Two norms on one residual stream, as blocks use them, against the chain in 64 bits."""
    x, weight, residual, dy, dsum = _rows(20, 48, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x, residual, weight)]
    y, s = _ops().rms_norm(leaves[0], leaves[2], residual=leaves[1])
    z, t = _ops().rms_norm(y, leaves[2], residual=s)
    (z * dy).sum().add((t * dsum).sum()).backward()
    plain = [v.detach().cpu().double().requires_grad_() for v in (x, residual, weight)]

    def norm(v):
        return v * (v.square().mean(1, keepdim=True) + 1e-6).rsqrt() * plain[2]

    s = plain[0] + plain[1]
    t = norm(s) + s
    ((norm(t) * dy.cpu().double()).sum() + (t * dsum.cpu().double()).sum()).backward()
    for a, b in zip(leaves, plain):
        # a few hundred float32 roundings of values of order 10
        assert torch.allclose(ref.wide(a.grad), b.grad, rtol=0, atol=2e-4)


def test_gradients_against_differences():
    x, weight, residual, dy, dsum = _rows(10, 40, torch.float32)
    leaves = [t.requires_grad_() for t in (x, weight, residual)]
    grads = torch.autograd.grad(_ops().rms_norm(leaves[0], leaves[1], residual=leaves[2]), leaves, [dy, dsum])
    gen = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        way = torch.randn(leaves[i].shape, generator=gen).double()

        def loss(step):
            t = [ref.wide(v) for v in leaves]
            t[i] = t[i] + step * way
            s = t[0] + t[2]
            y = s * (s.square().mean(1, keepdim=True) + 1e-6).rsqrt() * t[1]
            return (y * ref.wide(dy)).sum() + (s * ref.wide(dsum)).sum()

        along, size = (ref.wide(grad) * way).sum(), (ref.wide(grad) * way).abs().sum()
        # the difference's own error is of the order of step^2 = 1e-8, the gradient's of 2^-17
        assert abs((loss(1e-4) - loss(-1e-4)) / 2e-4 - along) <= 1e-4 * size


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_no_rows(dtype):
    x = torch.zeros(0, 32, device="cuda", dtype=dtype, requires_grad=True)
    weight = torch.ones(32, device="cuda", dtype=dtype, requires_grad=True)
    y, total = _ops().rms_norm(x, weight, residual=x)
    assert y.shape == total.shape == (0, 32)
    dx, dw = torch.autograd.grad(y.sum(), [x, weight])
    assert dx.shape == (0, 32) and (dw == 0).all()
    with torch.no_grad():
        codes, scale = _ops().quantize_int8(x)
    assert codes.shape == (0, 32) and scale.shape == (0,)


def test_results_repeat_bit_for_bit():
    x, weight, residual, dy, dsum = _rows(9000, 136, torch.float32)
    leaves = [t.requires_grad_() for t in (x, weight, residual)]
    first = None
    for _ in range(3):
        y, total = _ops().rms_norm(leaves[0], leaves[1], residual=leaves[2])
        now = (y, total, *torch.autograd.grad([y, total], leaves, [dy, dsum]))
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_rows_past_two_to_the_31():
    """More than 2^31 elements: the last rows are what they are by themselves."""
    N, D = (1 << 21) + 77, 1032
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(N, D, generator=gen, device="cuda", dtype=torch.bfloat16)
    weight = torch.ones(D, device="cuda", dtype=torch.bfloat16)
    leaf = x.requires_grad_()
    y, total = _ops().rms_norm(leaf, weight, residual=x.detach())
    (dx,) = torch.autograd.grad(y, [leaf], x.detach())
    with torch.no_grad():
        codes, scale, again = _ops().rms_norm_int8(x, weight, residual=x)
        tail = x[-50:].clone()
        value, bound = policy.norm(tail, weight, tail, 1e-6, tail)
        ref.assert_within(y[-50:], value["y"], bound["y"], "y")
        ref.assert_within(dx[-50:], value["dx"], bound["dx"], "dx")
        want = _ops().rms_norm_int8(tail, weight, residual=tail)
        for a, b in zip((codes, scale, again), want):
            assert torch.equal(a[-50:], b)
        assert torch.equal(total[-50:], want[2])


def test_another_stream_and_a_graph():
    x, weight, residual, dy, dsum = _rows(5000, 136, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, weight, residual)]

    def program():
        y, total = _ops().rms_norm(leaves[0], leaves[1], residual=leaves[2])
        grads = torch.autograd.grad([y, total], leaves, [dy, dsum])
        with torch.no_grad():
            codes = _ops().rms_norm_int8(*leaves[:2], residual=leaves[2])
        return (y.detach(), total.detach(), *grads, *codes)

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
