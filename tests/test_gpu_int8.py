"""Products in 8 bits on the GPU: sums are whole numbers and what follows is one
float32 operation a step, so results are compared for equality (the gated form,
which takes an exponential, within a bound)."""
from __future__ import annotations

import math

import pytest
import torch

import ops_reference as ref
import policy_reference as policy

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [(3767, 21), (1, 1), (1, 300), (300, 1), (7, 13), (15, 16), (16, 15), (17, 33), (63, 64), (64, 65), (65, 129), (127, 100), (128, 128), (129, 257),
         (256, 683), (683, 256), (1000, 70), (2049, 40)]


def _ops():
    from carl_amd import ops

    return ops


def _codes(rows, width, gen, padded=True):
    """All int8 values, -128 among them; in rows that begin every 16 bytes, the padding filled with other codes."""
    x = torch.randint(-128, 128, (rows, -(-width // 16) * 16), generator=gen, dtype=torch.int8).cuda()[:, :width]
    return x if padded else x.contiguous()


def _inputs(N, D, F, dtype, seed=0, padded=True):
    gen = torch.Generator().manual_seed(seed)
    x, w, up = _codes(N, D, gen, padded), _codes(F, D, gen, padded), _codes(F, D, gen, padded)
    # results of order 1, of float16's too
    x_scale, w_scale, up_scale = ((0.5 + torch.rand(n, generator=gen)).cuda() * c for n, c in ((N, 0.01), (F, D ** -0.5 / 50), (F, D ** -0.5 / 50)))
    return x, x_scale, w, w_scale, up, up_scale, torch.randn(F, generator=gen).to(dtype).cuda()


def _check(x, x_scale, w, w_scale, up, up_scale, bias, gated=True):
    dtype = bias.dtype
    for b in (None, bias):
        y = _ops().int8_linear(x, x_scale, w, w_scale, bias=b, dtype=dtype)
        assert y.shape == (*x.shape[:-1], w.shape[0]) and y.dtype == dtype
        assert torch.equal(y.cpu(), policy.product(x, x_scale, w, w_scale, b).to(dtype))
    for name in ("silu", "gelu") if gated else ():
        y = _ops().int8_gated_linear(x, x_scale, w, w_scale, up, up_scale, activation=name, dtype=dtype)
        ref.assert_within(y, *policy.gated(x, x_scale, w, w_scale, up, up_scale, name, dtype), name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N", [1, 2, 16, 17, 32, 33, 64, 65, 128, 129, 200, 257, 1000])
def test_rows(N, dtype):
    _check(*_inputs(N, 80, 136, dtype, seed=N))


@pytest.mark.parametrize("padded", [True, False])
@pytest.mark.parametrize("N", [20, 150])
@pytest.mark.parametrize("D,F", SIZES)
def test_widths(D, F, N, padded):
    _check(*_inputs(N, D, F, torch.bfloat16, seed=D * 1000 + F, padded=padded))


@pytest.mark.parametrize("padded", [True, False])
@pytest.mark.parametrize("N,D,F", [(4100, 100, 96), (5003, 136, 264), (9000, 257, 320), (20_000, 64, 512), (70_000, 33, 129), (300, 512, 3000)])
def test_many_tiles(N, D, F, padded):
    """Sizes on both sides of each rule that chooses tiles."""
    for dtype in (torch.float32, torch.bfloat16):
        _check(*_inputs(N, D, F, dtype, seed=N, padded=padded))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D", [16, 70, 128, 129, 200, 257, 400])
def test_large_tiles(D, dtype):
    """One to four stages of the largest tiles, whole ones and parts of them, one and two of them a workgroup."""
    for N in (27_001, 65_000):
        _check(*_inputs(N, D, 500, dtype, seed=D), gated=False)
    for N in (14_001, 32_600):
        x, x_scale, w, w_scale, up, up_scale, _ = _inputs(N, D, 500, dtype, seed=D)
        y = _ops().int8_gated_linear(x, x_scale, w, w_scale, up, up_scale, dtype=dtype)
        ref.assert_within(y, *policy.gated(x, x_scale, w, w_scale, up, up_scale, "silu", dtype), "silu")


@pytest.mark.parametrize("padded", [True, False])
@pytest.mark.parametrize("F", [1, 7, 18, 40, 100])
def test_many_rows_and_few_columns(F, padded):
    """Fewer columns than a tile of any size has, of rows that fill the GPU with the largest ones once and twice, or whose
    number makes them smaller: a policy's projections to its action heads and to a value."""
    for N, dtype in ((65_000, torch.bfloat16), (130_001, torch.float32), (80_003, torch.float16)):
        _check(*_inputs(N, 72, F, dtype, seed=F, padded=padded), gated=F in (1, 18))


@pytest.mark.parametrize("N,D,F,gated", [(1000, 60, 1000, True), (3000, 150, 700, True), (2000, 300, 1500, False), (700, 129, 500, False),
                                         (130, 40, 2100, True), (130, 40, 2100, False)])
def test_other_tiles(N, D, F, gated):
    for dtype in DTYPES:
        _check(*_inputs(N, D, F, dtype, seed=N), gated=gated)


@pytest.mark.parametrize("value", [-128, 127])
def test_the_largest_sums(value):
    """65,536 products of -128 by -128 add up to 2^30."""
    for N in (3, 200, 2000):
        x = torch.full((N, 65536), value, dtype=torch.int8, device="cuda")
        w = torch.full((20, 65536), value, dtype=torch.int8, device="cuda")
        w[3] = 127
        one = [torch.ones(n, device="cuda") for n in (N, 20)]
        y = _ops().int8_linear(x, one[0], w, one[1], dtype=torch.float32)
        want = torch.full((N, 20), float(value * value * 65536))
        want[:, 3] = float(value * 127 * 65536)
        assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("N", [40, 300])
def test_strides_leading_dimensions_and_odd_addresses(N):
    ops = _ops()
    x, x_scale, w, w_scale, up, up_scale, bias = _inputs(N, 96, 72, torch.bfloat16)
    want = ops.int8_linear(x, x_scale, w, w_scale, bias=bias)
    gated = ops.int8_gated_linear(x, x_scale, w, w_scale, up, up_scale)

    def cut(t):
        rows = torch.randint(-128, 128, (t.shape[0], t.shape[1] + 37), dtype=torch.int8, device="cuda")
        rows[:, 5:5 + t.shape[1]] = t
        return rows[:, 5:5 + t.shape[1]]

    def far(t):
        rows = torch.zeros(t.shape[0], t.shape[1] + 64, dtype=torch.int8, device="cuda")
        rows[:, 16:16 + t.shape[1]] = t
        return rows[:, 16:16 + t.shape[1]]

    def turned(t):
        return t.t().contiguous().t()

    for a in (lambda t: t, cut, far, turned):
        for b in (lambda t: t, cut, far, turned):
            assert torch.equal(ops.int8_linear(a(x), x_scale, b(w), w_scale, bias=bias), want)
            assert torch.equal(ops.int8_gated_linear(a(x), x_scale, w, w_scale, b(up), up_scale), gated)
    y = ops.int8_linear(x.view(2, N // 20, 10, 96), x_scale.view(2, N // 20, 10), w, w_scale, bias=bias)
    assert y.shape == (2, N // 20, 10, 72) and torch.equal(y.view(N, 72), want)
    doubled = torch.stack([x_scale, x_scale], 1)[:, 0]
    assert torch.equal(ops.int8_linear(x, doubled, w, torch.stack([w_scale] * 3, 1)[:, 1], bias=torch.stack([bias] * 2, 1)[:, 0]), want)
    # one row for all of them, and one weight for all columns
    same = ops.int8_linear(x[:1].expand(N, 96), x_scale, w[:1].expand(72, 96), w_scale, dtype=torch.float32)
    assert torch.equal(same.cpu(), policy.product(x[:1].expand(N, 96), x_scale, w[:1].expand(72, 96), w_scale))
    assert ops.int8_linear(x[0], x_scale[0], w, w_scale, bias=bias).shape == (72,)


@pytest.mark.parametrize("N", [40, 300])
def test_scales_that_are_not_finite_stay_their_own(N):
    x, x_scale, w, w_scale, up, up_scale, bias = _inputs(N, 48, 40, torch.float32)
    want = _ops().int8_linear(x, x_scale, w, w_scale, bias=bias, dtype=torch.float32)
    x_scale[3], w_scale[7] = math.nan, math.inf
    y = _ops().int8_linear(x, x_scale, w, w_scale, bias=bias, dtype=torch.float32)
    rest = [i for i in range(N) if i != 3]
    columns = [i for i in range(40) if i != 7]
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[:, 7]).any()
    assert torch.equal(y[rest][:, columns], want[rest][:, columns])


def test_gates_far_into_both_tails():
    x, x_scale, w, w_scale, up, up_scale, _ = _inputs(150, 48, 40, torch.float32)
    for name in ("silu", "gelu"):
        for factor in (30.0, 1e6, 1e20):
            y = _ops().int8_gated_linear(x, x_scale, w, w_scale * factor, up, up_scale, activation=name, dtype=torch.float32)
            ref.assert_within(y, *policy.gated(x, x_scale, w, w_scale * factor, up, up_scale, name, torch.float32), name)


@pytest.mark.parametrize("N", [60, 2500])
def test_gates_of_values_whose_product_float32_does_not_hold(N):
    x, x_scale, w, w_scale, up, up_scale, _ = _inputs(N, 48, 400, torch.float32)
    g, u = policy.product(x, x_scale, w, w_scale * 1e22), policy.product(x, x_scale, up, up_scale * 1e22)
    for name in ("silu", "gelu"):
        y = _ops().int8_gated_linear(x, x_scale, w, w_scale * 1e22, up, up_scale * 1e22, activation=name, dtype=torch.float32).cpu()
        assert not torch.isnan(y).any()
        assert (y[g < 0] == 0).all() and (y[(g > 1e20) & (u > 1e20)] == math.inf).all()


@pytest.mark.parametrize("N,F,padded", [(20, 40, True), (150, 3000, True), (2500, 400, True), (2500, 400, False), (14_001, 500, True)])
def test_gates_at_the_end_of_float32(N, F, padded):
    """Gates near float32's largest number, whose product with log2(e) it does not hold, in every form of the product."""
    x, w, up = (_codes(n, 40, torch.Generator().manual_seed(0), padded).zero_() for n in (N, F, F))
    x[:, 3], w[::2, 3], w[1::2, 3], up[:, 3] = 1, 1, -1, 1
    for value in (0.5, 2.0 ** -30):
        scales = [torch.full((n,), c, device="cuda") for n, c in ((N, 1.0), (F, 3e38), (F, value))]
        for name in ("silu", "gelu"):
            y = _ops().int8_gated_linear(x, scales[0], w, scales[1], up, scales[2], activation=name, dtype=torch.float32).cpu()
            # a gate's act is the gate itself, or 0; the reciprocal is good to a unit in the last place, products to half of one
            assert ((y[:, ::2] / value - 3e38).abs() <= 4 * 2.0 ** -24 * 3e38).all() and (y[:, 1::2] == 0).all()


@pytest.mark.parametrize("N,D,F,gated", [(400, 64, 20_000, False), (250, 200, 9001, False), (300, 130, 9000, True), (2300, 64, 3000, False),
                                         (140, 20, 65_536, True), (3, 20, 65_536, True), (16, 300, 17_000, False), (17, 100, 17_000, True),
                                         (32, 77, 9000, False), (33, 77, 9000, True), (64, 64, 9000, False), (90, 140, 5000, True)])
def test_more_columns_than_rows(N, D, F, gated):
    for padded in (True, False):
        _check(*_inputs(N, D, F, torch.bfloat16, seed=F, padded=padded), gated=gated)


def test_no_rows():
    x, w = torch.zeros(0, 3, 32, dtype=torch.int8, device="cuda"), torch.zeros(8, 32, dtype=torch.int8, device="cuda")
    assert _ops().int8_linear(x, torch.ones(0, 3, device="cuda"), w, torch.ones(8, device="cuda")).shape == (0, 3, 8)


def test_results_past_two_to_the_31():
    """More than 2^31 codes and results: the last rows are what they are by themselves."""
    N, D, F = (1 << 21) + 333, 1040, 1030
    x = torch.randint(-128, 128, (N, D), dtype=torch.int8, device="cuda")
    w = torch.randint(-128, 128, (F, D), dtype=torch.int8, device="cuda")
    x_scale, w_scale = torch.rand(N, device="cuda"), torch.rand(F, device="cuda") * 1e-4
    y = _ops().int8_linear(x, x_scale, w, w_scale)
    assert torch.equal(y[-400:].cpu(), policy.product(x[-400:], x_scale[-400:], w, w_scale).bfloat16())


def test_a_block_acting_in_8_bits():
    """The operators as a policy that acts uses them: norm, projections, gate and down projection, from weights put into
    8 bits once; against the same block in 64 bits on the values that the codes stand for."""
    ops = _ops()
    gen = torch.Generator().manual_seed(5)
    N, D, F = 200, 72, 136

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen) * scale).bfloat16().cuda()

    x, stream, weight = randn(N, D), randn(N, D, scale=2.0), randn(D, scale=0.2) + 1
    gate, up, down = (ops.quantize_int8(randn(a, b, scale=b ** -0.5)) for a, b in ((F, D), (F, D), (D, F)))
    codes, scale, stream = ops.rms_norm_int8(x, weight, residual=stream)
    inner = ops.int8_gated_linear(codes, scale, *gate, *up)
    inner_codes, inner_scale = ops.quantize_int8(inner)
    y = ops.int8_linear(inner_codes, inner_scale, *down)

    def value(codes, scale):
        return ref.wide(codes) * ref.wide(scale)[:, None]

    s = ref.wide(stream)
    normed = s * (s.square().mean(1, keepdim=True) + 1e-6).rsqrt() * ref.wide(weight)
    step = ref.wide(scale)[:, None]
    assert bool(((value(codes, scale) - normed).abs() <= 0.501 * step).all())       # half a code, and float32's roundings
    want, bound = policy.gated(codes, scale, *gate, *up, "silu", torch.bfloat16)
    ref.assert_within(inner, want, bound, "inner")
    assert bool(((value(inner_codes, inner_scale) - ref.wide(inner)).abs() <= 0.501 * ref.wide(inner_scale)[:, None]).all())
    assert torch.equal(y.cpu(), policy.product(inner_codes, inner_scale, *down).bfloat16())


def test_another_stream_and_a_graph():
    x, x_scale, w, w_scale, up, up_scale, bias = _inputs(3000, 96, 200, torch.bfloat16)

    def program():
        return (_ops().int8_linear(x, x_scale, w, w_scale, bias=bias), _ops().int8_gated_linear(x, x_scale, w, w_scale, up, up_scale),
                _ops().int8_linear(x[:40], x_scale[:40], w, w_scale))

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
