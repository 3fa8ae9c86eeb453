"""Linear attention on the GPU against the recurrence in 64 bits: outputs,
memories and gradients over lengths, widths, types, head layouts, strides and
masks; the recurrent form; streams and graphs."""
from __future__ import annotations

import itertools
import math

import pytest
import torch

import ops_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ops():
    from carl_amd import ops

    return ops


def _inputs(B, T, H, kv, dk, dv, dtype, *, seed=0, starts=0.1, carry=True, major=False):
    gen = torch.Generator().manual_seed(seed)

    def rows(heads, width):
        x = torch.randn(B, T, heads, width, generator=gen).to(dtype).cuda()
        return x.transpose(0, 1).contiguous().transpose(0, 1) if major else x

    q, k, v, dout = rows(H, dk), rows(kv, dk), rows(kv, dv), rows(H, dv)
    log_decay = torch.log1p(-torch.exp2(-torch.linspace(1.0, 8.0, H))).cuda()
    mask = (torch.rand(B, T, generator=gen) < starts).cuda() if starts is not None else None
    memory, dfinal = ((torch.randn(B, H, dk, dv, generator=gen).cuda() for _ in range(2)) if carry else (None, None))
    return q, k, v, log_decay, mask, memory, dout, dfinal


def _check(q, k, v, log_decay, starts, memory, dout, dfinal, scale=None):
    """Forward and backward against the recurrence, within the bounds."""
    ops = _ops()
    dtype, (B, T, H, dk), dv = q.dtype, q.shape, v.shape[3]
    leaves = [x.detach().requires_grad_() for x in (q, k, v)] + ([] if memory is None else [memory.detach().requires_grad_()])
    out, final = ops.linear_attention(*leaves[:3], log_decay, starts=starts, scale=scale,
                                      initial_state=None if memory is None else leaves[3])
    assert out.shape == (B, T, H, dv) and out.dtype == dtype and final.shape == (B, H, dk, dv)
    want, last = ref.attention(q, k, v, log_decay, starts, memory, scale)
    size, last_size = ref.magnitudes(ref.attention, q, k, v, log_decay, starts, memory, scale)
    ref.assert_within(out, want, ref.attention_bound(dtype, want, size, T, dk), "out")
    ref.assert_within(final, last, ref.memory_bound(last_size, T), "memory")
    pulls = [dout] if dfinal is None else [dout, dfinal]
    grads = torch.autograd.grad([out, final][: len(pulls)], leaves, pulls)
    names = dict(starts=starts, initial=memory, dfinal=dfinal, scale=scale)
    wants = ref.attention_gradients(q, k, v, log_decay, dout, **names)
    sizes = ref.magnitudes(ref.attention_gradients, q, k, v, log_decay, dout, **names)
    group = H // k.shape[2]
    for name, got, value, size, width in zip(("dq", "dk", "dv"), grads, wants, sizes, (dv, dv * group, dk * group)):
        assert got.dtype == dtype
        ref.assert_within(got, value, ref.attention_bound(dtype, value, size, T, width), name)
    if memory is not None:
        ref.assert_within(grads[3], wants[3], ref.memory_bound(sizes[3], T), "dinitial")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("T", [1, 2, 16, 31, 32, 33, 63, 64, 65, 130])
def test_lengths(T, dtype):
    _check(*_inputs(3, T, 2, 2, 32, 32, dtype, seed=T))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dk,dv", [(1, 1), (3, 5), (16, 128), (128, 16), (40, 64), (64, 40), (33, 65), (64, 64), (100, 100),
                                   (128, 128), (65, 32)])
def test_widths(dk, dv, dtype):
    _check(*_inputs(2, 70, 2, 1, dk, dv, dtype, seed=dk * 131 + dv))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("H,kv", [(1, 1), (6, 6), (6, 2), (6, 1), (5, 1)])
@pytest.mark.parametrize("major", [False, True])
def test_head_layouts_and_strides(H, kv, major, dtype):
    _check(*_inputs(2, 40, H, kv, 24, 48, dtype, seed=H * 7 + kv, major=major))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("T,dk,dv", [(257, 32, 64), (700, 64, 64), (1031, 48, 128)])
@pytest.mark.parametrize("starts", [None, 0.004, 0.05])
def test_sequences_split_over_workgroups(T, dk, dv, starts, dtype):
    _check(*_inputs(2, T, 2, 1, dk, dv, dtype, seed=T, starts=starts))


@pytest.mark.parametrize("T", [2248, 2560])       # five segments of 512 steps; of the last one 200, its second half empty
def test_segments_summed_in_halves(T):
    _check(*_inputs(1, T, 32, 4, 72, 66, torch.bfloat16, seed=T, starts=0.002))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("starts,carry", [(None, False), (None, True), (1.0, True), (0.5, False)])
def test_masks_and_memories(starts, carry, dtype):
    _check(*_inputs(3, 75, 2, 2, 32, 48, dtype, seed=5, starts=starts, carry=carry))


@pytest.mark.parametrize("where", ["first", "last", "chunk edge", "before the edge", "all"])
def test_a_start_at(where):
    q, k, v, log_decay, _, memory, dout, dfinal = _inputs(2, 150, 2, 2, 32, 32, torch.float32, starts=None)
    starts = torch.zeros(2, 150, dtype=torch.bool, device="cuda")
    starts[0, {"first": 0, "last": 149, "chunk edge": 64, "before the edge": 63, "all": slice(None)}[where]] = True
    _check(q, k, v, log_decay, starts, memory, dout, dfinal)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_decays_of_one_and_zero(dtype):
    q, k, v, _, starts, memory, dout, dfinal = _inputs(2, 90, 3, 3, 32, 32, dtype)
    _check(q, k, v, torch.tensor([0.0, -math.inf, -1e-6], device="cuda"), starts, memory, dout, dfinal)


def test_scale_is_an_argument():
    q, k, v, log_decay, starts, memory, dout, dfinal = _inputs(2, 70, 2, 2, 32, 32, torch.float32)
    _check(q, k, v, log_decay, starts, memory, dout, dfinal, scale=-1.7)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_at_odd_addresses_and_between_other_data(dtype):
    """One element off alignment, with heads and widths cut out of wider rows."""
    B, T, H, dk, dv = 2, 70, 2, 32, 24
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(B * T * 4 * 101 + 1, generator=gen).to(dtype).cuda()[1:].view(B, T, 4, 101)
    q, k, v = wide[:, :, :H, 1:1 + dk], wide[:, :, 2:, 1:1 + dk], wide[:, :, 2:, 40:40 + dv]
    _, _, _, log_decay, starts, memory, dout, dfinal = _inputs(B, T, H, H, dk, dv, dtype)
    _check(q, k, v, log_decay, starts, memory, dout, dfinal)


def test_broadcast_inputs_get_summed_gradients():
    ops = _ops()
    q, k, v, log_decay, starts, memory, dout, _ = _inputs(3, 40, 4, 4, 32, 32, torch.float32)
    leaf = k[:1, :, :1].detach().requires_grad_()
    out, _ = ops.linear_attention(q, leaf.expand(3, 40, 4, 32), v, log_decay, starts=starts, initial_state=memory)
    (got,) = torch.autograd.grad(out, [leaf], dout)
    full = ref.attention_gradients(q, k[:1, :, :1].expand(3, 40, 4, 32), v, log_decay, dout, starts=starts, initial=memory)
    size = ref.magnitudes(ref.attention_gradients, q, k[:1, :, :1].expand(3, 40, 4, 32), v, log_decay, dout, starts=starts, initial=memory)
    value, size = (x[1].sum((0, 2), keepdim=True) for x in (full, size))
    ref.assert_within(got, value, 16 * ref.EPS * size + ref.attention_bound(torch.float32, value, size, 40, 32), "dk")


@pytest.mark.parametrize("T", [100, 600])
def test_gradients_against_differences(T):
    """Along random directions, from central differences of the 64-bit outputs.  The loss is linear in each tensor by
    itself, so the difference is exact but for its own rounding."""
    ops = _ops()
    q, k, v, log_decay, starts, memory, dout, dfinal = _inputs(1, T, 2, 1, 16, 24, torch.float32, seed=11, starts=0.02)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, memory)]
    out, final = ops.linear_attention(*leaves[:3], log_decay, starts=starts, initial_state=leaves[3])
    grads = torch.autograd.grad([out, final], leaves, [dout, dfinal])
    gen = torch.Generator().manual_seed(1)
    for i, (x, grad) in enumerate(zip(leaves, grads)):
        way = torch.randn(x.shape, generator=gen).double()

        def loss(sign):
            tensors = [ref.wide(t) for t in leaves]
            tensors[i] = tensors[i] + sign * 0.5 * way
            o, f = ref.attention(*tensors[:3], log_decay, starts, tensors[3])
            return (o * ref.wide(dout)).sum() + (f * ref.wide(dfinal)).sum()

        along = (ref.wide(grad) * way).sum()
        size = (ref.wide(grad) * way).abs().sum()
        # each gradient element is good to about 2^-15 of the magnitudes it sums, which are at most 30 times it here
        assert abs(loss(1) - loss(-1) - along) <= 1e-3 * size


# ---------------------------------------------------------------- what is not seen

@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("T", [60, 600])
def test_nothing_of_an_earlier_episode_is_seen(T, bad, dtype):
    """Non-finite values before a start, in the carried memory and at later steps change nothing that does not see them."""
    ops = _ops()
    cut, late = T // 2 + 5, T - 7
    q, k, v, log_decay, _, memory, dout, _ = _inputs(2, T, 2, 2, 32, 48, dtype, starts=None)
    starts = torch.zeros(2, T, dtype=torch.bool, device="cuda")
    starts[0, cut] = True
    starts[1, 0] = True
    clean, _ = ops.linear_attention(q, k, v, log_decay, starts=starts, initial_state=memory)
    k2, v2, q2, memory2 = k.clone(), v.clone(), q.clone(), memory.clone()
    k2[0, cut - 1], v2[0, cut - 9], q2[0, cut - 2], memory2[:] = bad, bad, bad, bad
    v2[0, late], k2[0, late] = bad, bad
    leaves = [x.requires_grad_() for x in (q2, k2, v2)]
    out, final = ops.linear_attention(*leaves, log_decay, starts=starts, initial_state=memory2)
    # careful chunks sum the same products in another order
    size, _ = ref.magnitudes(ref.attention, q, k, v, log_decay, starts, memory)
    for b, steps in ((0, slice(cut, late)), (1, slice(0, T))):
        got, want = out[b, steps], ref.wide(clean)[b, steps]
        ref.assert_within(got, want, 2 * ref.attention_bound(dtype, want, size[b, steps], T, 32), "out")
    assert not torch.isfinite(out[0, late:].float()).all()
    assert torch.isfinite(final[1]).all()
    # gradients of steps that neither see nor are seen by them
    grads = torch.autograd.grad(out, leaves, dout)
    wants = ref.attention_gradients(q, k, v, log_decay, dout, starts=starts, initial=memory)
    sizes = ref.magnitudes(ref.attention_gradients, q, k, v, log_decay, dout, starts=starts, initial=memory)
    for name, got, value, size, width in zip(("dq", "dk", "dv"), grads, wants, sizes, (48, 48, 32)):
        ref.assert_within(got[1], value[1], 2 * ref.attention_bound(dtype, value, size, T, width)[1], name)
    ref.assert_within(grads[0][0, cut:late], wants[0][0, cut:late],
                      2 * ref.attention_bound(dtype, wants[0], sizes[0], T, 48)[0, cut:late], "dq")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("T", [70, 600])
def test_a_decay_that_is_not_a_number(T, dtype):
    """Its head gives NaN wherever a step before is seen, in both forms, and finite values at steps that begin an episode
    (at the ends of chunks and of segments among them); gradients likewise; other heads are as without it."""
    ops = _ops()
    q, k, v, log_decay, _, memory, dout, dfinal = _inputs(2, T, 3, 3, 32, 48, dtype, starts=None)
    starts = torch.zeros(2, T, dtype=torch.bool, device="cuda")
    starts[0, [20, 21, 31, 63, T - 1]] = starts[1, 0] = True
    if T > 256:
        starts[0, 255] = starts[1, 512] = True
    broken = log_decay.clone()
    broken[1] = math.nan
    results = []
    for decays in (log_decay, broken):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, memory)]
        out, final = ops.linear_attention(*leaves[:3], decays, starts=starts, initial_state=leaves[3])
        results.append([out.detach(), final.detach(), *torch.autograd.grad([out, final], leaves, [dout, dfinal])])
    heads = (2, 1, 2, 2, 2, 1)
    for want, got, dim in zip(*results, heads):
        assert torch.equal(want.select(dim, 0), got.select(dim, 0)) and torch.equal(want.select(dim, 2), got.select(dim, 2))
    isnan = [torch.isnan(x.select(dim, 1)) for x, dim in zip(results[1], heads)]
    # forwards all but a start sees a step before; backwards all but the step before a start, and the last, is seen by one after
    before = ~starts
    after = torch.cat((~starts[:, 1:], torch.zeros_like(starts[:, :1])), 1)
    for got, want in zip(isnan, (before, before[:, -1], before, after, after, ~starts[:, 0])):
        assert torch.equal(got.flatten(want.dim()).all(-1), want) and torch.equal(got.flatten(want.dim()).any(-1), want)
    # the recurrent form agrees
    state = memory.clone()
    for t in range(T):
        out = ops.linear_attention_step(q[:, t], k[:, t], v[:, t], broken, state, starts=starts[:, t])
        assert torch.equal(torch.isnan(out[:, 1]), isnan[0][:, t])
    assert torch.equal(torch.isnan(state[:, 1]), isnan[1])


@pytest.mark.parametrize("which", [0, 1, 2, 3, 5])
def test_forward_mode_tangents_are_refused(which):
    from torch.autograd import forward_ad

    ops = _ops()
    args = list(_inputs(2, 5, 2, 2, 16, 24, torch.float32)[:6])
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        q, k, v, log_decay, _, memory = args
        with pytest.raises(ValueError, match="has a forward-mode tangent"):
            ops.linear_attention(q, k, v, log_decay, initial_state=memory)
        with pytest.raises(ValueError, match="has a forward-mode tangent"):
            ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], log_decay, memory)


def test_a_decay_that_is_a_parameter():
    """Without gradients (acting, scoring) it is a tensor like any other; with them its own is missing, and refused."""
    ops = _ops()
    q, k, v, log_decay, starts, memory, _, _ = _inputs(2, 30, 2, 2, 16, 24, torch.float32)
    weight = torch.nn.Parameter(log_decay.clone())
    step = [x[:, 0] for x in (q, k, v)]
    states = [memory.clone() for _ in range(2)]
    with torch.no_grad():
        for a, b in zip(ops.linear_attention(q, k, v, weight, starts=starts), ops.linear_attention(q, k, v, log_decay, starts=starts)):
            assert torch.equal(a, b)
        a, b = (ops.linear_attention_step(*step, w, s) for w, s in zip((weight, log_decay), states))
    assert torch.equal(a, b) and torch.equal(*states)
    with pytest.raises(ValueError, match="log_decay has no gradient"):
        ops.linear_attention(q, k, v, weight)
    with pytest.raises(ValueError, match="log_decay has no gradient"):
        ops.linear_attention_step(*step, weight, states[0])
    # asked for after it was passed, it is no reason to refuse the backward pass
    late = log_decay.clone()
    out, _ = ops.linear_attention(q.requires_grad_(), k, v, late)
    late.requires_grad_()
    out.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dk", [3, 40, 64, 100])
def test_an_infinite_value_is_no_nan(dk, dtype):
    """With queries and keys above zero it makes its column of the memory, and the outputs from it on, infinite: whether
    the keys' width fills a tile or not."""
    q, k, v, log_decay, _, _, _, _ = _inputs(2, 200, 2, 2, dk, 48, dtype, starts=None)
    q, k = q.abs() + 0.125, k.abs() + 0.125
    v[0, 10, 1, 5] = math.inf
    out, final = _ops().linear_attention(q, k, v, torch.full_like(log_decay, -0.01))
    seen = torch.zeros(200, 48, dtype=torch.bool, device="cuda")
    seen[10:, 5] = True
    assert torch.equal(torch.isposinf(out[0, :, 1]), seen) and torch.equal(~torch.isfinite(out[0, :, 1]), seen)
    assert torch.isposinf(final[0, 1, :, 5]).all() and torch.isfinite(out[1]).all() and torch.isfinite(out[0, :, 0]).all()


@pytest.mark.parametrize("T", [100, 600])
def test_a_memory_that_is_not_a_number_is_never_forgotten(T):
    """Without a start its column is NaN to the end, though its weight is zero in float32 after some steps: whether the
    sequence is split or not, and in the gradients of a NaN after the last step."""
    ops = _ops()
    q, k, v, log_decay, _, memory, dout, dfinal = _inputs(2, T, 2, 2, 32, 48, torch.float32, starts=None)
    memory[0, 1, 3, 5], dfinal[0, 1, 3, 5] = math.nan, math.nan
    leaves = [x.requires_grad_() for x in (q, k, v, memory)]
    out, final = ops.linear_attention(*leaves[:3], torch.full_like(log_decay, -2.0), initial_state=leaves[3])
    assert torch.isnan(out[0, :, 1, 5]).all() and torch.isnan(final[0, 1, 3, 5]) and torch.isfinite(out[1]).all()
    dq, dk, dv, first = torch.autograd.grad([out, final], leaves, [dout, dfinal])
    assert torch.isnan(dk[0, :, 1, 3]).all() and torch.isnan(dv[0, :, 1, 5]).all() and torch.isnan(first[0, 1, 3, 5])
    assert torch.isnan(dq[0, :, 1, 3]).all() and all(bool(torch.isfinite(x[1]).all()) for x in (dq, dk, dv, first))


def test_no_steps_and_no_sequences():
    ops = _ops()
    q, k, v, log_decay, starts, memory, dout, dfinal = _inputs(3, 0, 2, 2, 16, 24, torch.float32)
    leaf = memory.clone().requires_grad_()
    out, final = ops.linear_attention(q, k, v, log_decay, starts=starts, initial_state=leaf)
    assert out.shape == (3, 0, 2, 24) and torch.equal(final, memory)
    (back,) = torch.autograd.grad(final, [leaf], dfinal)
    assert torch.equal(back, dfinal)
    assert torch.equal(ops.linear_attention(q, k, v, log_decay)[1], torch.zeros_like(memory))
    out, final = ops.linear_attention(q[:0], k[:0], v[:0], log_decay)
    assert out.shape == (0, 0, 2, 24) and final.shape == (0, 2, 16, 24)


def test_only_the_memory_is_differentiated():
    ops = _ops()
    q, k, v, log_decay, starts, memory, _, dfinal = _inputs(2, 70, 2, 2, 16, 24, torch.float32, starts=0.01)
    leaves = [x.requires_grad_() for x in (q, k, v, memory)]
    _, final = ops.linear_attention(*leaves[:3], log_decay, starts=starts, initial_state=leaves[3])
    grads = torch.autograd.grad(final, leaves, dfinal)
    none = torch.zeros(2, 70, 2, 24)
    wants = ref.attention_gradients(*(x.detach() for x in leaves[:3]), log_decay, none, starts=starts, initial=memory, dfinal=dfinal)
    sizes = ref.magnitudes(ref.attention_gradients, *(x.detach() for x in leaves[:3]), log_decay, none, starts=starts,
                           initial=memory.detach(), dfinal=dfinal)
    for got, want, size in zip(grads, wants, sizes):
        ref.assert_within(got, want, 200 * ref.EPS * size + 1e-30, "gradient")


# ------------------------------------------------------------------ recurrent form

@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,H,kv,dk,dv", [(1, 1, 1, 1, 1), (5, 4, 2, 64, 64), (3, 3, 1, 33, 65), (2, 2, 2, 128, 128), (7, 2, 2, 16, 6)])
def test_steps_follow_the_recurrence(B, H, kv, dk, dv, dtype):
    ops = _ops()
    q, k, v, log_decay, starts, memory, _, _ = _inputs(B, 5, H, kv, dk, dv, dtype, starts=0.2)
    want, last = ref.attention(q, k, v, log_decay, starts, memory)
    size, last_size = ref.magnitudes(ref.attention, q, k, v, log_decay, starts, memory)
    state = memory.clone()
    for t in range(5):
        out = ops.linear_attention_step(q[:, t], k[:, t], v[:, t], log_decay, state, starts=starts[:, t])
        bound = ref.UNIT[dtype] * want[:, t].abs() + (dk + 64) * ref.EPS * size[:, t] + ref.TINY[dtype]
        ref.assert_within(out, want[:, t], bound, "out")
    ref.assert_within(state, last, ref.memory_bound(last_size, 5), "memory")


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_step_that_starts_forgets(bad):
    ops = _ops()
    q, k, v, log_decay, _, memory, _, _ = _inputs(2, 1, 2, 2, 40, 48, torch.float32, starts=None)
    q, k, v = q[:, 0], k[:, 0], v[:, 0]
    state, other = torch.full_like(memory, bad), torch.zeros_like(memory)
    starts = torch.tensor([True, False], device="cuda")
    out = ops.linear_attention_step(q, k, v, log_decay, state, starts=starts)
    fresh = ops.linear_attention_step(q, k, v, log_decay, other)
    assert torch.equal(out[0], fresh[0]) and torch.equal(state[0], other[0])
    assert not torch.isfinite(out[1]).any()


def test_an_inference_state_is_refused_before_it_is_changed():
    """As torch's own changes in place are: outside inference mode, with the memory as it was."""
    ops = _ops()
    q, k, v, log_decay, _, memory, _, _ = _inputs(2, 1, 2, 2, 40, 48, torch.float32)
    q, k, v = q[:, 0], k[:, 0], v[:, 0]
    with torch.inference_mode():
        state = memory.clone()
    with pytest.raises(RuntimeError, match="inference tensor"):
        ops.linear_attention_step(q, k, v, log_decay, state)
    assert torch.equal(state, memory)
    with torch.inference_mode():
        ops.linear_attention_step(q, k, v, log_decay, state)
    assert not torch.equal(state, memory)


def test_a_state_at_an_odd_address():
    ops = _ops()
    q, k, v, log_decay, starts, memory, _, _ = _inputs(3, 1, 2, 2, 16, 32, torch.float32)
    args = [x[:, 0] for x in (q, k, v)]
    odd = torch.empty(memory.numel() + 1, device="cuda")[1:].view(memory.shape).copy_(memory)
    even = memory.clone()
    a = ops.linear_attention_step(*args, log_decay, odd, starts=starts[:, 0])
    b = ops.linear_attention_step(*args, log_decay, even, starts=starts[:, 0])
    assert torch.equal(a, b) and torch.equal(odd, even)


# ------------------------------------------------------------------ sizes past 32 bits

def test_rows_past_two_to_the_31():
    """The end of a sequence whose rows hold more than 2^31 elements is what its last episode gives by itself."""
    ops = _ops()
    T, tail, D = (1 << 24) + 300, 200, 128
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(1, T, 1, D, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    log_decay = torch.tensor([-0.01], device="cuda")
    starts = torch.zeros(1, T, dtype=torch.bool, device="cuda")
    starts[0, T - tail] = True
    out, final = ops.linear_attention(q, k, v, log_decay, starts=starts)
    ends = [x[:, T - tail:].clone() for x in (q, k, v)]
    want, last = ops.linear_attention(*ends, log_decay)
    size, last_size = ref.magnitudes(ref.attention, *ends, log_decay)
    ref.assert_within(out[:, T - tail:], ref.wide(want), 2 * ref.attention_bound(torch.bfloat16, ref.wide(want), size, tail, D), "out")
    ref.assert_within(final, ref.wide(last), 2 * ref.memory_bound(last_size, tail), "memory")


@pytest.mark.parametrize("backwards", [False, True])
@pytest.mark.parametrize("apart", [1 << 25, (1 << 26) + 8])
def test_steps_far_apart(apart, backwards):
    """Steps whose rows lie up to 4 GiB (the last that 32 bits reach) and 8 GiB apart over a chunk."""
    T, D = 70, 32
    gen = torch.Generator().manual_seed(0)
    rows = [torch.randn(1, T, 1, D, generator=gen).bfloat16().cuda() for _ in range(4)]
    q, k, v, dout = rows
    far = torch.empty((T - 1) * apart + D, device="cuda", dtype=torch.bfloat16).as_strided((1, T, 1, D), (1, apart, 1, 1)).copy_(q if backwards else k)
    log_decay = torch.tensor([-0.05], device="cuda")
    if backwards:
        _check(far, k, v, log_decay, None, None, dout, None)
    else:
        _check(q, far, v, log_decay, None, None, dout, None)


def test_one_row_for_every_step():
    """Keys expanded over time: rows past a short chunk's end are not that row again."""
    q, k, v, log_decay, starts, memory, dout, dfinal = _inputs(2, 90, 2, 2, 32, 32, torch.bfloat16)
    _check(q, k[:, :1].expand(2, 90, 2, 32), v, log_decay, starts, memory, dout, dfinal)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shared", [False, True])
def test_windows_that_slide_over_one_row(shared, dtype):
    """Rows one element apart (and heads that are the same rows): the inputs overlap themselves, their gradients do not."""
    B, T, H, D = 2, 31, 2 if shared else 1, 64
    gen = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(B, T + D - 1, generator=gen).to(dtype).cuda().unfold(1, D, 1)[:, :, None].expand(B, T, H, D) for _ in range(3))
    assert q.stride(1) == q.stride(3) == 1
    _, _, _, log_decay, starts, memory, dout, dfinal = _inputs(B, T, H, H, D, D, dtype)
    _check(q, k, v, log_decay, starts, memory, dout, dfinal)


def test_float16_weights_past_its_range():
    """q . k of 80,000 meets values of 0.01: the outputs and gradients are within float16's range."""
    q, k, v, log_decay, starts, memory, dout, dfinal = _inputs(2, 40, 2, 1, 64, 48, torch.float16)
    _check((100 + 0.1 * q).half(), (100 + 0.1 * k).half(), v * 0.01, log_decay, starts, memory * 0.01, dout * 0.001, dfinal * 0.01)


@pytest.mark.parametrize("T", [30, 600])
def test_float16_weights_below_its_range(T):
    """Weights about 2^-20, whose roundings in float16 would be a few hundredths of them: outputs and the queries'
    gradients (weights from small gradients of the outputs) are off by their own rounding and float32 sums alone."""
    q, k, v, log_decay, starts, _, dout, _ = _inputs(2, T, 2, 1, 64, 48, torch.float16)
    q, k, v = q * 2.0 ** -10, k * 2.0 ** -10, v * 32
    out, _ = _ops().linear_attention(q, k, v, log_decay, starts=starts)
    want, _ = ref.attention(q, k, v, log_decay, starts)
    size, _ = ref.magnitudes(ref.attention, q, k, v, log_decay, starts)

    def bound(value, size):
        return 2.0 ** -11 * value.abs() + (T + 64 + 64) * ref.EPS * size + 2.0 ** -24

    ref.assert_within(out, want, bound(want, size), "out")
    leaf, k, v, dout = q.requires_grad_(), k * 2.0 ** 15, v * 2.0 ** -11, dout * 2.0 ** -14
    out, _ = _ops().linear_attention(leaf, k, v, log_decay, starts=starts)
    (got,) = torch.autograd.grad(out, [leaf], dout)
    args = (leaf.detach(), k, v, log_decay, dout, starts)
    want, size = ref.attention_gradients(*args)[0], ref.magnitudes(ref.attention_gradients, *args)[0]
    ref.assert_within(got, want, bound(want, size), "dq")


# ------------------------------------------------------------------ streams and graphs

def test_another_stream_and_a_graph():
    """Captured forward, backward and step: every replay gives the eager results, with other work between replays."""
    ops = _ops()
    q, k, v, log_decay, starts, memory, dout, _ = _inputs(2, 600, 2, 1, 32, 64, torch.bfloat16)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    state = memory.clone()

    def program():
        out, final = ops.linear_attention(*leaves, log_decay, starts=starts, initial_state=memory)
        grads = torch.autograd.grad(out, leaves, dout)
        act = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], log_decay, state)
        return (out.detach(), final.detach(), *grads, act)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [x.clone() for x in program()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    state.copy_(memory)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = program()
    for seed in range(3):
        state.copy_(memory)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        torch.randn(1000, device="cuda").sum()


def test_results_repeat():
    args = _inputs(6, 700, 4, 2, 64, 64, torch.bfloat16)
    first, second = (_run_all(*args) for _ in range(2))
    for a, b in itertools.zip_longest(first, second):
        assert torch.equal(a, b)


def _run_all(q, k, v, log_decay, starts, memory, dout, dfinal):
    leaves = [x.detach().requires_grad_() for x in (q, k, v, memory)]
    out, final = _ops().linear_attention(*leaves[:3], log_decay, starts=starts, initial_state=leaves[3])
    return [out.detach(), final.detach(), *torch.autograd.grad([out, final], leaves, [dout, dfinal])]
