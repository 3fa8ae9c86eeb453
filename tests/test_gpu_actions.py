"""Log-probabilities, entropies, gradients and choices of actions on the GPU
against their definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import ops_reference as ref
import policy_reference as policy

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
CAR = (3, 3, 3, 2, 2, 3, 2)
# both forms, their borders (heads of 32; of 64, 128, 256, 1,024), lanes with nothing, several reads a lane
HEADS = [CAR, (1,), (2,), (1, 1), (32, 32), (31, 33), (32, 31, 1), (33,), (64,), (65,), (90,), (16,) * 5, (127, 2), (128,), (129,),
         (130, 1, 140), (256,), (257, 2), (513,), (1, 1024), (1, 1200, 3), (2100,), (3,) * 21, (2,) * 64]


def _ops():
    from carl_amd import ops

    return ops


def _rows(lead, heads, dtype, seed=0, mask=True, scale=2.0):
    gen = torch.Generator().manual_seed(seed)
    L = sum(heads)
    logits = (torch.randn(*lead, L, generator=gen) * scale).to(dtype)
    there = None
    if mask:
        there = torch.rand(*lead, L, generator=gen) < 0.6
        there[..., [sum(heads[:i]) for i in range(len(heads))]] = True
    actions = torch.stack([torch.randint(0, n, lead, generator=gen) for n in heads], -1)
    if mask:        # actions that can be taken: a head's first where the drawn one cannot
        first = torch.tensor([sum(heads[:i]) for i in range(len(heads))])
        actions = torch.where(there.gather(-1, actions + first), actions, 0)
    return logits.cuda(), actions.int().cuda(), None if there is None else there.cuda()


def _same(got, want, bound, what):
    """Equal infinities and NaN, and the rest within the bound."""
    got = ref.wide(got)
    plain = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~plain & ~torch.isnan(want)], want[~plain & ~torch.isnan(want)]), what
    ref.assert_within(got[plain], want[plain], bound[plain], what)


def _check(logits, actions, heads, mask=None):
    leaf = logits.detach().requires_grad_()
    log_prob, entropy = _ops().action_log_prob(leaf, actions, heads, mask=mask)
    assert log_prob.shape == entropy.shape == logits.shape[:-1] and log_prob.dtype == entropy.dtype == torch.float32
    (want, off), (want_entropy, entropy_off) = policy.log_prob(logits, actions, heads, mask)
    _same(log_prob, want, off, "log-probability")
    _same(entropy, want_entropy, entropy_off, "entropy")
    gen = torch.Generator().manual_seed(9)
    d = [torch.randn(logits.shape[:-1], generator=gen).cuda() for _ in range(2)]
    (grad,) = torch.autograd.grad([log_prob, entropy], [leaf], d)
    assert grad.shape == logits.shape and grad.dtype == logits.dtype
    _same(grad, *policy.log_prob_gradient(logits, actions, heads, *d, mask), "gradient")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_heads(heads, dtype):
    for mask in (False, True):
        logits, actions, there = _rows((37,), heads, dtype, mask=mask)
        _check(logits, actions, heads, there)
        _check(logits, actions.long(), heads, there)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 127, 200, 5000])
def test_rows(rows, dtype):
    for heads in (CAR, (90,), (300, 2)):
        logits, actions, there = _rows((rows,), heads, dtype, seed=rows)
        _check(logits, actions, heads, there)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,heads", [(16_385, (32, 32)), (16_390, (16,) * 5), (17_000, (3,) * 21), (16_400, (2,) * 64), (16_500, (30,) * 7),
                                        (70_001, CAR), (70_000, (20,)), (210_003, CAR), (210_000, (4,) * 5), (70_000, (5,) * 9)], ids=str)
def test_many_rows(rows, heads, dtype):
    """Every number of waves that share rows, and rows of more logits than few rows of that form have."""
    logits, actions, there = _rows((rows,), heads, dtype, seed=rows)
    _check(logits, actions, heads, there)
    noise = torch.randn(logits.shape, generator=torch.Generator().manual_seed(rows)).cuda()
    for k in (1, 2):
        best, log_prob = _ops().top_actions(logits, heads, k, mask=there, noise=noise)
        keys = (logits.float() + noise).masked_fill(~there, -math.inf).cpu()
        first = 0
        for h, n in enumerate(heads):
            order = torch.sort(keys[:, first:first + n], dim=1, descending=True, stable=True)
            want = torch.where(order[0][:, :k] == -math.inf, -1, order[1][:, :k])
            assert torch.equal(best[:, h, :min(k, n)].cpu().long(), want)
            head = policy.Head(logits[:, first:first + n].cpu().double(), there[:, first:first + n].cpu())
            at = want.clamp(min=0)
            _same(log_prob[:, h, :min(k, n)], torch.where(want < 0, policy.NONE, head.logs.gather(1, at)), head.logs_off.gather(1, at), "log-probability")
            first += n


@pytest.mark.parametrize("heads", [CAR, (70, 3), (2,) * 9, (400,)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_what_is_not_available(heads, dtype):
    """Masked places hold NaN, infinities and the type's lowest value; rows and heads with nothing; actions that are none,
    masked or past the last."""
    L, first = sum(heads), [sum(heads[:i]) for i in range(len(heads))]
    logits, actions, there = _rows((24,), heads, dtype)
    there[3], there[4, :heads[0]] = False, False
    there[5], there[5, first] = False, True
    actions[5] = 0
    odd = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min], dtype=dtype, device="cuda")
    logits = torch.where(there, logits, odd[torch.arange(24 * L, device="cuda").view(24, L) % 4])
    actions[6], actions[7, -1], actions[8, 0] = -1, -5, heads[0]
    actions[9, 0], there[9, 0] = 0, False
    actions[10, 0] = 2 ** 31 - 1
    _check(logits, actions, heads, there)
    # the same without a mask: what is not available is -infinity
    _check(logits.masked_fill(~there, -math.inf), actions, heads)
    # the type's lowest value in the mask's place is a logit like others, and weighs nothing beside larger ones
    _check(logits.masked_fill(~there, torch.finfo(dtype).min), actions.clamp(min=0), heads)


def test_large_logits():
    """Differences of more than float32's range, and rows of one value."""
    logits = torch.zeros(4, 6, device="cuda")
    logits[0] = torch.tensor([3e38, -3e38, 0.0, 1.0, 2.0, 3.0])
    logits[1], logits[2] = 1e30, -3e38
    logits[3] = torch.tensor([1e4, -1e4, 88.0, -88.0, 0.0, 1e-30])
    for heads in ((6,), (3, 3), (2, 4)):
        actions = torch.zeros(4, len(heads), dtype=torch.int32, device="cuda")
        leaf = logits.clone().requires_grad_()
        log_prob, entropy = _ops().action_log_prob(leaf, actions, heads)
        (want, off), (want_entropy, entropy_off) = policy.log_prob(logits, actions, heads)
        _same(log_prob, want, off, "log-probability")
        _same(entropy, want_entropy, entropy_off, "entropy")
        (grad,) = torch.autograd.grad(log_prob.sum() + entropy.sum(), [leaf])
        _same(grad, *policy.log_prob_gradient(logits, actions, heads, torch.ones(()), torch.ones(())), "gradient")


@pytest.mark.parametrize("heads", [CAR, (70, 30), (300,)], ids=str)
def test_a_non_finite_logit_makes_its_row_nan(heads):
    logits, actions, _ = _rows((20,), heads, torch.float32, mask=False)
    want = _ops().action_log_prob(logits, actions, heads)
    logits[3, 1], logits[4, 0] = math.nan, math.inf
    logits[5, :heads[0]] = math.nan
    leaf = logits.requires_grad_()
    got = _ops().action_log_prob(leaf, actions, heads)
    rest = [i for i in range(20) if i not in (3, 4, 5)]
    for a, b in zip(got, want):
        assert torch.equal(a[rest], b[rest]) and torch.isnan(a[[3, 4, 5]]).all()
    (grad,) = torch.autograd.grad(got[0].sum() + got[1].sum(), [leaf])
    assert torch.isfinite(grad[rest]).all() and torch.isnan(grad[[3, 4, 5], : heads[0]]).all()
    assert torch.isfinite(grad[[3, 4, 5], heads[0]:]).all()


def test_strides_leading_dimensions_and_broadcasts():
    ops = _ops()
    logits, actions, there = _rows((6, 10), CAR, torch.bfloat16)
    want = ops.action_log_prob(logits, actions, CAR, mask=there)
    L = sum(CAR)

    def same(l, a, m):
        for x, y in zip(ops.action_log_prob(l, a, CAR, mask=m), want):
            assert torch.equal(x, y)

    wide_rows = torch.full((6, 10, L + 4), math.nan, device="cuda", dtype=torch.bfloat16)
    wide_rows[..., 3:L + 3] = logits
    wide_mask = torch.zeros(6, 10, L + 1, device="cuda", dtype=torch.bool)
    wide_mask[..., 1:] = there
    wide_actions = torch.full((6, 10, 9), 77, device="cuda", dtype=torch.int64)
    wide_actions[..., 1:8] = actions
    same(wide_rows[..., 3:L + 3], wide_actions[..., 1:8], wide_mask[..., 1:])
    same(logits.transpose(0, 1).contiguous().transpose(0, 1), actions.transpose(0, 1).contiguous().transpose(0, 1), there)
    same(logits.mT.contiguous().mT, actions.mT.contiguous().mT, there.mT.contiguous().mT)
    one = there[:1, :1].expand_as(there)
    for x, y in zip(ops.action_log_prob(logits, actions * 0, CAR, mask=one), ops.action_log_prob(logits, actions * 0, CAR, mask=one.contiguous())):
        assert torch.equal(x, y)
    for row in (0, 5):       # one row without leading dimensions
        for x, y in zip(ops.action_log_prob(logits[row, 3], actions[row, 3], CAR, mask=there[row, 3]), want):
            assert x.shape == () and torch.equal(x, y[row, 3])
    _check(wide_rows[..., 3:L + 3], wide_actions[..., 1:8], CAR, wide_mask[..., 1:])


def test_gradients_of_one_result_and_of_a_mean():
    logits, actions, there = _rows((50,), CAR, torch.float32)
    zero = torch.zeros(())
    for pick, weights in ((lambda r: r[0].mean(), (torch.tensor(0.02), zero)), (lambda r: r[1].sum(), (zero, torch.ones(()))),
                          (lambda r: r[0].mean() - 0.01 * r[1].mean(), (torch.tensor(0.02), torch.tensor(-0.0002)))):
        leaf = logits.clone().requires_grad_()
        (grad,) = torch.autograd.grad(pick(_ops().action_log_prob(leaf, actions, CAR, mask=there)), [leaf])
        _same(grad, *policy.log_prob_gradient(logits, actions, CAR, *weights, there), "gradient")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads", [CAR, (70, 30), (300, 2)], ids=str)
def test_an_entropys_gradient_has_nothing_to_do_with_the_actions(heads, dtype):
    """An action past its head's last makes log-probabilities NaN, and gradients by them: not those of the entropy alone."""
    logits, actions, there = _rows((70,), heads, dtype)
    wrong = actions.clone()
    wrong[::2, 0], wrong[1::3, -1] = heads[0], 2 ** 31 - 1
    for mask in (None, there):
        leaf = logits.clone().requires_grad_()
        grads = [torch.autograd.grad(_ops().action_log_prob(leaf, a, heads, mask=mask)[1].sum(), [leaf])[0] for a in (wrong, actions)]
        _same(grads[0], *policy.log_prob_gradient(logits, actions * 0, heads, torch.zeros(()), torch.ones(()), mask), "gradient")
        assert torch.equal(*grads)


def test_gradients_against_differences():
    heads, gen = (5, 3, 40), torch.Generator().manual_seed(1)
    logits, actions, there = _rows((8,), heads, torch.float32)
    leaf = logits.clone().requires_grad_()
    a, b = torch.randn(8, generator=gen).double(), torch.randn(8, generator=gen).double()
    results = _ops().action_log_prob(leaf, actions, heads, mask=there)
    (grad,) = torch.autograd.grad(results, [leaf], [a.float().cuda(), b.float().cuda()])
    way = torch.randn(logits.shape, generator=gen).double()

    def loss(step):
        (lp, _), (h, _) = policy.log_prob(ref.wide(logits) + step * way, actions, heads, there)
        return (lp * a.float().double() + h * b.float().double()).sum()

    # the difference's own error is of the order of step^2 = 1e-8, the gradient's of 2^-17
    along, size = (ref.wide(grad) * way).sum(), (ref.wide(grad) * way).abs().sum()
    assert abs((loss(1e-4) - loss(-1e-4)) / 2e-4 - along) <= 1e-4 * size


# ------------------------------------------------------------------- best actions

def _check_top(logits, heads, k, mask=None, noise=None):
    best, log_prob = _ops().top_actions(logits, heads, k, mask=mask, noise=noise)
    want, logs, off = policy.top(logits, heads, k, mask, noise)
    assert best.dtype == torch.int32 and torch.equal(best.cpu(), want)
    assert log_prob.dtype == torch.float32
    _same(log_prob, logs, off, "log-probability")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_best_actions(heads, dtype):
    gen = torch.Generator().manual_seed(3)
    for k in (1, 3):
        logits, _, there = _rows((9,), heads, dtype, seed=k)
        noise = -torch.log(-torch.log(torch.rand(logits.shape, generator=gen))).cuda()
        _check_top(logits, heads, k)
        _check_top(logits, heads, k, there, noise)


@pytest.mark.parametrize("heads", [(7, 5), (70,), (300,)], ids=str)
def test_all_of_a_heads_actions_in_order(heads):
    logits, _, there = _rows((6,), heads, torch.float32)
    there[2], there[3, 1:] = False, False
    _check_top(logits, heads, 64, there)
    _check_top(logits.masked_fill(~there, -math.inf), heads, 10)


@pytest.mark.parametrize("heads", [(513,), (769,), (900, 3), (1025, 2, 800), (5000,), (16_384,)], ids=str)
def test_many_actions_of_long_heads(heads):
    logits, _, there = _rows((5,), heads, torch.bfloat16, mask=True)
    noise = torch.randn(logits.shape, generator=torch.Generator().manual_seed(1)).cuda()
    there[2], there[3, 7:] = False, False           # nothing to take, and fewer than are asked for
    logits[4, ::3] = 1.0                            # many equal ones
    for k in (2, 64):
        _check_top(logits, heads, k, there)
        best, _ = _ops().top_actions(logits, heads, k, mask=there, noise=noise)
        want, _, _ = policy.top(logits, heads, k, there, noise)
        assert torch.equal(best.cpu(), want)


@pytest.mark.parametrize("heads", [(700,), (800,), (1100, 5)], ids=str)
def test_many_rows_of_several_actions(heads):
    """As many as are taken by lanes, and by workgroups: the same as of a few rows."""
    logits, _, there = _rows((2100,), heads, torch.float32)
    best, logs = _ops().top_actions(logits, heads, 6, mask=there)
    few = [_ops().top_actions(logits[i:i + 300], heads, 6, mask=there[i:i + 300]) for i in range(0, 2100, 300)]
    assert torch.equal(best, torch.cat([b for b, _ in few]))
    # sums of a thousand terms in another order, at logarithms of order 10
    assert torch.allclose(logs, torch.cat([v for _, v in few]), rtol=0, atol=1e-4)
    _check_top(logits[:3], heads, 6, there[:3])


@pytest.mark.parametrize("heads", [(8,), (40, 30), (600,), (1200,)], ids=str)
def test_equal_keys_go_by_their_index(heads):
    logits = torch.randint(-1, 2, (12, sum(heads)), generator=torch.Generator().manual_seed(0)).float().cuda()
    logits = torch.where((logits == 0) & (torch.arange(sum(heads), device="cuda") % 2 == 1), -0.0, logits)      # both zeros
    _check_top(logits, heads, 9)
    _check_top(torch.zeros_like(logits), heads, 5)
    # equal sums of unequal logits
    noise = -logits
    _check_top(logits, heads, 5, None, noise)


@pytest.mark.parametrize("heads", [(8,), (70,), (300,), (1030,)], ids=str)
def test_keys_that_are_not_finite(heads):
    """A NaN among the logits goes first and makes the log-probabilities NaN; noise may be infinite or NaN, and counts
    only where an action is available."""
    logits, _, _ = _rows((6,), heads, torch.float32, mask=False)
    logits[0, 5] = math.nan
    logits[1, 0], logits[1, 6] = math.nan, math.inf
    best, log_prob = _ops().top_actions(logits, heads, 2)
    assert best[0, 0, 0] == 5 and best[1, 0].tolist() == [0, 6] and torch.isnan(log_prob[:2]).all()
    assert torch.isfinite(log_prob[2:]).all()
    noise = torch.zeros_like(logits)
    noise[2, 3], noise[3, 2], noise[4] = math.inf, math.nan, -math.inf
    there = torch.ones_like(logits, dtype=torch.bool)
    there[3, 2], noise[3, 4] = False, math.nan
    best, log_prob = _ops().top_actions(logits, heads, 1, mask=there, noise=noise)
    assert best[2:5, 0, 0].tolist() == [3, 4, 0] and torch.isfinite(log_prob[2:]).all()


def test_samples_follow_the_policy():
    """200,000 samples of one row: each count within 5 standard deviations of its expectation."""
    n, heads = 200_000, (4, 70)
    logits, _, there = _rows((1,), heads, torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(0)
    noise = -torch.log(-torch.log(torch.rand(n, sum(heads), generator=gen, device="cuda").clamp(1e-7, 1 - 1e-7)))
    best, log_prob = _ops().top_actions(logits.expand(n, -1), heads, mask=there.expand(n, -1), noise=noise)
    lp, _ = _ops().action_log_prob(logits.expand(n, -1), best.squeeze(-1), heads, mask=there.expand(n, -1))
    assert torch.allclose(lp, log_prob.squeeze(-1).sum(-1), rtol=0, atol=1e-5)
    first = 0
    for i, size in enumerate(heads):
        x = logits[0, first:first + size].double().masked_fill(~there[0, first:first + size], -math.inf)
        p = x.softmax(0)
        count = torch.bincount(best[:, i, 0].long(), minlength=size)
        assert bool(((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1).all())
        first += size


@pytest.mark.parametrize("heads", [CAR, (90,)], ids=str)
def test_no_rows(heads):
    L = sum(heads)
    leaf = torch.zeros(0, 3, L, device="cuda", requires_grad=True)
    actions = torch.zeros(0, 3, len(heads), dtype=torch.int32, device="cuda")
    log_prob, entropy = _ops().action_log_prob(leaf, actions, heads)
    (grad,) = torch.autograd.grad(log_prob.sum() + entropy.sum(), [leaf])
    assert log_prob.shape == (0, 3) and grad.shape == leaf.shape
    best, logs = _ops().top_actions(leaf.detach(), heads, 2)
    assert best.shape == logs.shape == (0, 3, len(heads), 2)


@pytest.mark.parametrize("heads", [(30, 30), (120,)], ids=str)
def test_rows_past_two_to_the_31(heads):
    """More than 2^31 logits: the last rows' results."""
    L = sum(heads)
    N = (1 << 31) // L + 1000
    gen = torch.Generator(device="cuda").manual_seed(0)
    logits = torch.randn(N, L, generator=gen, device="cuda", dtype=torch.bfloat16)
    actions = torch.randint(0, heads[0], (N, len(heads)), generator=gen, device="cuda", dtype=torch.int32)
    leaf = logits.requires_grad_()
    log_prob, entropy = _ops().action_log_prob(leaf, actions, heads)
    (grad,) = torch.autograd.grad(log_prob.sum() + entropy.sum(), [leaf])
    best, logs = _ops().top_actions(logits.detach(), heads)
    tail, taken, one = logits[-70:].detach(), actions[-70:], torch.ones(())
    (want, off), (want_entropy, entropy_off) = policy.log_prob(tail, taken, heads)
    _same(log_prob[-70:], want, off, "log-probability")
    _same(entropy[-70:], want_entropy, entropy_off, "entropy")
    _same(grad[-70:], *policy.log_prob_gradient(tail, taken, heads, one, one), "gradient")
    want, want_logs, off = policy.top(tail, heads, 1)
    assert torch.equal(best[-70:].cpu(), want)
    _same(logs[-70:], want_logs, off, "best log-probability")


def test_another_stream_and_a_graph():
    logits, actions, there = _rows((3000,), CAR, torch.bfloat16)
    wide_logits, wide_actions, _ = _rows((500,), (300, 4), torch.float32, mask=False)
    leaves = [logits.requires_grad_(), wide_logits.requires_grad_()]
    d = torch.randn(3000, device="cuda"), torch.randn(500, device="cuda")

    def program():
        a = _ops().action_log_prob(leaves[0], actions, CAR, mask=there)
        b = _ops().action_log_prob(leaves[1], wide_actions, (300, 4))
        grads = torch.autograd.grad([*a, *b], leaves, [d[0], d[0], d[1], d[1]])
        top = _ops().top_actions(leaves[0].detach(), CAR, 2, mask=there)
        return (*(t.detach() for t in (*a, *b)), *grads, *top)

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
