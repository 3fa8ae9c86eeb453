"""AdamW on the GPU against its formulas restated in float32, bit for bit: sizes, types, alignments, 8-bit moments,
values that are not finite, the optimizer."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import ops_reference as ref

pytestmark = pytest.mark.gpu

HYPER = {"lr": 3e-3, "betas": (0.9, 0.99), "eps": 1e-8, "weight_decay": 0.1}


def _optim():
    from carl_amd import optim

    return optim


def _host(x):
    return x.detach().cpu().float().numpy().reshape(-1)


def _tensors(sizes, dtype, grad_dtype, bits, seed=0, offset=0):
    """Lists on the GPU; `offset` elements off an aligned address."""
    gen = torch.Generator().manual_seed(seed)

    def place(x):
        return torch.empty(x.numel() + offset, dtype=x.dtype, device="cuda")[offset:].copy_(x)

    lists = {n: [] for n in ("params", "grads", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
    for i, n in enumerate(sizes):
        size = 10.0 ** (-(i % 4))
        m, v = torch.randn(n, generator=gen) * size, torch.randn(n, generator=gen).square() * size * size
        v[torch.rand(n, generator=gen) < 0.05] = 0
        lists["params"].append(place(torch.randn(n, generator=gen).to(dtype)))
        lists["grads"].append(place((torch.randn(n, generator=gen) * size).to(grad_dtype)))
        if bits == 8:
            for name, x, second in (("exp_avg", m, False), ("exp_avg_sq", v, True)):
                code, scale = ref.encode(x.numpy(), second)
                lists[name].append(place(torch.from_numpy(code)))
                lists[name + "_scale"].append(place(torch.from_numpy(scale)))
        else:
            lists["exp_avg"].append(place(m))
            lists["exp_avg_sq"].append(place(v))
    return lists


def _check(lists, bits, step=7, grad_scale=None, hyper=HYPER):
    before = {n: [_host(x) if x.dtype in (torch.bfloat16, torch.float16) else x.cpu().numpy().reshape(-1).copy() for x in xs]
              for n, xs in lists.items()}
    scales = {n: lists[n] for n in ("exp_avg_scale", "exp_avg_sq_scale")} if bits == 8 else {}
    factor = None if grad_scale is None else torch.tensor([grad_scale], device="cuda")
    _optim().adamw_step(lists["params"], lists["grads"], lists["exp_avg"], lists["exp_avg_sq"], step=step, grad_scale=factor,
                        **hyper, **scales)
    for i, p in enumerate(lists["params"]):
        m, v = before["exp_avg"][i], before["exp_avg_sq"][i]
        if bits == 8:
            m = ref.decode(m, before["exp_avg_scale"][i], False)
            v = ref.decode(v, before["exp_avg_sq_scale"][i], True)
        want_p, want_m, want_v = ref.adamw(before["params"][i], before["grads"][i], m, v, step, grad_scale=grad_scale, **hyper)
        want_p = torch.from_numpy(np.ascontiguousarray(want_p)).to(p.dtype).float().numpy()
        np.testing.assert_array_equal(_host(p), want_p)
        np.testing.assert_array_equal(_host(lists["grads"][i]), before["grads"][i])
        for name, want, second in (("exp_avg", want_m, False), ("exp_avg_sq", want_v, True)):
            got = lists[name][i].cpu().numpy().reshape(-1)
            if bits == 32:
                np.testing.assert_array_equal(got, want)
                continue
            code, scale = ref.encode(want, second)
            got_scale = lists[name + "_scale"][i].cpu().numpy()
            np.testing.assert_array_equal(got_scale, scale)
            whole = np.repeat(np.isfinite(scale), ref.BLOCK)[: len(code)]
            np.testing.assert_array_equal(got[whole], code[whole])


SIZES = [1, 3, 4, 255, 256, 257, 1000, 1024, 4096, 4097, 70001]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_sizes_and_addresses(offset, bits):
    _check(_tensors(SIZES, torch.float32, torch.float32, bits, offset=offset), bits)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_types(dtype, grad_dtype, bits):
    _check(_tensors([5, 512, 3001], dtype, grad_dtype, bits, seed=1), bits)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("count", [1, 59, 60, 61, 121, 300])
def test_more_tensors_than_a_launch_holds(count, bits):
    _check(_tensors([17 * (i % 40) + 1 for i in range(count)], torch.float32, torch.float32, bits, seed=2), bits)


@pytest.mark.parametrize("bits", [8, 32])
def test_many_elements(bits):
    """Past the size from which a wave takes four blocks."""
    _check(_tensors([3_000_001, 70_000, 1_500_000, 257], torch.float32, torch.bfloat16, bits, seed=3), bits)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("step", [1, 2, 1000, 10 ** 7])
def test_step_counts(step, bits):
    _check(_tensors([1000], torch.float32, torch.float32, bits), bits, step=step)


@pytest.mark.parametrize("hyper", [{"lr": 0.0}, {"eps": 0.0}, {"weight_decay": 0.0}, {"betas": (0.0, 0.0)}, {"betas": (0.95, 0.9999)}])
@pytest.mark.parametrize("bits", [8, 32])
def test_hyperparameters(hyper, bits):
    lists = _tensors([1000], torch.float32, torch.float32, bits)
    _check(lists, bits, hyper=HYPER | hyper)


@pytest.mark.parametrize("bits", [8, 32])
def test_gradients_are_scaled_on_the_gpu(bits):
    _check(_tensors([1000, 300], torch.float32, torch.bfloat16, bits), bits, grad_scale=0.37)


def test_eight_bit_moments_start_at_zero_and_follow():
    lists = _tensors([700], torch.float32, torch.float32, 8)
    for name in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
        lists[name][0].zero_()
    for step in range(1, 6):
        _check(lists, 8, step=step)
        lists["grads"][0].mul_(0.5).add_(0.01)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_block_that_is_not_finite(bad):
    """8-bit: the block decodes to NaN throughout, the others are untouched.  32-bit: the element alone."""
    optim = _optim()
    lists = _tensors([600], torch.float32, torch.float32, 8)
    lists["grads"][0][300] = bad
    _check(lists, 8)
    m, v = optim.decode_moments(lists["exp_avg"][0], lists["exp_avg_scale"][0], lists["exp_avg_sq"][0], lists["exp_avg_sq_scale"][0])
    for x in (m, v):
        assert torch.isnan(x[256:512]).all() and torch.isfinite(x[:256]).all() and torch.isfinite(x[512:]).all()
    lists = _tensors([600], torch.float32, torch.float32, 32)
    lists["grads"][0][300] = bad
    _check(lists, 32)


@pytest.mark.parametrize("n", [1, 255, 256, 1000, 100_003])
@pytest.mark.parametrize("offset", [0, 1])
def test_encoding_and_decoding(n, offset):
    optim = _optim()
    gen = torch.Generator().manual_seed(n)
    m = torch.randn(n, generator=gen) * torch.exp2(torch.randint(-30, 10, (n,), generator=gen).float())
    v = m.square()
    place = lambda x: torch.empty(n + offset, dtype=x.dtype, device="cuda")[offset:].copy_(x)  # noqa: E731
    mc, ms, vc, vs = optim.encode_moments(place(m), place(v))
    for got, scale, x, second in ((mc, ms, m, False), (vc, vs, v, True)):
        code, want = ref.encode(x.numpy(), second)
        np.testing.assert_array_equal(got.cpu().numpy(), code)
        np.testing.assert_array_equal(scale.cpu().numpy(), want)
    md, vd = optim.decode_moments(place(mc.cpu()), ms, place(vc.cpu()), vs)
    np.testing.assert_array_equal(md.cpu().numpy(), ref.decode(mc.cpu().numpy(), ms.cpu().numpy(), False))
    np.testing.assert_array_equal(vd.cpu().numpy(), ref.decode(vc.cpu().numpy(), vs.cpu().numpy(), True))


# ------------------------------------------------------------------ the optimizer

def test_float32_optimizer_follows_torch():
    """Against torch's AdamW in 64 bits: a step's float32 roundings move a parameter by a few units of the update."""
    optim = _optim()
    gen = torch.Generator().manual_seed(0)
    shapes = [(33, 7), (5,), (1000,)]
    start = [torch.randn(s, generator=gen) for s in shapes]
    mine = [torch.nn.Parameter(x.cuda()) for x in start]
    theirs = [torch.nn.Parameter(x.double()) for x in start]
    a = optim.AdamW(mine, lr=1e-2, weight_decay=0.1)
    b = torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.1)
    for _ in range(10):
        for p, r in zip(mine, theirs):
            g = torch.randn(p.shape, generator=gen)
            p.grad, r.grad = g.cuda(), g.double()
        a.step()
        b.step()
    for p, r in zip(mine, theirs):
        # ten steps of at most 1e-2, each good to 2^-20, and ten roundings of the parameter
        assert ((p.detach().cpu().double() - r.detach()).abs() <= 10 * (1e-2 * 2.0 ** -20 + 2.0 ** -24 * (r.detach().abs() + 1))).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_minimises_and_resumes(bits):
    """Resumed from a saved state, the steps are the same bits; groups and parameters without a gradient are kept apart."""
    optim = _optim()
    gen = torch.Generator().manual_seed(0)
    target = torch.randn(40, 30, generator=gen).cuda()
    w, extra, idle = (torch.nn.Parameter(torch.zeros(s, device="cuda")) for s in ((40, 30), (7,), (3,)))
    groups = [{"params": [w, idle]}, {"params": [extra], "lr": 1e-3}]
    opt = optim.AdamW(groups, lr=2e-2, weight_decay=0.0, bits=bits)

    def loss():
        return (w - target).square().sum() + (extra - 1).square().sum()

    first = loss().item()
    for i in range(200):
        opt.zero_grad()
        loss().backward()
        if i == 100:
            saved, copies = opt.state_dict(), [p.detach().clone() for p in (w, extra)]
            saved = {"state": {k: {n: x.clone() if torch.is_tensor(x) else x for n, x in s.items()} for k, s in saved["state"].items()},
                     "param_groups": saved["param_groups"]}
        opt.step()
    assert loss().item() < 0.01 * first and bool((idle == 0).all()) and idle not in opt.state
    w2, extra2 = (torch.nn.Parameter(x) for x in copies)
    idle2 = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    again = optim.AdamW([{"params": [w2, idle2]}, {"params": [extra2], "lr": 1e-3}], lr=2e-2, weight_decay=0.0, bits=bits)
    again.load_state_dict(saved)
    for _ in range(100):
        again.zero_grad()
        ((w2 - target).square().sum() + (extra2 - 1).square().sum()).backward()
        again.step()
    assert torch.equal(w, w2) and torch.equal(extra, extra2)
    moments = opt.state[w]["exp_avg"]
    assert moments.dtype == (torch.int8 if bits == 8 else torch.float32)


def test_versions_tell_autograd():
    """A tensor saved for a backward pass that a step then changed is refused, as after torch's own steps."""
    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    opt = _optim().AdamW([p])
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("bits", [8, 32])
def test_a_graph_of_the_step(bits):
    lists = _tensors([1000, 3000], torch.float32, torch.float32, bits)
    first = {n: [x.clone() for x in xs] for n, xs in lists.items()}
    scales = {n: lists[n] for n in ("exp_avg_scale", "exp_avg_sq_scale")} if bits == 8 else {}

    def program():
        _optim().adamw_step(lists["params"], lists["grads"], lists["exp_avg"], lists["exp_avg_sq"], step=7, **HYPER, **scales)

    program()
    torch.cuda.synchronize()
    want = {n: [x.clone() for x in xs] for n, xs in lists.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        program()
    for _ in range(3):
        for n, xs in lists.items():
            for x, y in zip(xs, first[n]):
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for n, xs in lists.items():
            for x, y in zip(xs, want[n]):
                assert torch.equal(x, y)


def test_the_optimizer_refuses_to_be_captured():
    """A captured step would repeat its bias correction; the same optimizer then steps eagerly."""
    p, q = (torch.nn.Parameter(torch.ones(10, device="cuda")) for _ in range(2))
    p.grad, q.grad = torch.full_like(p, 0.5), torch.full_like(q, 0.5)
    opt, other = (_optim().AdamW([x]) for x in (p, q))
    torch.cuda.synchronize()
    graph, kept = torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
    with torch.cuda.graph(graph):
        kept += 1
        with pytest.raises(RuntimeError, match="counts its steps on the host"):
            opt.step()
    assert not opt.state
    graph.replay()
    opt.step()
    other.step()
    assert torch.equal(p, q) and kept.item() == 1.0


def test_inference_tensors_are_refused_before_they_are_changed():
    lists = [torch.ones(10, device="cuda") for _ in range(4)]
    with torch.inference_mode():
        lists[3] = torch.ones(10, device="cuda")
    with pytest.raises(RuntimeError, match="inference tensor"):
        _optim().adamw_step(*([x] for x in lists), step=1, lr=1e-3)
    assert all(bool((x == 1).all()) for x in lists)
