"""Cases of the operators around a policy's layers: what a program that acts in the
simulator, and trains on what it saw, has the GPU do between the large products
and after the last one.

A case's `op` is one of
  act      the best action of each head of every agent, or a sample where noise
           is added to the logits, with its log-probability (or the `k` best)
  logp+    log-probability and entropy of a rollout's actions, and the gradient
           of both by the logits
  norm     root-mean-square norm, forward only
  norm+    the norm of a residual stream that an addition has just reached, with
           the gradients of both, of the weight and of the stream that goes on
  norm8    acting in 8 bits: the addition, the norm and its 8-bit output, and
           the projection that reads it (`gated`: the two of a gated block)
  rows8    acting in 8 bits: rows put into 8 bits, and their projection
  linear8  a projection of rows that are in 8 bits already

Actions: `heads` are the sizes of a policy's action heads, whose logits lie next
to each other in a row; a masked action is never taken and weighs nothing.

Codes in 8 bits: a row of values t has one float32 scale; with m the largest
magnitude (at least 2^-100) and i = 127 / m its codes are round(t i), to even,
and stand for code m / 127.  A norm's row is t = s w, with s the sum as it is
kept, and its scale holds the norm's factor too.  Codes lie in rows that begin
every 16 bytes, as the operators that make them write them.
"""
from __future__ import annotations

import math

import torch

own = False          # set by whoever imports this file: the framework's operators, or their plain forms

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CAR = "car"          # the simulator's own heads: throttle, steer, pitch, powerslide, boost, air roll, jump
CAR_HEADS = (3, 3, 3, 2, 2, 3, 2)
CAR_MASKED = (10, 12, 17)      # the logits of powerslide, boost and jump, which are not always to be had
EPS = 1e-6
LEAST = 2.0 ** -100


def _heads_of(case: dict) -> tuple[int, ...]:
    return CAR_HEADS if case["heads"] == CAR else (case["heads"],) * case["copies"]


def _act(name, N, *, heads=CAR, copies=1, dtype="bf16", k=1, noise=True, mask=True):
    return {"name": name, "op": "act", "N": N, "heads": heads, "copies": copies, "dtype": dtype, "k": k, "noise": noise, "mask": mask}


def _logp(name, N, *, heads=CAR, copies=1, dtype="bf16", mask=True):
    return {"name": name, "op": "logp+", "N": N, "heads": heads, "copies": copies, "dtype": dtype, "mask": mask}


def _norm(name, N, D, *, op="norm+", dtype="bf16"):
    return {"name": name, "op": op, "N": N, "D": D, "dtype": dtype}


def _eight(name, op, N, D, F, *, gated=False, bias=False, dtype="bf16"):
    return {"name": name, "op": op, "N": N, "D": D, "F": F, "gated": gated, "bias": bias, "dtype": dtype}


def listed() -> list[dict]:
    return [
        # both cars of 17 matches act once: a small evaluation, where latency counts
        _act("act 34 agents", 34, dtype="f32"),
        # both cars of the headline benchmark's 65,536 matches act once
        _act("act 131072 agents", 131072),
        # rollouts of 1,000 1v1 matches, 31 steps, of a policy with one table of actions for a car
        _logp("logp+ 62000 of 90", 62000, heads=90, dtype="f32", mask=False),
        # rollouts of 8,192 1v1 matches, 64 steps, of a policy with the simulator's heads
        _logp("logp+ 1048576", 1048576),
        # both cars of 17 matches, an odd width
        _norm("norm 34 x 683", 34, 683, op="norm", dtype="f16"),
        # a training pass over 2,000 agents x 31 steps in the engine's own type
        _norm("norm+ 62000 f32", 62000, 256, dtype="f32"),
        # a training pass over 8,192 agents x 32 steps
        _norm("norm+ 262144", 262144, 512),
        # queries, keys and values of both cars of 17 matches
        _eight("norm8 34", "norm8", 34, 256, 768),
        # gate and up projections of every car of the headline benchmark's matches
        _eight("norm8 gated 131072", "norm8", 131072, 512, 1408, gated=True),
        # a block's inner values and its down projection, for as many
        _eight("rows8 131072", "rows8", 131072, 1408, 512),
        # an odd projection of a middling evaluation, results in float32
        _eight("linear8 2001 x 683", "linear8", 2001, 683, 257, bias=True, dtype="f32"),
        # a wide policy's projection
        _eight("linear8 16384 x 1024", "linear8", 16384, 1024, 2816, bias=True),
    ]


def draw(rng) -> dict:
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng) -> dict:
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["act", "logp+", "norm", "norm+", "norm8", "rows8", "linear8"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("act", "logp+"):
        heads = rng.choice([CAR, CAR, log(2, 33), log(34, 2000)])
        copies = 1 if heads == CAR or heads > 200 else rng.randint(1, 8)
        logits = sum(CAR_HEADS) if heads == CAR else heads * copies
        N = log(1, min(1048576, 20_000_000 // logits))
        mask = rng.random() < 0.6
        if op == "logp+":
            return _logp("", N, heads=heads, copies=copies, dtype=dtype, mask=mask)
        k = 1 if heads == CAR else rng.choice([1, 1, 2, 5])
        return _act("", N, heads=heads, copies=copies, dtype=dtype, k=k, noise=rng.random() < 0.7, mask=mask)
    odd = 1 if rng.random() < 0.3 else 0
    if op.startswith("norm") and op != "norm8":
        D = log(16, 8192) | odd
        return _norm("", log(1, min(262144, 100_000_000 // D)), D, op=op, dtype=dtype)
    D, F = log(16, 4096) | odd, log(16, 2816) | (1 if rng.random() < 0.3 else 0)
    gated = op == "norm8" and rng.random() < 0.5
    most = min(131072, 40_000_000 // max(D, F), 80_000_000_000 // (D * F))
    return _eight("", op, log(1, most), D, F, gated=gated, bias=not gated and rng.random() < 0.5, dtype=dtype)


# ------------------------------------------------------------------ the inputs

def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, N, op = DTYPES[case["dtype"]], case["N"], case["op"]
    state = {"case": case}

    def randn(*shape, scale=1.0, to=dtype):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).mul_(scale).to(to)

    if op in ("act", "logp+"):
        heads = _heads_of(case)
        L = sum(heads)
        state["logits"] = randn(N, L, scale=2.0)
        mask = None
        if case["mask"]:
            # what the simulator masks, or a table's actions that are no use just now; a head's first is always to be had
            mask = torch.ones(N, L, dtype=torch.bool, device=DEVICE)
            some = torch.rand(N, L, generator=gen, device=DEVICE) < 0.7
            if case["heads"] == CAR:
                mask[:, CAR_MASKED] = some[:, CAR_MASKED]
            else:
                mask = some
                mask[:, ::case["heads"]] = True
        state["mask"] = mask
        gumbel = -torch.log(-torch.log(torch.rand(N, L, generator=gen, device=DEVICE).clamp(1e-7, 1.0 - 1e-7)))
        if op == "act":
            state["noise"] = gumbel if case["noise"] else None
            return state
        key = state["logits"].float() + gumbel      # actions as the policy itself drew them
        if mask is not None:
            key = key.masked_fill(~mask, -math.inf)
        state["actions"] = torch.stack([h.argmax(-1) for h in key.split(heads, -1)], -1).int()
        state["d_log_prob"], state["d_entropy"] = randn(N, to=torch.float32), torch.full((N,), -0.01, device=DEVICE)
        state["logits"].requires_grad_()
        return state

    D = case["D"]
    if op in ("norm", "norm+", "norm8"):
        state["x"] = randn(N, D)
        state["weight"] = (1.0 + randn(D, scale=0.2, to=torch.float32)).to(dtype)
        if op != "norm":
            state["residual"] = randn(N, D, scale=3.0)
        if op == "norm+":
            state["dy"], state["dsum"] = randn(N, D), randn(N, D)
            state["leaves"] = [state[n].requires_grad_() for n in ("x", "residual", "weight")]
    if op in ("norm", "norm+"):
        return state
    F = case["F"]
    if op == "rows8":
        state["x"] = randn(N, D)
    elif op == "linear8":
        state["codes"], state["scale"] = _encode(randn(N, D, to=torch.float32))
    for name in ("gate", "up") if case["gated"] else ("w",):
        state[name], state[name + "_scale"] = _encode(randn(F, D, scale=D ** -0.5, to=torch.float32))
    state["bias"] = randn(F) if case["bias"] else None
    return state


# ------------------------------------------------------------------ plain forms

def _encode(t):
    """Codes, in rows padded to 16 bytes, and the scales of float32 rows."""
    most = t.abs().amax(-1).clamp(min=LEAST)
    inverse = torch.full_like(most, 127.0) / most        # (127.0 / most would be a reciprocal, rounded, and its product)
    rows = torch.zeros(t.shape[0], -(-t.shape[1] // 16) * 16, dtype=torch.int8, device=t.device)
    codes = rows[:, :t.shape[1]]
    codes.copy_(torch.round(t * inverse[:, None]))
    return codes, most / 127.0


def _split_logits(state):
    heads = _heads_of(state["case"])
    x = state["logits"].detach().float()
    if state["mask"] is not None:
        x = x.masked_fill(~state["mask"], -math.inf)
    return heads, x


def _log_softmax(x):
    x = x - x.amax(-1, keepdim=True)
    return x - torch.log(torch.exp(x).sum(-1, keepdim=True))


def _plain_act(state):
    heads, x = _split_logits(state)
    k = state["case"]["k"]
    key = x if state["noise"] is None else x + state["noise"]
    actions, log_prob = [], []
    for h, y in zip(x.split(heads, -1), key.split(heads, -1)):
        order = torch.sort(y, dim=-1, descending=True, stable=True)[1][:, :k] if k > 1 else y.argmax(-1, keepdim=True)
        picked = _log_softmax(h).gather(-1, order)
        short = k - order.shape[1]
        if short > 0:
            order, picked = torch.nn.functional.pad(order, (0, short), value=-1), torch.nn.functional.pad(picked, (0, short), value=-math.inf)
        actions.append(torch.where(torch.isinf(picked), -1, order).int())
        log_prob.append(picked)
    return {"actions": torch.stack(actions, 1), "log_prob": _finite(torch.stack(log_prob, 1))}


def _finite(x):
    """What is not there has the log-probability -infinity: given as a number, so that it can be compared."""
    return torch.where(torch.isinf(x), -1e4, x)


def _plain_logp(state):
    heads, x = _split_logits(state)
    actions = state["actions"].long()
    log_prob, entropy, grads = 0.0, 0.0, []
    for i, h in enumerate(x.split(heads, -1)):
        logs = _log_softmax(h)
        p = torch.exp(logs)
        weighed = torch.where(p > 0, p * logs, 0.0)
        own_entropy = -weighed.sum(-1)
        log_prob = log_prob + logs.gather(-1, actions[:, i:i + 1]).squeeze(-1)
        entropy = entropy + own_entropy
        there = torch.arange(h.shape[1], device=DEVICE) == actions[:, i:i + 1]
        grad = state["d_log_prob"][:, None] * (there.float() - p) - state["d_entropy"][:, None] * (weighed + p * own_entropy[:, None])
        grads.append(torch.where(torch.isinf(h), 0.0, grad))
    return {"log_prob": log_prob, "entropy": entropy, "dlogits": torch.cat(grads, -1).to(state["logits"].dtype)}


def _added(state):
    x = state["x"].detach()
    if "residual" not in state:
        return x
    return (x.float() + state["residual"].detach().float()).to(x.dtype)


def _plain_norm(state):
    dtype, w = state["x"].dtype, state["weight"].detach().float()
    total = _added(state)
    s = total.float()
    r = 1.0 / torch.sqrt((s * s).mean(-1, keepdim=True) + EPS)
    unit = s * r
    outputs = {"y": (unit * w).to(dtype)}
    if state["case"]["op"] == "norm":
        return outputs
    dy = state["dy"].float()
    g = dy * w
    d = r * (g - unit * (g * unit).mean(-1, keepdim=True)) + state["dsum"].float()
    outputs |= {"sum": total, "dx": d.to(dtype), "dresidual": d.to(dtype), "dweight": (dy * unit).sum(0).to(dtype)}
    return outputs


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _plain_eight(state):
    case, dtype = state["case"], DTYPES[state["case"]["dtype"]]
    outputs = {}
    if case["op"] == "linear8":
        codes, scale = state["codes"], state["scale"]
    elif case["op"] == "rows8":
        codes, scale = _encode(state["x"].float())
    else:
        outputs["sum"] = _added(state)
        s = outputs["sum"].float()
        codes, scale = _encode(s * state["weight"].float())
        scale = scale / torch.sqrt((s * s).mean(-1) + EPS)
    x = codes.float()

    def product(name):
        return (x @ state[name].float().t()) * scale[:, None] * state[name + "_scale"]

    if case["gated"]:
        y = _silu(product("gate")) * product("up")
    else:
        y = product("w")
        if state["bias"] is not None:
            y = y + state["bias"].float()
    outputs["y"] = y.to(dtype)
    return outputs


# ------------------------------------------------------------------ one pass

def _own(state):
    from carl_amd import ops

    case, op = state["case"], state["case"]["op"]
    if op == "act":
        actions, log_prob = ops.top_actions(state["logits"], _heads_of(case), case["k"], mask=state["mask"], noise=state["noise"])
        # one action of each head is always to be had; of more, those that are not there are told by their numbers
        return {"actions": actions, "log_prob": log_prob if case["k"] == 1 else _finite(log_prob)}
    if op == "logp+":
        log_prob, entropy = ops.action_log_prob(state["logits"], state["actions"], _heads_of(case), mask=state["mask"])
        (grad,) = torch.autograd.grad([log_prob, entropy], [state["logits"]], [state["d_log_prob"], state["d_entropy"]])
        return {"log_prob": log_prob.detach(), "entropy": entropy.detach(), "dlogits": grad}
    if op == "norm":
        return {"y": ops.rms_norm(state["x"], state["weight"], eps=EPS)}
    if op == "norm+":
        y, total = ops.rms_norm(state["x"], state["weight"], residual=state["residual"], eps=EPS)
        grads = torch.autograd.grad([y, total], state["leaves"], [state["dy"], state["dsum"]])
        return {"y": y.detach(), "sum": total.detach(), "dx": grads[0], "dresidual": grads[1], "dweight": grads[2]}
    dtype = DTYPES[case["dtype"]]
    outputs = {}
    if op == "linear8":
        codes, scale = state["codes"], state["scale"]
    elif op == "rows8":
        codes, scale = ops.quantize_int8(state["x"])
    else:
        codes, scale, outputs["sum"] = ops.rms_norm_int8(state["x"], state["weight"], residual=state["residual"], eps=EPS)
    if case["gated"]:
        outputs["y"] = ops.int8_gated_linear(codes, scale, state["gate"], state["gate_scale"], state["up"], state["up_scale"], dtype=dtype)
    else:
        outputs["y"] = ops.int8_linear(codes, scale, state["w"], state["w_scale"], bias=state["bias"], dtype=dtype)
    return outputs


def run(state: dict):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "act":
        return _plain_act(state)
    if op == "logp+":
        return _plain_logp(state)
    if op in ("norm", "norm+"):
        return _plain_norm(state)
    return _plain_eight(state)


# ------------------------------------------------------------------ what it takes

def work(case: dict) -> dict:
    """Bytes: every input read once, every output written once, with the codes between two operators of a pass, which
    are an output of one and an input of the other.  Operations: about ten for each logit and element, a gradient's as
    many again, and the products."""
    size, N, op = 4 if case["dtype"] == "f32" else 2, case["N"], case["op"]
    if op in ("act", "logp+"):
        heads = _heads_of(case)
        L = sum(heads)
        read = N * L * (size + (1 if case["mask"] else 0))
        if op == "act":
            return {"bytes": read + (4 * N * L if case["noise"] else 0) + 8 * N * len(heads) * case["k"], "flops": 10 * N * L}
        return {"bytes": read + 4 * N * len(heads) + 16 * N + N * L * size, "flops": 20 * N * L}
    D = case["D"]
    rows = N * D * size
    if op == "norm":
        return {"bytes": 2 * rows + D * size, "flops": 5 * N * D}
    if op == "norm+":
        # x, the residual and both gradients in, y, the sum and one gradient (of x and of the residual alike) out
        return {"bytes": 7 * rows + 2 * D * size, "flops": 15 * N * D}
    F, weights = case["F"], 2 if case["gated"] else 1
    total = weights * F * (D + 4) + N * F * size + (F * size if case["bias"] else 0) + N * (D + 4)
    if op != "linear8":
        total += N * (D + 4) + (3 * rows + D * size if op == "norm8" else rows)
    return {"bytes": total, "flops": 2 * weights * N * D * F}


# ------------------------------------------------------------------ 64 bits

def exact(case: dict, seed: int):
    """The operators as they are defined, in 64 bits; what the definition rounds (a sum that is kept, the key of a
    choice, what a code is rounded from) is rounded there."""
    state = prepare(case, seed)
    op = case["op"]
    if op in ("act", "logp+"):
        return _exact_actions(state)
    total = None
    if "x" in state:
        total = state["x"].detach().double()
        if "residual" in state:
            total = (total + state["residual"].detach().double()).to(DTYPES[case["dtype"]]).double()
    if op in ("norm", "norm+"):
        w = state["weight"].detach().double()
        var = total.square().mean(1, keepdim=True) + EPS
        outputs = {"y": w * total / var.sqrt()}
        if op == "norm+":
            dy = state["dy"].double()
            inner = (dy * w * total).mean(1, keepdim=True)
            d = dy * w / var.sqrt() - total * inner / var ** 1.5 + state["dsum"].double()
            outputs |= {"sum": total, "dx": d, "dresidual": d, "dweight": torch.mv((dy * total).t(), var.rsqrt().squeeze(1))}
        return outputs
    outputs = {}
    if op == "linear8":
        values = state["codes"].double() * state["scale"].double()[:, None]
    else:
        t, factor = total, 1.0
        if op == "norm8":
            outputs["sum"] = total
            t = (total * state["weight"].double()).float().double()
            factor = (total.square().mean(1, keepdim=True) + EPS).rsqrt()
        most = t.abs().max(1, keepdim=True)[0].clamp(min=LEAST)
        codes = (t * (127 / most).float().double()).float().round().double()
        values = codes * most / 127 * factor

    def product(name):
        return torch.mm(values, (state[name].double() * state[name + "_scale"].double()[:, None]).t())

    if case["gated"]:
        gate = product("gate")
        outputs["y"] = gate * torch.sigmoid(gate) * product("up")
    else:
        outputs["y"] = product("w")
        if state["bias"] is not None:
            outputs["y"] += state["bias"].double()
    return outputs


def _exact_actions(state):
    case = state["case"]
    N, rows = case["N"], torch.arange(case["N"], device=DEVICE)
    logits = state["logits"].detach().double()
    there = torch.ones_like(logits, dtype=torch.bool) if state["mask"] is None else state["mask"]
    first, actions, log_prob, entropy = 0, [], [], torch.zeros(N, dtype=torch.float64, device=DEVICE)
    total, grad = torch.zeros_like(entropy), torch.zeros_like(logits)
    for i, n in enumerate(_heads_of(case)):
        at = slice(first, first + n)
        x, have = logits[:, at], there[:, at]
        top = torch.where(have, x, -1e300).max(1, keepdim=True)[0]
        weight = torch.where(have, torch.exp(x - top), 0.0)
        z = weight.sum(1, keepdim=True)
        logs, p = x - top - torch.log(z), weight / z
        if case["op"] == "act":
            key = x if state["noise"] is None else (x + state["noise"][:, at].double()).float().double()
            key = torch.where(have, key, -1e300)
            for _ in range(case["k"]):
                best = (key == key.max(1, keepdim=True)[0]).long().argmax(1)
                left = key[rows, best] > -1e300
                actions.append(torch.where(left, best, -1).int())
                log_prob.append(torch.where(left, logs[rows, best], -1e4))
                key = key.clone()
                key[rows, best] = -1e300
        else:
            a = state["actions"][:, i].long()
            own_entropy = -(p * torch.where(have, logs, 0.0)).sum(1)
            total += logs[rows, a]
            entropy += own_entropy
            slope = -p
            slope[rows, a] += 1.0
            g = slope * state["d_log_prob"].double()[:, None]
            g -= state["d_entropy"].double()[:, None] * p * (torch.where(have, logs, 0.0) + own_entropy[:, None])
            grad[:, at] = torch.where(have, g, 0.0)
        first += n
    if case["op"] == "act":
        shape = (N, len(_heads_of(case)), case["k"])
        return {"actions": torch.stack(actions, 1).view(shape), "log_prob": torch.stack(log_prob, 1).view(shape)}
    return {"log_prob": total, "entropy": entropy, "dlogits": grad}
