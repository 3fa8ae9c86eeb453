"""The operators around a policy's layers restated on the CPU: in 64 bits with
bounds on a kernel's error, or, where every step of the definition is one
float32 operation (sums that are kept, keys, codes, scaled products), rounding
for rounding, to be compared for equality.

Bounds count float32's roundings (2^-24 each) and one rounding to the results'
type.  Functions of the math library are taken to be good to 4 units.
"""
from __future__ import annotations

import math

import torch

from ops_reference import EPS, TINY, UNIT, wide

NONE = -math.inf
LEAST = torch.tensor(2.0 ** -100)


# --------------------------------------------------------------------- actions

def _heads(logits, heads, mask):
    """For each head its logits in 64 bits and what is available of them."""
    x = wide(logits).reshape(-1, logits.shape[-1])
    there = x != NONE
    if mask is not None:
        there &= mask.cpu().expand(logits.shape).reshape(x.shape)
    first = 0
    for n in heads:
        yield x[:, first:first + n], there[:, first:first + n]
        first += n


class Head:
    """log p, p and H of a head's rows, and what float32 sums may be off by."""

    def __init__(self, x, there):
        zero = torch.zeros(()).double()
        self.there, n = there, x.shape[1]
        self.some = there.any(1)
        most = torch.where(there, x, NONE).amax(1, keepdim=True)
        most = torch.where(self.some[:, None], most, zero)
        d = torch.where(there, x - most, zero)
        e = torch.where(there, torch.exp(d), zero)
        z = e.sum(1, keepdim=True)
        log_z = torch.where(self.some[:, None], torch.log(z), zero)
        self.p = torch.where(self.some[:, None], e / z, zero)
        self.logs = torch.where(there, d - log_z, NONE)
        self.entropy = -(self.p * torch.where(there, d - log_z, zero)).sum(1)
        # of Z, relative: a term's exponent is rounded once, the sum n times; then of log p and of H
        spread = (self.p * d.abs()).sum(1, keepdim=True)
        square = (self.p * d * d).sum(1, keepdim=True)
        z_off = EPS * (n + 16 + spread)
        self.logs_off = z_off + EPS * 4 * (d.abs() + log_z.abs())
        self.entropy_off = (z_off * (1 + spread) + EPS * ((n + 16) * spread + square + 4 * log_z.abs())).squeeze(1)
        self.p_off = self.p * (z_off + EPS * (d.abs() + 8))


def log_prob(logits, actions, heads, mask=None):
    """(log-probability, entropy), each with its bound."""
    actions = actions.cpu().reshape(-1, len(heads)).long()
    total = entropy = off = entropy_off = size = 0.0
    for i, (x, there) in enumerate(_heads(logits, heads, mask)):
        h, a, n = Head(x, there), actions[:, i], x.shape[1]
        at = a.clamp(0, n - 1)[:, None]
        own = torch.where(a < 0, 0.0, torch.where(a >= n, math.nan, h.logs.gather(1, at).squeeze(1)))
        total, entropy = total + own, entropy + h.entropy
        off = off + torch.where(a < 0, 0.0, h.logs_off.gather(1, at).squeeze(1))
        entropy_off = entropy_off + h.entropy_off
        size = size + torch.where(torch.isfinite(own), own.abs(), 0.0)
    lead, sums = logits.shape[:-1], len(heads) * EPS
    return ((total.view(lead), (off + sums * size).view(lead)),
            (entropy.view(lead), (entropy_off + sums * entropy).view(lead)))


def log_prob_gradient(logits, actions, heads, d_log_prob, d_entropy, mask=None):
    """d logits and its bound."""
    dtype, actions = logits.dtype, actions.cpu().reshape(-1, len(heads)).long()
    rows = actions.shape[0]
    lp, ent = (wide(d).expand(logits.shape[:-1]).reshape(rows, 1) for d in (d_log_prob, d_entropy))
    grads, bounds = [], []
    for i, (x, there) in enumerate(_heads(logits, heads, mask)):
        h, a, n = Head(x, there), actions[:, i:i + 1], x.shape[1]
        share = torch.where(a < 0, 0.0, torch.where(a >= n, math.nan, lp))
        hit = (torch.arange(n) == a).double()
        inner = torch.where(there, h.logs, 0.0) + h.entropy[:, None]
        g = torch.where(there, share * (hit - h.p) - ent * h.p * inner, 0.0)
        off = share.abs() * (h.p_off + 2 * EPS * (hit + h.p))
        off = off + ent.abs() * (h.p_off * inner.abs() + h.p * (h.logs_off + h.entropy_off[:, None] + 4 * EPS * (h.logs.abs().clamp(max=1e3) + h.entropy[:, None])))
        off = torch.where(there, off, 0.0)         # (what is not available gets 0, exactly)
        grads.append(g)
        bounds.append(UNIT[dtype] * g.abs() + off + TINY[dtype] + 2.0 ** -120)
    return torch.cat(grads, 1).view(logits.shape), torch.cat(bounds, 1).view(logits.shape)


def top(logits, heads, k, mask=None, noise=None):
    """(actions, log-probabilities, their bound); keys are float32 sums."""
    lead = logits.shape[:-1]
    noise = None if noise is None else noise.cpu().expand(logits.shape).reshape(-1, logits.shape[-1])
    best, logs, offs, first = [], [], [], 0
    for x, there in _heads(logits, heads, mask):
        n = x.shape[1]
        h = Head(x, there)
        key = x.float() if noise is None else x.float() + noise[:, first:first + n]
        rank = torch.where(torch.isnan(key), math.inf, key.double())       # (a NaN goes before all: tested by itself)
        for r in range(x.shape[0]):
            order = sorted((j for j in range(n) if there[r, j]), key=lambda j: (-rank[r, j].item(), j))[:k]
            for i in range(k):
                best.append(order[i] if i < len(order) else -1)
                logs.append(h.logs[r, order[i]].item() if i < len(order) else NONE)
                offs.append(h.logs_off[r, order[i]].item() if i < len(order) else 0.0)
        first += n

    def shaped(x, dtype):
        return torch.tensor(x, dtype=dtype).view(len(heads), -1, k).transpose(0, 1).reshape(*lead, len(heads), k)

    return shaped(best, torch.int32), shaped(logs, torch.float64), shaped(offs, torch.float64)


# ------------------------------------------------------------------------ norm

# Roundings of a sum over a row: at most 32 in a lane, 6 over a wave, 16 over a workgroup; a few for mean, root and reciprocal.
ROW = 64 * EPS
# bfloat16's numbers below 2^-126 lie 2^-133 apart, so a rounding there is off by up to 2^-134 (float32's by 2^-150)
LAST = 2.0 ** -134 + 2.0 ** -140


def kept_sum(x, residual):
    x, residual = x.detach().cpu(), residual.detach().cpu()
    return (x.float() + residual.float()).to(x.dtype)


def norm(x, weight, residual=None, eps=1e-6, dy=None, dsum=None):
    """({"y", "dx", "dweight"}, bounds) of the norm of x, or of the kept sum."""
    dtype, u = x.dtype, UNIT[x.dtype]
    s = wide(x) if residual is None else kept_sum(x, residual).double()
    w, D = wide(weight), x.shape[-1]
    s = s.reshape(-1, D)
    r = (s.square().mean(1, keepdim=True) + eps).rsqrt()
    unit = s * r
    value = {"y": unit * w}
    bound = {"y": u * value["y"].abs() + 2 * ROW * value["y"].abs() + TINY[dtype] + LAST}
    if dy is not None:
        dy = wide(dy).expand(x.shape).reshape(-1, D)
        g = dy * w
        inner, size = (g * unit).mean(1, keepdim=True), (g * unit).abs().mean(1, keepdim=True)
        on = torch.zeros(()).double() if dsum is None else wide(dsum).expand(x.shape).reshape(-1, D)
        value["dx"] = r * (g - unit * inner) + on
        bound["dx"] = (u * value["dx"].abs() + 4 * ROW * r * (g.abs() + unit.abs() * size) + EPS * on.abs() + TINY[dtype] + LAST)
        value["dweight"] = (dy * unit).sum(0)
        rows = dy.shape[0] / 256 + 200        # a lane's rows, a workgroup's lanes, the workgroups
        bound["dweight"] = u * value["dweight"].abs() + (rows * EPS + 2 * ROW) * (dy * unit).abs().sum(0) + TINY[dtype] + LAST
    return ({n: v.view(x.shape) if n != "dweight" else v for n, v in value.items()},
            {n: v.view(x.shape) if n != "dweight" else v for n, v in bound.items()})


def codes(t):
    """Codes and m / 127 of float32 rows t, rounding for rounding."""
    t = t.reshape(-1, t.shape[-1])
    most = t.abs().amax(1)
    finite = torch.isfinite(most)
    most = torch.maximum(torch.where(finite, most, torch.ones(())), LEAST)
    inverse = torch.full_like(most, 127.0) / most
    code = torch.round(t * inverse[:, None])
    code = torch.where(finite[:, None], code, torch.zeros(()))
    scale = torch.where(finite, most / torch.full_like(most, 127.0), torch.tensor(math.nan))
    return code.to(torch.int8), scale


# ------------------------------------------------------------ products in 8 bits

def product(x, x_scale, w, w_scale, bias=None):
    """Rounding for rounding, in float32."""
    acc = (x.cpu().double() @ w.cpu().double().t()).float()          # whole numbers below 2^53: exact, then rounded once
    y = acc * x_scale.cpu()[..., None] * w_scale.cpu()
    return y if bias is None else y + bias.cpu().float()


def gated(x, x_scale, gate, gate_scale, up, up_scale, name, dtype):
    """Value and bound, from both products' float32 values."""
    g, u = product(x, x_scale, gate, gate_scale).double(), product(x, x_scale, up, up_scale).double()
    # (1 + tanh v) / 2 = s(2 v): the left side has lost its digits where tanh is near -1
    z = g if name == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    y = g * torch.sigmoid(z) * u
    z = z.abs()
    # act(g) = g s(z): z's rounding and the exponential's, which s passes on where it is small
    off = (32 + 8 * z.clamp(max=200.0)) * EPS * y.abs()
    # (s below float32's normal numbers is given as zero)
    return y, UNIT[dtype] * y.abs() + off + TINY[dtype] + 2.0 ** -120 * (1 + (g * u).abs())
