"""The learner's operators restated in 64 bits, with bounds on a kernel's error.

Linear attention and the feed-forward block run as they are defined, step by
step and product by product, on CPU tensors.  Beside each value goes the sum
of the magnitudes that it is made of: a float32 sum of n products is off by at
most n 2^-24 of that, and a rounding to the elements' type by at most its unit
roundoff (2^-8 bfloat16, 2^-11 float16, 2^-24 float32) of what is rounded.
AdamW is restated in float32, rounding for rounding, and is compared for
equality.
"""
from __future__ import annotations

import math

import numpy as np
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
EPS = 2.0 ** -24
# a product below float16's normal numbers is rounded to a multiple of 2^-24
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}


def wide(x):
    return None if x is None else x.detach().cpu().double()


# ------------------------------------------------------------ linear attention

def attention(q, k, v, log_decay, starts=None, initial=None, scale=None):
    """(out, final memory) of the recurrence."""
    q, k, v, log_decay, initial = (wide(x) for x in (q, k, v, log_decay, initial))
    B, T, H, dk = q.shape
    group = H // k.shape[2]
    k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    scale = dk ** -0.5 if scale is None else scale
    S = torch.zeros(B, H, dk, v.shape[3], dtype=torch.float64) if initial is None else initial.clone()
    decay = log_decay.exp()[None, :, None, None]
    out = torch.empty(B, T, H, v.shape[3], dtype=torch.float64)
    for t in range(T):
        if starts is not None:
            S = torch.where(starts[:, t].cpu()[:, None, None, None], torch.zeros(()).double(), S)
        S = S * decay + k[:, t, :, :, None] * v[:, t, :, None, :]
        out[:, t] = scale * (q[:, t, :, :, None] * S).sum(-2)
    return out, S


def attention_gradients(q, k, v, log_decay, dout, starts=None, initial=None, dfinal=None, scale=None):
    """(dq, dk, dv, dinitial) from the recurrence run both ways."""
    q, k, v, log_decay, dout, initial, dfinal = (wide(x) for x in (q, k, v, log_decay, dout, initial, dfinal))
    B, T, H, dk = q.shape
    group, dv = H // k.shape[2], v.shape[3]
    ks, vs = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    scale = dk ** -0.5 if scale is None else scale
    decay = log_decay.exp()[None, :, None, None]
    zero = torch.zeros(()).double()

    def cut(S, t):
        return S if starts is None else torch.where(starts[:, t].cpu()[:, None, None, None], zero, S)

    S = torch.zeros(B, H, dk, dv, dtype=torch.float64) if initial is None else initial.clone()
    R = torch.zeros_like(S) if dfinal is None else dfinal.clone()
    dq, dks, dvs = torch.empty_like(q), torch.empty_like(ks), torch.empty_like(vs)
    for t in range(T):
        S = cut(S, t) * decay + ks[:, t, :, :, None] * vs[:, t, :, None, :]
        dq[:, t] = scale * (S * dout[:, t, :, None, :]).sum(-1)
    for t in reversed(range(T)):
        R = R + scale * q[:, t, :, :, None] * dout[:, t, :, None, :]
        dks[:, t] = (R * vs[:, t, :, None, :]).sum(-1)
        dvs[:, t] = (R * ks[:, t, :, :, None]).sum(-2)
        R = cut(R, t) * decay
    share = lambda x: x.view(B, T, -1, group, x.shape[3]).sum(3)  # noqa: E731
    return dq, share(dks), share(dvs), R


def magnitudes(fn, *args, **kwargs):
    """fn on the magnitudes of its tensors and of the scale (decays and starts as they are)."""
    def size(x):
        return x if x is None or torch.is_tensor(x) and x.dtype == torch.bool else abs(x)

    return fn(*(x if i == 3 else size(x) for i, x in enumerate(args)), **{n: size(x) for n, x in kwargs.items()})


def attention_bound(dtype, value, size, steps, width):
    """Of a row's error: its own rounding, one rounding of the weights within a chunk, the carried memory read as two
    terms (16-bit types; their second is off by its own rounding), and float32 sums over steps and width, with decays
    good to a few units."""
    u = UNIT[dtype]
    sums = (steps + width + 64) * EPS
    carried = 0.0 if dtype == torch.float32 else u * u
    return u * value.abs() + (u + carried + sums) * size + TINY[dtype] * (1.0 + size)


def memory_bound(size, steps):
    """Of a memory's element: float32 sums of products whose factors are exact or split into three terms."""
    return (steps + 64) * EPS * size + 2.0 ** -40


# ---------------------------------------------------------- feed-forward block

GELU = math.sqrt(2 / math.pi)


def activation(name, g):
    """(value, slope)"""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s + g * s * (1 - s)
    t = torch.tanh(GELU * (g + 0.044715 * g ** 3))
    return g * (1 + t) / 2, (1 + t) / 2 + g / 2 * (1 - t * t) * GELU * (1 + 0.134145 * g * g)


def ffn(x, w_gate, w_up, w_down, name, dy=None):
    """{"y", "dx", "dw_gate", "dw_up", "dw_down"} and a bound on the error of each."""
    dtype = x.dtype
    u = UNIT[dtype]
    x, wg, wu, wd, dy = (wide(t) for t in (x, w_gate, w_up, w_down, dy))
    N, D = x.shape
    F = wg.shape[0]
    e = lambda n: (n + 16) * EPS  # noqa: E731  a float32 sum of n products, and what follows it
    g, up = x @ wg.t(), x @ wu.t()
    g_off, up_off = e(D) * (x.abs() @ wg.abs().t()), e(D) * (x.abs() @ wu.abs().t())
    act, slope = activation(name, g)
    h = act * up
    # slopes of both activations are below 1.13, their curvature below 1
    act_off = 1.13 * g_off + 2.0 ** -20 * act.abs()
    h_off = u * h.abs() + act_off * up.abs() + act.abs() * up_off + act_off * up_off + TINY[dtype]
    y = h @ wd.t()
    value = {"y": y}
    bound = {"y": u * y.abs() + h_off @ wd.abs().t() + e(F) * (h.abs() @ wd.abs().t()) + TINY[dtype]}
    if dy is None:
        return value, bound
    dh = dy @ wd
    dh_off = e(D) * (dy.abs() @ wd.abs())
    slope_off = g_off + 2.0 ** -20
    dg, du = dh * up * slope, dh * act
    dg_off = u * dg.abs() + 1.2 * (dh_off * up.abs() + dh.abs() * up_off) + (dh * up).abs() * slope_off + TINY[dtype]
    du_off = u * du.abs() + dh_off * act.abs() + dh.abs() * act_off + TINY[dtype]
    value |= {"dx": dg @ wg + du @ wu, "dw_gate": dg.t() @ x, "dw_up": du.t() @ x, "dw_down": dy.t() @ h}
    sums = {
        "dx": (dg_off @ wg.abs() + du_off @ wu.abs(), e(2 * F) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())),
        "dw_gate": (dg_off.t() @ x.abs(), e(N) * (dg.abs().t() @ x.abs())),
        "dw_up": (du_off.t() @ x.abs(), e(N) * (du.abs().t() @ x.abs())),
        "dw_down": (dy.abs().t() @ h_off, e(N) * (dy.abs().t() @ h.abs())),
    }
    for n, (given, summed) in sums.items():
        bound[n] = u * value[n].abs() + given + summed + TINY[dtype]
    return value, bound


def assert_within(got, want, bound, what):
    off = (wide(got) - want).abs()
    worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0 and bool(torch.isfinite(off).all()), f"{what}: {worst:.2f} times the bound"


# ----------------------------------------------------------------------- AdamW

BLOCK = 256
F = np.float32


def _blocks(x):
    """Rows of 256 elements, the last filled up with zeros."""
    pad = -len(x) % BLOCK
    return np.concatenate([x, np.zeros(pad, x.dtype)]).reshape(-1, BLOCK)


def decode(code, scale, second):
    u = code.astype(F) * F(1 / 255 if second else 1 / 127)
    s = np.repeat(scale, BLOCK)[: len(code)]
    if second:
        u = u * u
        return u * u * s
    return u * np.abs(u) * s


def encode(x, second):
    rows = _blocks(x)
    scale = np.abs(rows).max(1).astype(F)
    scale[~np.isfinite(rows).all(1)] = np.nan
    safe = np.where(scale > 0, scale, F(1))[:, None]
    with np.errstate(invalid="ignore"):
        root = np.sqrt(np.abs(rows) / safe)
        if second:
            code = np.maximum(np.rint(F(255) * np.sqrt(root)), F(1)) * (rows > 0)
        else:
            code = np.rint(F(127) * root) * np.sign(rows)
    code = np.where(scale[:, None] > 0, code, 0)
    return code.reshape(-1)[: len(x)].astype(np.uint8 if second else np.int8), scale


def adamw(p, g, m, v, step, lr, betas, eps, weight_decay, grad_scale=None):
    """(p, m, v) after the step, all float32, rounding for rounding."""
    b1, b2 = betas
    if grad_scale is not None:
        g = g * F(grad_scale)
    with np.errstate(all="ignore"):
        m = m * F(b1) + g * F(1 - b1)
        v = v * F(b2) + (g * g) * F(1 - b2)
        root = np.sqrt(v) * F(1 / math.sqrt(1 - b2 ** step)) + F(eps)
        p = p * F(1 - lr * weight_decay) - (m * F(lr / (1 - b1 ** step))) / root
    return p, m, v
