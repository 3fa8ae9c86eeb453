"""Calls of the operators around a policy's layers that their torch layer refuses, for each check of a type or a shape:
pointers reach the kernels without extents, so nothing else keeps a wrong shape from being read past its end."""
from __future__ import annotations

import torch

HEADS = "head sizes must be at least 1, and 16,384 in all at most"
F32, BF16, F16, F64, I8, U8, I16, I32, I64, BOOL = (torch.float32, torch.bfloat16, torch.float16, torch.float64, torch.int8, torch.uint8,
                                                    torch.int16, torch.int32, torch.int64, torch.bool)


def calls(device):
    """For each operator a call that fits, as a function of the arguments that are to differ."""
    from carl_amd import ops

    def new(*shape, dtype=F32):
        return torch.zeros(shape, dtype=dtype, device=device)

    def log_prob(**other):
        a = dict(logits=new(4, 6, 8), actions=new(4, 6, 2, dtype=I32), heads=(5, 3), mask=new(4, 6, 8, dtype=BOOL)) | other
        return ops.action_log_prob(a.pop("logits"), a.pop("actions"), a.pop("heads"), **a)

    def top(**other):
        a = dict(logits=new(4, 6, 8), heads=(5, 3), k=1, mask=new(4, 6, 8, dtype=BOOL), noise=new(4, 6, 8)) | other
        return ops.top_actions(a.pop("logits"), a.pop("heads"), a.pop("k"), **a)

    def norm(call):
        def run(**other):
            a = dict(x=new(4, 6, 16, dtype=BF16), weight=new(16, dtype=BF16), residual=new(4, 6, 16, dtype=BF16)) | other
            return call(a.pop("x"), a.pop("weight"), **a)
        return run

    def quantize(**other):
        return ops.quantize_int8(**(dict(x=new(4, 6, 16)) | other))

    def linear(**other):
        a = dict(x=new(4, 6, 32, dtype=I8), x_scale=new(4, 6), weight=new(12, 32, dtype=I8), weight_scale=new(12), bias=new(12, dtype=BF16)) | other
        return ops.int8_linear(*[a.pop(n) for n in ("x", "x_scale", "weight", "weight_scale")], **a)

    def gated(**other):
        a = dict(x=new(4, 6, 32, dtype=I8), x_scale=new(4, 6), w_gate=new(12, 32, dtype=I8), gate_scale=new(12), w_up=new(12, 32, dtype=I8),
                 up_scale=new(12)) | other
        return ops.int8_gated_linear(*[a.pop(n) for n in ("x", "x_scale", "w_gate", "gate_scale", "w_up", "up_scale")], **a)

    return {"action_log_prob": log_prob, "top_actions": top, "rms_norm": norm(ops.rms_norm), "rms_norm_int8": norm(ops.rms_norm_int8),
            "quantize_int8": quantize, "int8_linear": linear, "int8_gated_linear": gated}


def _tensor(*shape, dtype=F32):
    return lambda device: torch.zeros(shape, dtype=dtype, device=device)


def _logits():
    heads_fit = "logits must have shape"
    for name in ("action_log_prob", "top_actions"):
        for heads, message in (((), "heads must have 1 to 64 sizes"), ((1,) * 65, "heads must have 1 to 64 sizes"), ((8, 0), HEADS),
                               ((-1, 9), HEADS), ((2 ** 40,), HEADS), ((9000, 9000), HEADS), ((5, 4), heads_fit), ((5, 2), heads_fit),
                               ((8, 8), heads_fit)):
            yield name, {"heads": heads}, ValueError, message
        for dtype in (F64, I32, BOOL):
            yield name, {"logits": _tensor(4, 6, 8, dtype=dtype)}, TypeError, "logits must have dtype float32, bfloat16 or float16"
        for shape in ((4, 6, 7), (4, 6, 9), (4, 6, 1), (4, 6, 0), (), (8, 6, 4)):
            yield name, {"logits": _tensor(*shape)}, ValueError, heads_fit
        for dtype in (U8, F32, I64):
            yield name, {"mask": _tensor(4, 6, 8, dtype=dtype)}, TypeError, "mask must have dtype bool"
        for shape in ((4, 6, 7), (4, 6), (6, 8), (4, 5, 8), (3, 6, 8), (1, 1, 8), (8,), (24, 8), (4, 6, 1), (6, 4, 8)):
            yield name, {"mask": _tensor(*shape, dtype=BOOL)}, ValueError, "mask must have the logits' shape"


def _choices():
    for dtype in (I16, I8, F32, BOOL):
        yield "action_log_prob", {"actions": _tensor(4, 6, 2, dtype=dtype)}, TypeError, "actions must have dtype int32 or int64"
    for dtype in (I32, I64):
        for shape in ((4, 6, 1), (4, 6, 3), (4, 6), (4, 5, 2), (3, 6, 2), (24, 2), (2,), (), (1, 6, 2), (6, 4, 2)):
            yield "action_log_prob", {"actions": _tensor(*shape, dtype=dtype)}, ValueError, "actions must have shape"
    for k in (0, 65, -1):
        yield "top_actions", {"k": k}, ValueError, r"k must be in \[1, 64\]"
    for dtype in (BF16, F16, F64, I32):
        yield "top_actions", {"noise": _tensor(4, 6, 8, dtype=dtype)}, TypeError, "noise must have dtype float32"
    for shape in ((4, 6, 7), (4, 5, 8), (6, 8), (24, 8), (8,), (1, 6, 8), (6, 4, 8)):
        yield "top_actions", {"noise": _tensor(*shape)}, ValueError, "noise must have the logits' shape"


def _norms():
    for name in ("rms_norm", "rms_norm_int8"):
        for dtype in (F32, F16):
            yield name, {"weight": _tensor(16, dtype=dtype)}, TypeError, "x and weight must have the same dtype"
            yield name, {"residual": _tensor(4, 6, 16, dtype=dtype)}, TypeError, "x and residual must have the same dtype"
        for shape in ((15,), (17,), (1,), (0,), (1, 16), (16, 1), ()):
            yield name, {"weight": _tensor(*shape, dtype=BF16)}, ValueError, r"weight must have shape \[width\]"
        for shape in ((4, 6, 15), (4, 5, 16), (3, 6, 16), (6, 16), (24, 16), (16,), (1, 1, 16), (6, 4, 16)):
            yield name, {"residual": _tensor(*shape, dtype=BF16)}, ValueError, "residual must have x's shape"
        for eps in (0.0, 9e-31, -1.0, float("inf"), float("nan"), 1e39):
            yield name, {"eps": eps}, ValueError, "eps must be finite and at least 1e-30"
    for name in ("rms_norm", "rms_norm_int8", "quantize_int8"):
        for dtype in (F64, I8, I32):
            yield name, {"x": _tensor(4, 6, 16, dtype=dtype)}, TypeError, "x must have dtype float32, bfloat16 or float16"
        yield name, {"x": _tensor(dtype=BF16)}, ValueError, r"x must have shape \[..., width\]"
        for width in (0, 16_385):
            yield name, {"x": _tensor(2, width, dtype=BF16)}, ValueError, r"width must be in \[1, 16384\]"


def _products():
    for name, weights in (("int8_linear", (("weight", "weight_scale"),)), ("int8_gated_linear", (("w_gate", "gate_scale"), ("w_up", "up_scale")))):
        for dtype in (U8, I16, F32):
            yield name, {"x": _tensor(4, 6, 32, dtype=dtype)}, TypeError, "x must have dtype int8"
        yield name, {"x": _tensor(dtype=I8)}, ValueError, r"x must have shape \[..., width\]"
        for width in (31, 33, 1, 0):
            yield name, {"x": _tensor(4, 6, width, dtype=I8)}, ValueError, rf"{weights[0][0]} must have shape \[columns, width\]"
        for dtype in (BF16, F64, I32):
            yield name, {"x_scale": _tensor(4, 6, dtype=dtype)}, TypeError, "x_scale must have dtype float32"
        for shape in ((4,), (6,), (24,), (4, 5), (3, 6), (4, 6, 1), (1, 1), (6, 4), ()):
            yield name, {"x_scale": _tensor(*shape)}, ValueError, "x_scale must have a value for each row of x"
        for w, scale in weights:
            for dtype in (U8, F32):
                yield name, {w: _tensor(12, 32, dtype=dtype)}, TypeError, f"{w} must have dtype int8"
            for shape in ((12, 31), (12, 33), (32,), (1, 12, 32), (), (32, 12)):
                yield name, {w: _tensor(*shape, dtype=I8)}, ValueError, rf"{w} must have shape \[columns, width\]"
            for dtype in (BF16, I32):
                yield name, {scale: _tensor(12, dtype=dtype)}, TypeError, f"{scale} must have dtype float32"
            for shape in ((11,), (13,), (1,), (12, 1), (1, 12), ()):
                yield name, {scale: _tensor(*shape)}, ValueError, rf"{scale} must have shape \[columns\]"
        for dtype in (I8, F64, None, "float32"):
            yield name, {"dtype": dtype}, TypeError, "dtype must be float32, bfloat16 or float16"
        wide = {"x": _tensor(1, 65_537, dtype=I8), "x_scale": _tensor(1)} | {w: _tensor(12, 65_537, dtype=I8) for w, _ in weights}
        yield name, wide, ValueError, r"width must be in \[1, 65536\]"
        none = {"x": _tensor(1, 0, dtype=I8), "x_scale": _tensor(1)} | {w: _tensor(12, 0, dtype=I8) for w, _ in weights}
        yield name, none, ValueError, r"width must be in \[1, 65536\]"
        for columns in (0, 65_537):
            high = {w: _tensor(columns, 32, dtype=I8) for w, _ in weights} | {s: _tensor(columns) for _, s in weights}
            yield name, high, ValueError, r"columns must be in \[1, 65536\]"
    yield "int8_gated_linear", {"w_up": _tensor(11, 32, dtype=I8), "up_scale": _tensor(11)}, ValueError, "w_up must have shape"
    yield "int8_gated_linear", {"activation": "relu"}, ValueError, "activation must be 'silu' or 'gelu'"
    for dtype in (F32, F16):
        yield "int8_linear", {"bias": _tensor(12, dtype=dtype)}, TypeError, "bias must have the result's dtype"
    yield "int8_linear", {"dtype": F32}, TypeError, "bias must have the result's dtype"
    for shape in ((11,), (13,), (1,), (1, 12), (), (4, 6, 12)):
        yield "int8_linear", {"bias": _tensor(*shape, dtype=BF16)}, ValueError, r"bias must have shape \[columns\]"


# by operator and argument
GROUPS = {}
for _case in (*_logits(), *_choices(), *_norms(), *_products()):
    GROUPS.setdefault("-".join((_case[0], *_case[1])), []).append(_case)


def made(changes, device):
    """The arguments, with tensors on the device."""
    return {n: v(device) if callable(v) else v for n, v in changes.items()}
