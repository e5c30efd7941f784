"""Norms before and after a block, fused with the block's gate and the residual.

A block ``f`` of a network that keeps a residual stream ``x`` (a layer of
experts, ``expert_mlp``, is one) is used as

    ``x <- x + scale * gate * (norm_out * h / rms(h))``, ``h = f(norm_in * x / rms(x))``,

with ``rms(v) = sqrt(mean(v ** 2) + eps)`` over the channels. ``residual_norm``
computes, in one pass, what follows a block: the stream's update and the next
block's normalised input; ``rms_norm`` is the norm alone, before the first
block. Both have reverse-mode gradients, and run on torch's current CUDA
stream with no wait of the host.
"""

from __future__ import annotations

import math

import torch

from . import _lib as L
from .experts import _DTYPES, _call, _code, _empty, _no_tangent, _number, _on_gpu, _ptr, _rows, _scratch, _together

MIN_EPS = 1e-30


def _stride(t):
    return t.stride(0) if t is not None else 0


def _forward(x, h, norm_in, norm_out, gate, kind, scale, eps, keep):
    """(out or None, y or None, stats or None)"""
    dev, (T, D) = x.device, x.shape
    out = _empty(T, D, x.dtype, dev) if h is not None else None
    y = _empty(T, D, x.dtype, dev) if norm_in is not None else None
    stats = _empty(T, 2, torch.float32, dev) if keep else None
    weight = norm_in if norm_in is not None else norm_out
    _call("es_residual_norm", dev, x.data_ptr(), x.stride(0), _ptr(h), _stride(h), _DTYPES[x.dtype], T, D,
          _ptr(norm_in), _ptr(norm_out), _DTYPES[x.dtype if weight is None else weight.dtype], _ptr(gate), kind,
          _stride(gate) if kind != L.ES_GATE_CHANNEL else 0, scale, eps, _ptr(out), _ptr(y), _ptr(stats))
    return out, y, stats


def _column(n, dtype, dev):
    return torch.empty_strided((n,), (1,), dtype=dtype, device=dev)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, norm_in, norm_out, gate, kind, scale, eps):
        out, y, stats = _forward(x, h, norm_in, norm_out, gate, kind, scale, eps, True)
        ctx.save_for_backward(x, h, norm_in, norm_out, gate, stats)
        ctx.kind, ctx.scale = kind, scale
        ctx.set_materialize_grads(False)
        return out, y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dy):
        if dout is None and dy is None:
            return (None,) * 8
        x, h, norm_in, norm_out, gate, stats = ctx.saved_tensors
        _no_tangent("residual_norm", *(d for d in (dout, dy) if d is not None))
        dev, dtype, (T, D), kind = x.device, x.dtype, x.shape, ctx.kind
        if dout is not None:
            dout = _rows(dout)
        if dy is not None:
            dy = _rows(dy)
        need = ctx.needs_input_grad
        dx = _empty(T, D, dtype, dev) if need[0] else None
        dh = _empty(T, D, dtype, dev) if need[1] else None
        weight = norm_in if norm_in is not None else norm_out
        dnorm_in = _column(D, weight.dtype, dev) if need[2] else None
        dnorm_out = _column(D, weight.dtype, dev) if need[3] else None
        columns = (dnorm_out is not None) + (dnorm_in is not None and dy is not None)
        dgate = None
        if need[4]:
            if kind == L.ES_GATE_CHANNEL:
                dgate = _column(D, dtype, dev)
                columns += 1
            else:
                dgate = _empty(T, gate.shape[1], dtype, dev)
        if dnorm_in is not None and dy is None:
            dnorm_in.zero_()
        code = _DTYPES[dtype]
        nbytes = L.lib().es_residual_norm_grad_workspace_size(code, T, D, columns) if columns else 0
        ws = _scratch(nbytes, dev)
        _call("es_residual_norm_grad", dev, x.data_ptr(), x.stride(0), _ptr(h), _stride(h), code, T, D, _ptr(norm_in),
              _ptr(norm_out), code if weight is None else _DTYPES[weight.dtype], _ptr(gate), kind,
              _stride(gate) if kind != L.ES_GATE_CHANNEL else 0, ctx.scale, stats.data_ptr(), _ptr(dout),
              _stride(dout), _ptr(dy), _stride(dy), _ptr(dx), _ptr(dh), _ptr(dgate),
              _ptr(dnorm_in) if dy is not None else None, _ptr(dnorm_out), _ptr(ws), nbytes)
        return dx, dh, dnorm_in, dnorm_out, dgate, None, None, None


def _weight(fn, name, w, x):
    if w is None:
        return None
    if w.shape != x.shape[1:]:
        raise ValueError(f"{fn}: {name} has shape {tuple(w.shape)}, wanted ({x.shape[1]},)")
    if w.dtype != x.dtype and w.dtype != torch.float32:
        raise TypeError(f"{fn}: {name} must be {x.dtype} or float32, got {w.dtype}")
    return w.contiguous()


def _run(fn, x, h, norm_in, norm_out, gate, scale, eps):
    tensors = [t for t in (x, h, norm_in, norm_out, gate) if t is not None]
    if not _together(*tensors):
        _on_gpu(fn, **{n: t for n, t in zip(("x", "h", "norm_in", "norm_out", "gate"), (x, h, norm_in, norm_out, gate))
                       if t is not None})
    _code(fn, "x", x.dtype)
    if x.dim() != 2:
        raise ValueError(f"{fn}: x must be (num_tokens, width), got {tuple(x.shape)}")
    T, D = x.shape
    if h is not None and (h.shape != x.shape or h.dtype != x.dtype):
        raise ValueError(f"{fn}: h is {h.dtype} {tuple(h.shape)}, x is {x.dtype} {tuple(x.shape)}")
    _number(fn, "scale", scale)
    scale, eps = float(scale), float(eps)
    if not MIN_EPS <= eps < math.inf:
        raise ValueError(f"{fn}: eps={eps} is not in [{MIN_EPS}, inf)")
    norm_in, norm_out = _weight(fn, "norm_in", norm_in, x), _weight(fn, "norm_out", norm_out, x)
    if norm_in is not None and norm_out is not None and norm_in.dtype != norm_out.dtype:
        raise TypeError(f"{fn}: norm_in is {norm_in.dtype}, norm_out is {norm_out.dtype}")
    kind = L.ES_GATE_NONE
    if gate is not None:
        if gate.dtype != x.dtype:
            raise TypeError(f"{fn}: gate is {gate.dtype}, x is {x.dtype}")
        if gate.shape == (D,) or gate.shape == (1, D):
            kind, gate = L.ES_GATE_CHANNEL, gate.reshape(D).contiguous()
        elif gate.shape == (T, 1):
            kind = L.ES_GATE_TOKEN
        elif gate.shape == (T, D):
            kind, gate = L.ES_GATE_FULL, _rows(gate)
        else:
            raise ValueError(f"{fn}: gate has shape {tuple(gate.shape)}, wanted ({D},), (1, {D}), ({T}, 1) or "
                             f"({T}, {D})")
    _no_tangent(fn, *tensors)
    x, h = _rows(x), None if h is None else _rows(h)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return _ResidualNorm.apply(x, h, norm_in, norm_out, gate, kind, scale, eps)
    return _forward(x, h, norm_in, norm_out, gate, kind, scale, eps, False)[:2]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``x * weight / rms(x)`` for each row of ``x`` (num_tokens, width), in
    fp32 and rounded once to x's type. ``weight`` (width,) of x's type or
    float32. Differentiable in both."""
    if weight is None:
        raise TypeError("rms_norm: weight must be a torch tensor, got NoneType")
    return _run("rms_norm", x, None, weight, None, None, 1.0, eps)[1]


def residual_norm(x: torch.Tensor, h: torch.Tensor, norm_in: torch.Tensor | None = None,
                  norm_out: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
                  eps: float = 1e-6):
    """``(out, y)`` after a block whose output is ``h``:
    ``out = x + scale * gate * (norm_out * h / rms(h))`` and the next block's
    input ``y = norm_in * out / rms(out)``, from ``out`` before its rounding.

    ``x``, ``h`` (num_tokens, width) of one type (float32, bfloat16, float16).
    ``norm_out`` None: ``h`` is added as it is; ``norm_in`` None: ``y`` is
    None. The norms' weights (width,) have x's type or float32, both the
    same. ``gate`` of x's type: one value a channel (width,), a token
    (num_tokens, 1), or each value's own (num_tokens, width). ``eps`` is at
    least 1e-30. ``scale`` and ``eps`` are numbers and have no gradient. fp32 throughout, each output rounded once; rows whose squares pass the
    largest value are normalised all the same. Differentiable in every
    tensor; sums over tokens repeat to the bit."""
    if h is None:
        raise TypeError("residual_norm: h must be a torch tensor, got NoneType")
    return _run("residual_norm", x, h, norm_in, norm_out, gate, scale, eps)
