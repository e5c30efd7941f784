"""Gated products, ``act(x @ gate) * (x @ up)``: the first half of a gated feed-forward block, dense or by expert."""

from __future__ import annotations

import torch

from . import _lib as L
from .experts import (_DTYPES, ExpertPlan, _call, _check_rows, _code, _combine, _empty, _grouped, _no_tangent, _on_gpu,
                      _product, _rows, _together, _wgrad)

ACTIVATIONS = {"silu": L.ES_ACT_SILU, "gelu": L.ES_ACT_GELU, "gelu_tanh": L.ES_ACT_GELU_TANH, "relu": L.ES_ACT_RELU}


def _activation(fn: str, name) -> int:
    code = ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"{fn}: activation {name!r} is none of {', '.join(ACTIVATIONS)}")
    return code


def _gated(x, w, plan, gather, act, keep):
    """``(h, slopes or None)`` for w (num_experts or 1, K, 2 F)."""
    dev = x.device
    K, F = w.shape[1], w.shape[2] // 2
    E, R = (plan.num_experts, plan.num_rows) if plan is not None else (0, x.shape[0])
    h = _empty(R, F, x.dtype, dev)
    slopes = _empty(R, 2 * F, torch.float32, dev) if keep else None
    args = (x.data_ptr(), _DTYPES[x.dtype], x.shape[0], x.stride(0), w.data_ptr(), E, K, F, *w.stride(),
            plan.offsets.data_ptr() if E else None, plan.order.data_ptr() if gather else None, plan.top_k if E else 1,
            R)
    _product("es_gated_matmul", dev, args, (act, h.data_ptr(), slopes.data_ptr() if keep else None),
             gather or x.dtype == torch.float32)
    return h, slopes


class _GatedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, plan, gather, act):
        h, slopes = _gated(x, w, plan, gather, act, True)
        ctx.save_for_backward(x, w, slopes)
        ctx.plan, ctx.gather = plan, gather
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, w, slopes = ctx.saved_tensors
        plan, gather, dev = ctx.plan, ctx.gather, x.device
        _no_tangent("gated_matmul", dh)
        dh = _rows(dh)
        R, F = dh.shape
        dy = _empty(R, 2 * F, dh.dtype, dev)
        _call("es_gated_matmul_grad", dev, dh.data_ptr(), _DTYPES[dh.dtype], dh.stride(0), slopes.data_ptr(), R, F,
              plan.offsets.data_ptr() + 4 * plan.num_experts if plan is not None else None, dy.data_ptr())
        dx = dw = None
        if ctx.needs_input_grad[0]:
            # a token's rows are summed before its gradient is rounded
            dx = _grouped(dy, w.transpose(1, 2), plan, False, torch.float32 if gather else x.dtype)
            if gather:
                dx = _combine(dx, None, plan, x.dtype)
        if ctx.needs_input_grad[1]:
            dw = _wgrad(x, dy, w, plan, gather)
        return dx, dw, None, None, None


def gated_matmul(x: torch.Tensor, w: torch.Tensor, plan: ExpertPlan | None = None, gather: bool = False,
                 activation: str = "silu") -> torch.Tensor:
    """``act(x @ gate) * (x @ up)`` with ``w = [gate | up]`` side by side:
    both products, the activation and their product, sums in fp32, rounded once.

    Without a ``plan``: ``x`` (rows, K), ``w`` (K, 2 F), any strides. With
    one the products are grouped by expert as in ``grouped_matmul``: ``w``
    (num_experts, K, 2 F), and ``x`` (num_rows, K) in the plan's order or,
    with ``gather``, (num_tokens, K). ``activation`` is ``"silu"``, ``"gelu"``
    (by erf), ``"gelu_tanh"`` or ``"relu"``. Returns (rows, F) of x's type
    (float32, bfloat16, float16); rows of no expert are zero. Differentiable
    in ``x`` and ``w``; a training step keeps the output's slopes in both
    products, (rows, 2 F) float32, 8 F bytes a row. F a multiple of 8 (16
    bits) is fastest: else half of the weights or all are copied in every call."""
    if plan is not None and not isinstance(plan, ExpertPlan):
        raise TypeError(f"gated_matmul: plan must be an ExpertPlan or None, got {type(plan).__name__}")
    if not _together(x, w, x if plan is None else plan.offsets):
        _on_gpu("gated_matmul", x=x, w=w, plan=x if plan is None else plan.offsets)
    _code("gated_matmul", "x", x.dtype)
    act = _activation("gated_matmul", activation)
    if w.dtype != x.dtype:
        raise TypeError(f"gated_matmul: x is {x.dtype}, w is {w.dtype}")
    if w.dim() != (2 if plan is None else 3) or w.shape[-1] % 2 or (plan is not None and
                                                                   w.shape[0] != plan.num_experts):
        raise ValueError(f"gated_matmul: w has shape {tuple(w.shape)}, wanted "
                         + ("(K, 2 F)" if plan is None else f"({plan.num_experts}, K, 2 F)"))
    gather = bool(gather)
    if plan is not None:
        _check_rows("gated_matmul", x, "x", plan, gather, w.shape[1])
    elif gather or x.dim() != 2 or x.shape[1] != w.shape[0]:
        raise ValueError(f"gated_matmul: x has shape {tuple(x.shape)}, wanted (rows, {w.shape[0]}); "
                         "gather needs a plan")
    _no_tangent("gated_matmul", x, w)
    x, w = _rows(x), w if plan is not None else w.unsqueeze(0)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        return _GatedMatmul.apply(x, w, plan, gather, act)
    return _gated(x, w, plan, gather, act, False)[0]
