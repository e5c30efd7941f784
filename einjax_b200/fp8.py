"""Products of 8-bit floating point (e4m3) with a scale for each block of 128: the serving form beside ``int8_matmul``.

Rows are rounded as they come, with a scale for each 128 values; weights are
rounded once, with a scale for each 128 x 128 block, or taken from a checkpoint
that holds them so. Nothing here is differentiable."""

from __future__ import annotations

import math

import torch

from . import _lib as L
from .experts import (ExpertPlan, _call, _check_rows, _code, _empty, _groups, _on_gpu, _product, _rows, _together)
from .gated import _activation

BLOCK = 128

_E4M3 = torch.float8_e4m3fn


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def quantize_blocks(x: torch.Tensor, activation: str | None = None):
    """``(q, scale)``: each row of ``x`` (rows, width) in e4m3 with a float32
    scale for each 128 of its values, (rows, ceil(width / 128)). A scale is the
    smallest power of two ``s`` (at least 2^-126) with ``max |x| <= 448 s``;
    ``q = e4m3(x / s)`` is rounded to nearest, ties to even. A block with an
    infinity or NaN has scale and values NaN.

    With an ``activation`` (as in ``gated_matmul``) ``x`` is (rows, 2 width),
    gate and up side by side, and what is rounded is ``act(gate) * up``, made
    in fp32. Not differentiable: the result has no history."""
    if not _together(x):
        _on_gpu("quantize_blocks", x=x)
    code = _code("quantize_blocks", "x", x.dtype)
    act = -1 if activation is None else _activation("quantize_blocks", activation)
    if x.dim() != 2 or (act >= 0 and x.shape[1] % 2):
        raise ValueError(f"quantize_blocks: x must be (rows, {'width' if act < 0 else '2 width'}), got {tuple(x.shape)}")
    dev, x = x.device, _rows(x)
    R, K = x.shape
    if act >= 0:
        K //= 2
    q = _empty(R, K, _E4M3, dev)
    scale = _empty(R, _blocks(K), torch.float32, dev)
    _call("es_quantize_blocks", dev, x.data_ptr(), code, R, K, x.stride(0), act, q.data_ptr(), scale.data_ptr())
    return q, scale


def quantize_block_weights(w: torch.Tensor):
    """Weights ``w`` (..., K, N) as ``fp8_matmul`` takes them: ``(wq, scale)``
    with ``wq`` e4m3 (..., N, K), contiguous along K, and a float32 scale for
    each 128 x 128 block, (..., ceil(N / 128), ceil(K / 128)), by the rule of
    ``quantize_blocks``."""
    if not isinstance(w, torch.Tensor) or w.dim() < 2:
        raise ValueError("quantize_block_weights: w must be a tensor (..., K, N)")
    _on_gpu("quantize_block_weights", w=w)
    code = _code("quantize_block_weights", "w", w.dtype)
    wt = w.detach().transpose(-1, -2).contiguous()
    dev, lead, (N, K) = w.device, wt.shape[:-2], wt.shape[-2:]
    q = torch.empty(wt.shape, dtype=_E4M3, device=dev)
    scale = torch.empty((*lead, _blocks(N), _blocks(K)), dtype=torch.float32, device=dev)
    _call("es_quantize_block_weights", dev, wt.data_ptr(), code, math.prod(lead), N, K, q.data_ptr(),
          scale.data_ptr())
    return q, scale


def fp8_matmul(q: torch.Tensor, scale: torch.Tensor, wq: torch.Tensor, wscale: torch.Tensor,
               plan: ExpertPlan | None = None, gather: bool = False, out_dtype=torch.bfloat16) -> torch.Tensor:
    """Product of 8-bit floating-point numbers with block scales:
    ``y[r, n] = sum_b scale[r, b] * wscale[n // 128, b] * sum_{k in b} q[r, k] * wq[n, k]``
    over the blocks ``b`` of 128 of the depth, sums in fp32, rounded once.

    ``q`` e4m3 (rows, K) and ``scale`` float32 (rows, ceil(K / 128)) as from
    ``quantize_blocks``; ``wq`` e4m3 (N, K), ``wscale`` float32
    (ceil(N / 128), ceil(K / 128)). Scales may be any float32 numbers (where a
    row has a product of two scales of 2^36 or more, its terms below 2^-85 may
    be lost). With a
    ``plan`` the products are grouped by expert as in ``grouped_matmul``:
    ``wq`` and ``wscale`` have a leading num_experts, and with ``gather`` ``q``
    and ``scale`` are by token. Returns (rows, N) of ``out_dtype`` (float32,
    bfloat16, float16); rows of no expert are zero. Not differentiable: the
    result has no history."""
    if plan is not None and not isinstance(plan, ExpertPlan):
        raise TypeError(f"fp8_matmul: plan must be an ExpertPlan or None, got {type(plan).__name__}")
    if not _together(q, scale, wq, wscale, q if plan is None else plan.offsets):
        _on_gpu("fp8_matmul", q=q, scale=scale, wq=wq, wscale=wscale, plan=q if plan is None else plan.offsets)
    code = _code("fp8_matmul", "out_dtype", out_dtype)
    if q.dtype != _E4M3 or wq.dtype != _E4M3:
        raise TypeError(f"fp8_matmul: q and wq must be float8_e4m3fn, got {q.dtype} and {wq.dtype}")
    if scale.dtype != torch.float32 or wscale.dtype != torch.float32:
        raise TypeError(f"fp8_matmul: scale and wscale must be float32, got {scale.dtype} and {wscale.dtype}")
    lead = () if plan is None else (plan.num_experts,)
    if wq.dim() != 2 + len(lead) or wq.shape[:-2] != lead:
        raise ValueError(f"fp8_matmul: wq has shape {tuple(wq.shape)}, wanted "
                         + (f"({plan.num_experts}, N, K)" if lead else "(N, K)"))
    N, K = wq.shape[-2:]
    if wscale.shape != (*lead, _blocks(N), _blocks(K)):
        raise ValueError(f"fp8_matmul: wscale has shape {tuple(wscale.shape)}, wanted {(*lead, _blocks(N), _blocks(K))}")
    gather = bool(gather)
    if plan is not None:
        _check_rows("fp8_matmul", q, "q", plan, gather, K)
    elif gather or q.dim() != 2 or q.shape[1] != K:
        raise ValueError(f"fp8_matmul: q has shape {tuple(q.shape)}, wanted (rows, {K}); gather needs a plan")
    if scale.shape != (q.shape[0], _blocks(K)):
        raise ValueError(f"fp8_matmul: scale has shape {tuple(scale.shape)}, wanted {(q.shape[0], _blocks(K))}")
    q, scale, wscale = _rows(q), scale.contiguous(), wscale.contiguous()
    if wq.stride(-1) != 1 or wq.stride(-2) < K:
        wq = wq.contiguous()
    dev = q.device
    E, offsets, order, top_k, R = _groups(q, plan, gather)
    y = _empty(R, N, out_dtype, dev)
    args = (q.data_ptr(), scale.data_ptr(), q.shape[0], q.stride(0), wq.data_ptr(), wscale.data_ptr(), E, K, N,
            wq.stride(0) if E else 0, wq.stride(-2), offsets, order, top_k, R)
    _product("es_fp8_matmul", dev, args, (y.data_ptr(), code), gather)
    return y
