"""Mixture of experts: routing, products grouped by expert, the weighted sum back to tokens, 8-bit products.

A layer of experts is the contraction ``te,td,edf->tf`` with a token x expert
matrix of ``top_k`` nonzeros a row. Its blocks are ragged in the token axis,
so it runs beside the tile-COO path instead of on it:

* ``route_experts``: the chosen experts of each token and their weights;
* ``plan_experts``: the order that groups the choices by expert;
* ``grouped_matmul``: each group's rows times its expert's matrix;
* ``combine_experts``: the weighted sum of a token's rows;
* ``quantize_rows``, ``quantize_experts``, ``int8_matmul``: the serving form
  in 8-bit integers with a scale for each token and output channel;
* ``expert_mlp``: a gated layer made of these.

Gradients are reverse-mode; a forward-mode tangent is refused. All of it runs
on torch's current CUDA stream with no wait of the host. What
only the device can see (a choice of an expert that does not exist, a bounded
wait that ran out) is raised by ``check_device_errors``.
"""

from __future__ import annotations

import math

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib as L
from .sparse import _STATUS, _raw_stream

MAX_EXPERTS, MAX_TOP_K, MAX_INT8_DEPTH = 1024, 32, 131071

_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device

_DTYPES = {torch.float32: L.ES_F32, torch.bfloat16: L.ES_BF16, torch.float16: L.ES_F16}


def _code(fn: str, name: str, dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"{fn}: {name} must be float32, bfloat16 or float16, got {dtype}")
    return code


def _on_gpu(fn: str, **tensors):
    """Raises unless all are CUDA tensors of one device."""
    dev = None
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{fn}: {name} must be a torch tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise ValueError(f"{fn}: {name} must be a CUDA tensor")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"{fn}: {name} is on {t.device}, the other operands on {dev}")


def _no_tangent(fn: str, *tensors):
    """Raises where forward-mode differentiation is on for one of ``tensors``: the kernels would drop its tangent."""
    if _forward_ad._current_level >= 0 and any(_forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{fn}: no forward-mode derivative; gradients are reverse-mode only")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` (2-D) with a contiguous last dimension and rows that do not overlap."""
    if t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t
    return t.contiguous()


def _status(fn: str, dev, *args) -> int:
    """The entry point's answer on ``dev`` and its current stream (its last argument)."""
    index = dev.index
    here = _current_device()
    if here == index:
        return getattr(L.lib(), fn)(*args, _raw_stream(index))
    torch.cuda.set_device(index)
    try:
        return getattr(L.lib(), fn)(*args, _raw_stream(index))
    finally:
        torch.cuda.set_device(here)


def _call(fn: str, dev, *args):
    status = _status(fn, dev, *args)
    if status:
        L.check(fn, status)


def _product(fn: str, dev, args, outs, need: bool):
    """Calls ``fn(*args, *outs, workspace, its size, status word, stream)``. The
    workspace's size is asked for when the call surely takes one (``need``), or
    once the call has said so (operands that have to be laid out anew)."""
    word = _STATUS.address(fn, dev.index)
    if not need:
        status = _status(fn, dev, *args, *outs, None, 0, word)
        if status != L.ES_ERR_WORKSPACE:
            if status:
                L.check(fn, status)
            return
    nbytes = getattr(L.lib(), fn + "_workspace_size")(*args)
    ws = _scratch(nbytes, dev)
    _call(fn, dev, *args, *outs, _ptr(ws), nbytes, word)


def _empty(rows: int, cols: int, dtype, dev):
    """``torch.empty((rows, cols))``, which takes twice as long from a tuple."""
    return torch.empty_strided((rows, cols), (cols or 1, 1), dtype=dtype, device=dev)


def _scratch(nbytes: int, dev):
    """A workspace that is held until the call is queued (torch's allocator
    hands it out again only behind that on the stream), or None."""
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _ptr(t):
    return t.data_ptr() if t is not None else None


class ExpertPlan:
    """Row order of the routed choices, all int32 and contiguous on the device.

    Expert ``e`` owns rows ``offsets[e]`` to ``offsets[e + 1]``; row ``r``
    holds choice ``order[r]`` (``token * top_k + j``); ``position[token, j]``
    is the row of that choice. -1: no row, no choice. The rows from
    ``offsets[num_experts]`` on belong to no expert and are zero in every
    output. ``plan_experts`` makes one; so does a caller that has the three
    arrays (offsets that ascend from 0, ``position`` the inverse of ``order``)."""

    __slots__ = ("offsets", "order", "position", "device", "num_experts", "num_tokens", "top_k", "num_rows")

    def __init__(self, offsets: torch.Tensor, order: torch.Tensor, position: torch.Tensor):
        _on_gpu("ExpertPlan", offsets=offsets, order=order, position=position)
        i32 = torch.int32
        if offsets.dtype != i32 or order.dtype != i32 or position.dtype != i32:
            raise TypeError("ExpertPlan: offsets, order and position must be int32")
        if not (offsets.is_contiguous() and order.is_contiguous() and position.is_contiguous()):
            raise ValueError("ExpertPlan: offsets, order and position must be contiguous")
        E, R, P = offsets.shape, order.shape, position.shape
        if len(E) != 1 or len(R) != 1 or len(P) != 2 or E[0] < 2 or P[1] < 1 or P[0] * P[1] != R[0]:
            raise ValueError(f"ExpertPlan: shapes {tuple(E)}, {tuple(R)} and {tuple(P)} are not "
                             "(num_experts + 1,), (num_tokens * top_k,) and (num_tokens, top_k)")
        if E[0] - 1 > MAX_EXPERTS:
            raise ValueError(f"ExpertPlan: at most {MAX_EXPERTS} experts, got {E[0] - 1}")
        self._set(offsets, order, position)

    def _set(self, offsets, order, position):
        self.offsets, self.order, self.position = offsets, order, position
        self.device = offsets.device
        self.num_experts = offsets.shape[0] - 1
        self.num_tokens, self.top_k = position.shape
        self.num_rows = order.shape[0]
        return self

    @property
    def counts(self) -> torch.Tensor:
        """Rows of each expert, int32 (num_experts,)."""
        return self.offsets[1:] - self.offsets[:-1]


# ------------------------------------------------------------------- routing

def _route(logits, top_k, renormalize):
    dev = logits.device
    T, E = logits.shape
    weights = _empty(T, top_k, torch.float32, dev)
    experts = _empty(T, top_k, torch.int32, dev)
    _call("es_route_experts", dev, logits.data_ptr(), _DTYPES[logits.dtype], T, E, logits.stride(0), top_k,
          renormalize, weights.data_ptr(), experts.data_ptr())
    return weights, experts


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, renormalize):
        weights, experts = _route(logits, top_k, renormalize)
        ctx.mark_non_differentiable(experts)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, weights, experts)
        ctx.renormalize = renormalize
        return weights, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, _):
        if dweights is None:
            return None, None, None
        _no_tangent("route_experts", dweights)
        logits, weights, experts = ctx.saved_tensors
        dev = logits.device
        T, E = logits.shape
        dweights = dweights.contiguous()
        dlogits = _empty(T, E, logits.dtype, dev)
        _call("es_route_experts_grad", dev, logits.data_ptr(), _DTYPES[logits.dtype], T, E, logits.stride(0),
              experts.shape[1], ctx.renormalize, weights.data_ptr(), experts.data_ptr(), dweights.data_ptr(),
              dlogits.data_ptr())
        return dlogits, None, None


def route_experts(logits: torch.Tensor, top_k: int, renormalize: bool = True):
    """The ``top_k`` experts of each token and their softmax weights.

    ``logits`` (num_tokens, num_experts). Returns ``(weights, experts)``,
    float32 and int32 (num_tokens, top_k), largest logit first, ties to the
    lowest expert. The softmax runs over the chosen experts (``renormalize``)
    or over all of them. ``-inf`` masks an expert: it is never chosen, and a
    token with fewer than ``top_k`` experts left gets -1 with weight 0. The
    type's lowest finite value is a logit like any other. A NaN logit is never
    chosen and makes all weights of its token NaN. ``weights`` carries a
    gradient to ``logits``."""
    _on_gpu("route_experts", logits=logits)
    if logits.dim() != 2:
        raise ValueError(f"route_experts: logits must be (num_tokens, num_experts), got {tuple(logits.shape)}")
    _code("route_experts", "logits", logits.dtype)
    E, top_k = logits.shape[1], int(top_k)
    if not 1 <= top_k <= min(E, MAX_TOP_K) or E > MAX_EXPERTS:
        raise ValueError(f"route_experts: top_k={top_k} of {E} experts; 1 <= top_k <= min(num_experts, {MAX_TOP_K}) "
                         f"and num_experts <= {MAX_EXPERTS}")
    _no_tangent("route_experts", logits)
    run = _Route.apply if logits.requires_grad and torch.is_grad_enabled() else _route
    return run(_rows(logits), top_k, 1 if renormalize else 0)


def plan_experts(experts: torch.Tensor, num_experts: int) -> ExpertPlan:
    """Groups the choices ``experts`` (num_tokens, top_k; -1: none) by expert,
    in ascending token and choice inside an expert. An entry outside
    ``[-1, num_experts)`` counts as -1 and is raised as ``ValueError`` by the
    next ``check_device_errors``."""
    _on_gpu("plan_experts", experts=experts)
    if experts.dim() != 2 or experts.shape[1] < 1:
        raise ValueError(f"plan_experts: experts must be (num_tokens, top_k), got {tuple(experts.shape)}")
    if experts.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"plan_experts: experts must be int32 or int64, got {experts.dtype}")
    E = int(num_experts)
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"plan_experts: num_experts={E} is not in [1, {MAX_EXPERTS}]")
    if experts.dtype == torch.int64:  # a value past 32 bits must not wrap into the range
        experts = experts.clamp(-2, E).to(torch.int32)
    experts = experts.contiguous()
    dev, n = experts.device, experts.numel()
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    order = torch.empty(n, dtype=torch.int32, device=dev)
    position = torch.empty_like(experts)
    nbytes = L.lib().es_expert_plan_workspace_size(n, E)
    ws = _scratch(nbytes, dev)
    _call("es_expert_plan", dev, experts.data_ptr(), n, E, _ptr(ws), nbytes, offsets.data_ptr(), order.data_ptr(),
          position.data_ptr(), _STATUS.address("es_expert_plan", dev.index))
    return ExpertPlan.__new__(ExpertPlan)._set(offsets, order, position)


# ---------------------------------------------------------- grouped products

def _grouped(x, w, plan, gather, out_dtype):
    """``w`` (num_experts, K, N), any strides."""
    dev = x.device
    E, K, N = w.shape
    R, code = plan.num_rows, _DTYPES[x.dtype]
    y = _empty(R, N, out_dtype, dev)
    args = (x.data_ptr(), code, x.shape[0], x.stride(0), w.data_ptr(), E, K, N, *w.stride(), plan.offsets.data_ptr(),
            plan.order.data_ptr() if gather else None, plan.top_k, R)
    # fp32 mostly needs no workspace for up to 24 rows a group (12.8 us for 14.9 a small call)
    need = R > 24 * E if code == L.ES_F32 else gather
    _product("es_grouped_matmul", dev, args, (y.data_ptr(), _DTYPES[out_dtype]), need)
    return y


def _wgrad(x, dy, w, plan, gather):
    dev = x.device
    E, K, N = w.shape
    # the gradient takes w's layout when it is a transposed view
    dw = torch.empty((E, N, K), dtype=w.dtype, device=dev).transpose(1, 2) if w.stride(1) == 1 and w.stride(2) != 1 \
        else torch.empty((E, K, N), dtype=w.dtype, device=dev)
    R, code = plan.num_rows, _DTYPES[x.dtype]
    args = (x.data_ptr(), code, x.shape[0], x.stride(0), dy.data_ptr(), dy.stride(0), E, K, N, plan.offsets.data_ptr(),
            plan.order.data_ptr() if gather else None, plan.top_k, R, dw.data_ptr(), *dw.stride())
    _product("es_grouped_matmul_wgrad", dev, args, (), gather or code == L.ES_F32)
    return dw


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, plan, gather):
        ctx.save_for_backward(x, w)
        ctx.plan, ctx.gather = plan, gather
        return _grouped(x, w, plan, gather, x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        plan, gather = ctx.plan, ctx.gather
        _no_tangent("grouped_matmul", dy)
        dy = _rows(dy)
        dx = dw = None
        if ctx.needs_input_grad[0]:
            # a token's rows are summed before its gradient is rounded
            dx = _grouped(dy, w.transpose(1, 2), plan, False, torch.float32 if gather else x.dtype)
            if gather:
                dx = _combine(dx, None, plan, x.dtype)
        if ctx.needs_input_grad[1]:
            dw = _wgrad(x, dy, w, plan, gather)
        return dx, dw, None, None


def _check_rows(fn, x, name, plan, gather, K):
    want = plan.num_tokens if gather else plan.num_rows
    if x.dim() != 2 or x.shape[0] != want or (K is not None and x.shape[1] != K):
        raise ValueError(f"{fn}: {name} has shape {tuple(x.shape)}, the plan's {'tokens' if gather else 'rows'} and "
                         f"the weights want ({want}, {'...' if K is None else K})")


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, plan: ExpertPlan, gather: bool = False) -> torch.Tensor:
    """Each expert's rows times its matrix: ``y[r] = x[r] @ w[e]`` for the rows
    ``r`` of expert ``e``, ragged group sizes, sums in fp32, rounded once.

    ``w`` (num_experts, K, N) of x's type (float32, bfloat16, float16), with
    any strides (a transposed view is read as it lies). ``x``: (num_rows, K)
    in the plan's order, or with ``gather`` (num_tokens, K), where row ``r`` is
    the token of its choice. Returns (num_rows, N); rows of no expert are
    zero. Differentiable in ``x`` and ``w``."""
    if not isinstance(plan, ExpertPlan):
        raise TypeError(f"grouped_matmul: plan must be an ExpertPlan, got {type(plan).__name__}")
    _on_gpu("grouped_matmul", x=x, w=w, plan=plan.offsets)
    _code("grouped_matmul", "x", x.dtype)
    if w.dtype != x.dtype:
        raise TypeError(f"grouped_matmul: x is {x.dtype}, w is {w.dtype}")
    if w.dim() != 3 or w.shape[0] != plan.num_experts:
        raise ValueError(f"grouped_matmul: w has shape {tuple(w.shape)}, wanted ({plan.num_experts}, K, N)")
    _check_rows("grouped_matmul", x, "x", plan, gather, w.shape[1])
    _no_tangent("grouped_matmul", x, w)
    x, gather = _rows(x), bool(gather)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        return _GroupedMatmul.apply(x, w, plan, gather)
    return _grouped(x, w, plan, gather, x.dtype)


# ------------------------------------------------------ weighted sum to tokens

def _combine(y, weights, plan, out_dtype):
    dev, D = y.device, y.shape[1]
    out = _empty(plan.num_tokens, D, out_dtype, dev)
    _call("es_combine_experts", dev, y.data_ptr(), _DTYPES[y.dtype], y.shape[0], y.stride(0), _ptr(weights),
          plan.position.data_ptr(), plan.num_tokens, plan.top_k, D, out.data_ptr(), _DTYPES[out_dtype])
    return out


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, plan):
        ctx.save_for_backward(y, weights)
        ctx.plan = plan
        return _combine(y, weights, plan, y.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, weights = ctx.saved_tensors
        plan, dev = ctx.plan, y.device
        _no_tangent("combine_experts", dout)
        dout = _rows(dout)
        dy = _empty(*y.shape, y.dtype, dev)
        dweights = torch.empty_like(weights)
        _call("es_combine_experts_grad", dev, y.data_ptr(), _DTYPES[y.dtype], y.shape[0], y.stride(0),
              weights.data_ptr(), plan.position.data_ptr(), plan.offsets.data_ptr() + 4 * plan.num_experts,
              plan.num_tokens, plan.top_k, y.shape[1], dout.data_ptr(), dout.stride(0), dy.data_ptr(),
              dweights.data_ptr())
        return dy, dweights, None


def combine_experts(y: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * y[position[t, j]]``: the weighted sum
    of each token's rows of ``y`` (num_rows, width), in fp32, rounded once to
    y's type. ``weights`` float32 (num_tokens, top_k). A choice without a row
    adds nothing. Differentiable in ``y`` and ``weights``."""
    if not isinstance(plan, ExpertPlan):
        raise TypeError(f"combine_experts: plan must be an ExpertPlan, got {type(plan).__name__}")
    _on_gpu("combine_experts", y=y, weights=weights, plan=plan.offsets)
    _code("combine_experts", "y", y.dtype)
    if weights.dtype != torch.float32:
        raise TypeError(f"combine_experts: weights must be float32, got {weights.dtype}")
    _check_rows("combine_experts", y, "y", plan, False, None)
    if weights.shape != plan.position.shape:
        raise ValueError(f"combine_experts: weights have shape {tuple(weights.shape)}, the plan's choices "
                         f"{tuple(plan.position.shape)}")
    _no_tangent("combine_experts", y, weights)
    y, weights = _rows(y), weights.contiguous()
    if torch.is_grad_enabled() and (y.requires_grad or weights.requires_grad):
        return _Combine.apply(y, weights, plan)
    return _combine(y, weights, plan, y.dtype)


# ------------------------------------------------------------ 8-bit products

def quantize_rows(x: torch.Tensor):
    """``(q, scale)``: each row of ``x`` (rows, width) in 8-bit integers with
    ``scale = max |x| / 127`` (float32), ``q = rint(x / scale)``. A row of
    zeros has scale 0; a row with an infinity or NaN has scale NaN. Not
    differentiable: the result has no history."""
    _on_gpu("quantize_rows", x=x)
    code = _code("quantize_rows", "x", x.dtype)
    if x.dim() != 2:
        raise ValueError(f"quantize_rows: x must be (rows, width), got {tuple(x.shape)}")
    dev, x = x.device, _rows(x.detach())
    q = _empty(*x.shape, torch.int8, dev)
    scale = torch.empty(x.shape[0], dtype=torch.float32, device=dev)
    _call("es_quantize_rows", dev, x.data_ptr(), code, x.shape[0], x.shape[1], x.stride(0), q.data_ptr(),
          scale.data_ptr())
    return q, scale


def quantize_experts(w: torch.Tensor):
    """Weights ``w`` (..., K, N) as ``int8_matmul`` takes them: ``(wq, scale)``
    with ``wq`` int8 (..., N, K), contiguous along K, and a float32 scale for
    each output channel (..., N)."""
    if not isinstance(w, torch.Tensor) or w.dim() < 2:
        raise ValueError("quantize_experts: w must be a tensor (..., K, N)")
    wt = w.detach().transpose(-1, -2).contiguous()
    q, scale = quantize_rows(wt.reshape(math.prod(wt.shape[:-1]), wt.shape[-1]))
    return q.reshape(wt.shape), scale.reshape(wt.shape[:-1])


def int8_matmul(q: torch.Tensor, scale: torch.Tensor, wq: torch.Tensor, wscale: torch.Tensor,
                plan: ExpertPlan | None = None, gather: bool = False, out_dtype=torch.bfloat16) -> torch.Tensor:
    """Product of 8-bit integers with scales: ``y[r, n] = scale[r] *
    wscale[n] * sum_k q[r, k] * wq[n, k]``, the sum exact in 32-bit integers.

    ``q`` int8 (rows, K) and ``scale`` float32 (rows,) as from
    ``quantize_rows``; ``wq`` int8 (N, K), ``wscale`` float32 (N,). With a
    ``plan`` the products are grouped by expert as in ``grouped_matmul``:
    ``wq`` (num_experts, N, K), ``wscale`` (num_experts, N), and with
    ``gather`` ``q`` and ``scale`` are by token. Returns (rows, N) of
    ``out_dtype`` (float32, bfloat16, float16). K is at most 131,071. Not
    differentiable: the result has no history."""
    _on_gpu("int8_matmul", q=q, scale=scale, wq=wq, wscale=wscale, plan=q if plan is None else plan.offsets)
    code = _code("int8_matmul", "out_dtype", out_dtype)
    if q.dtype != torch.int8 or wq.dtype != torch.int8:
        raise TypeError(f"int8_matmul: q and wq must be int8, got {q.dtype} and {wq.dtype}")
    if scale.dtype != torch.float32 or wscale.dtype != torch.float32:
        raise TypeError(f"int8_matmul: scale and wscale must be float32, got {scale.dtype} and {wscale.dtype}")
    E = plan.num_experts if plan is not None else 0
    if wq.dim() != (3 if E else 2) or (E and wq.shape[0] != E) or wscale.shape != wq.shape[:-1]:
        raise ValueError(f"int8_matmul: wq {tuple(wq.shape)} and wscale {tuple(wscale.shape)} are not "
                         + (f"({E}, N, K) and ({E}, N)" if E else "(N, K) and (N,)"))
    N, K = wq.shape[-2], wq.shape[-1]
    if plan is not None:
        _check_rows("int8_matmul", q, "q", plan, gather, K)
    elif gather or q.dim() != 2 or q.shape[1] != K:
        raise ValueError(f"int8_matmul: q has shape {tuple(q.shape)}, wanted (rows, {K}); gather needs a plan")
    if scale.dim() != 1 or scale.shape[0] != q.shape[0]:
        raise ValueError(f"int8_matmul: scale has shape {tuple(scale.shape)}, wanted ({q.shape[0]},)")
    if K > MAX_INT8_DEPTH:
        raise ValueError(f"int8_matmul: K={K} is over {MAX_INT8_DEPTH}, where 32-bit sums can overflow")
    q, scale, wscale = _rows(q), scale.contiguous(), wscale.contiguous()
    if wq.stride(-1) != 1 or wq.stride(-2) < K:
        wq = wq.contiguous()
    dev = q.device
    R = plan.num_rows if plan is not None else q.shape[0]
    y = _empty(R, N, out_dtype, dev)
    args = (q.data_ptr(), scale.data_ptr(), q.shape[0], q.stride(0), wq.data_ptr(), wscale.data_ptr(), E, K, N,
            wq.stride(0) if E else 0, wq.stride(-2), plan.offsets.data_ptr() if E else None,
            plan.order.data_ptr() if gather else None, plan.top_k if E else 1, R)
    _product("es_int8_matmul", dev, args, (y.data_ptr(), code), gather)
    return y


# ----------------------------------------------------------- a layer of experts

class _Served(torch.autograd.Function):
    """The 8-bit layer's output. A gradient through it would hold the routing's share alone, so there is none."""

    @staticmethod
    def forward(ctx, out, x, router):
        return out.view_as(out)

    @staticmethod
    def backward(ctx, dout):
        raise RuntimeError("expert_mlp: the 8-bit form has no gradient; train with the weights' tensors")


def _layer(x, router, w_in, w_out, top_k, renormalize, quantized):
    weights, experts = route_experts(x.float() @ router.float(), top_k, renormalize)
    plan = plan_experts(experts, router.shape[1])
    if quantized:
        h = int8_matmul(*quantize_rows(x), *w_in, plan, gather=True, out_dtype=x.dtype)
    else:
        h = grouped_matmul(x, w_in, plan, gather=True)
    gate, up = h.chunk(2, dim=1)
    h = torch.nn.functional.silu(gate) * up
    y = int8_matmul(*quantize_rows(h), *w_out, plan, out_dtype=x.dtype) if quantized else \
        grouped_matmul(h, w_out, plan)
    return combine_experts(y, weights, plan)


def expert_mlp(x: torch.Tensor, router: torch.Tensor, w_in, w_out, top_k: int, renormalize: bool = True):
    """A gated layer of experts: for each token ``x`` (num_tokens, D) the
    weighted sum, over its ``top_k`` experts ``e``, of
    ``(silu(x @ gate_e) * (x @ up_e)) @ w_out_e``.

    ``router`` (D, num_experts). ``w_in`` (num_experts, D, 2 F) holds gate and
    up side by side, ``w_out`` (num_experts, F, D): tensors of x's type for
    training (differentiable in everything), or both ``(wq, scale)`` pairs
    of ``quantize_experts`` for serving in 8-bit integers, where a gradient
    through the result raises."""
    quantized = isinstance(w_in, (tuple, list))
    if quantized != isinstance(w_out, (tuple, list)):
        raise TypeError("expert_mlp: w_in and w_out must both be tensors or both be (wq, scale) pairs")
    if not quantized:
        return _layer(x, router, w_in, w_out, top_k, renormalize, False)
    with torch.no_grad():
        out = _layer(x, router, w_in, w_out, top_k, renormalize, True)
    if torch.is_grad_enabled() and (x.requires_grad or router.requires_grad):
        return _Served.apply(out, x, router)
    return out
