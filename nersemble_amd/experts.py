"""Routed experts: every row (a sample, a token) goes to ``top_k`` of E experts.

    weights, chosen = route_experts(logits, top_k)            # which experts, with what weight
    plan = expert_plan(chosen, n_experts)                     # the (row, choice) entries in the experts' order
    h = expert_linear(x, w1, plan, gather=True, relu=True)    # [T * top_k, n] in that order
    y = expert_linear(h, w2, plan, gather=False)
    out = expert_combine(y, weights, plan)                    # [T, n]

(The reference's only mixture is the dense blend of all hash grids, hash_ensemble.py:133-156; ``tcnn.RoutedNetwork`` is the
module built on these calls.)  All four launch on torch's current stream, keep nothing between calls, never read the device from the host and can be captured into a graph.  Under
``_lib.device_count`` rows behind the device-side count are not routed, and not written by ``route_experts`` and
``expert_combine``.  A plan's numbers are bounded inside the kernels; equal inputs give equal bits.
"""
import ctypes as C
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check, lib, ndev, ptr, stream

_DTYPE = {torch.float32: _lib.NSX_DTYPE_F32, torch.float16: _lib.NSX_DTYPE_F16, torch.bfloat16: _lib.NSX_DTYPE_BF16}
_SCORES = {"softmax": 0, "sigmoid": 1}


@dataclass(frozen=True)
class ExpertPlan:
    """Entries (row * top_k + choice) ordered by expert (``expert_plan``): int32 device tensors.

    offsets [E + 1]: the ordered rows of expert e are offsets[e] .. offsets[e + 1]; rows [T * top_k]: entry of every ordered
    row, -1 behind the last segment; positions [T, top_k]: ordered row of every entry, -1 for an entry that is not routed."""
    offsets: torch.Tensor
    rows: torch.Tensor
    positions: torch.Tensor

    @property
    def n_experts(self) -> int:
        return self.offsets.shape[0] - 1

    @property
    def top_k(self) -> int:
        return self.positions.shape[1]


def _plan_check(plan: ExpertPlan, what: str) -> None:
    o, r, p = plan.offsets, plan.rows, plan.positions
    if o.dim() != 1 or o.shape[0] < 2 or r.dim() != 1 or p.dim() != 2 or p.numel() != r.shape[0]:
        raise RuntimeError(f"{what}: the plan's offsets [E + 1], rows [T * top_k], positions [T, top_k] have shapes "
                           f"{tuple(o.shape)}, {tuple(r.shape)}, {tuple(p.shape)}")


def _rows_of(t: torch.Tensor, align: int) -> Tuple[torch.Tensor, int]:
    """``t`` as rows of consecutive values whose distance is a multiple of ``align`` elements (and which start on 16 bytes if
    ``align`` > 1), and that distance; copied where it is laid out otherwise."""
    n, w = t.shape
    s = t.stride(0) if n > 1 else -(-w // align) * align
    if (w > 1 and t.stride(1) != 1) or s < w or s % align or (align > 1 and (t.data_ptr() % 16 or s > _lib.NSX_MAX_EXPERT_STRIDE)):
        t, s = t.contiguous(), w
        if align > 1 and t.data_ptr() % 16:
            t = t.clone()
    return t, s


def _at(t: torch.Tensor) -> C.c_void_p:
    """``ptr`` for rows that need not lie next to each other."""
    if t.is_contiguous():
        return ptr(t)
    ptr(t[:1, :1])                   # (device checks)
    return C.c_void_p(t.data_ptr())


# ------------------------------------------------------------------------------------------------
# choice
# ------------------------------------------------------------------------------------------------
def _route(logits, stride, bias, selector, top_k, sigmoid, n_groups, top_groups, group_top, renorm, scale):
    T, E = logits.shape
    weights = torch.empty((T, top_k), dtype=torch.float32, device=logits.device)
    chosen = torch.empty((T, top_k), dtype=torch.int32, device=logits.device)
    check(lib().nsx_expert_route_fwd(_at(logits), _DTYPE[logits.dtype], T, E, stride, ptr(bias, torch.float32),
                                     ptr(selector, torch.uint8), top_k, sigmoid, n_groups, top_groups, group_top, renorm, scale,
                                     ptr(weights), ptr(chosen), ndev(T), stream()), "nsx_expert_route_fwd")
    return weights, chosen


class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, selector, cfg):
        x, stride = _rows_of(logits.detach(), 1)
        weights, chosen = _route(x, stride, bias, selector, *cfg)
        ctx.save_for_backward(x, weights, chosen)
        ctx.cfg, ctx.stride = cfg, stride
        ctx.mark_non_differentiable(chosen)
        ctx.set_materialize_grads(False)
        return weights, chosen

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return None, None, None, None
        x, weights, chosen = ctx.saved_tensors
        top_k, sigmoid, _, _, _, renorm, scale = ctx.cfg
        T, E = x.shape
        g = g.to(torch.float32).contiguous()
        d = torch.empty((T, E), dtype=x.dtype, device=x.device)
        check(lib().nsx_expert_route_bwd(_at(x), _DTYPE[x.dtype], T, E, ctx.stride, top_k, sigmoid, renorm, scale, ptr(weights),
                                         ptr(chosen), ptr(g), ptr(d), ndev(T), stream()), "nsx_expert_route_bwd")
        return d, None, None, None


def route_experts(logits: torch.Tensor, top_k: int, scores: str = "softmax", bias: Optional[torch.Tensor] = None,
                  n_groups: int = 1, top_groups: Optional[int] = None, group_top: int = 1, renormalise: bool = True,
                  scale: float = 1.0, selector: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Choice of ``top_k`` experts for every row of ``logits`` [T, E] (fp32, fp16 or bf16): (weights [T, top_k] fp32, chosen
    [T, top_k] int32), differentiable w.r.t. ``logits``.

    The choice goes by the scores ("softmax" over the experts or "sigmoid") plus ``bias`` [E] fp32 (which balances the load and
    has no part in the weights); equal values go by rising index.  ``n_groups`` > 1: only the ``top_groups`` groups of
    consecutive experts with the largest sum of their ``group_top`` (1 or 2) best take part.  ``renormalise``: the weights are
    the chosen scores over their sum; times ``scale``.  A logit of -inf takes the expert out for its row.  ``selector`` uint8
    [T]: rows with 0 are not routed.  Where there is no expert to choose: chosen -1, weight 0.  A row with a NaN logit has NaN
    weights."""
    if logits.dim() != 2 or logits.dtype not in _DTYPE:
        raise RuntimeError(f"route_experts: logits are [T, E] in fp32, fp16 or bf16 (got {tuple(logits.shape)} {logits.dtype})")
    if scores not in _SCORES:
        raise RuntimeError(f"route_experts: scores are 'softmax' or 'sigmoid' (got {scores!r})")
    T, E = logits.shape
    if bias is not None:
        if bias.shape != (E,):
            raise RuntimeError(f"route_experts: bias has shape {tuple(bias.shape)}, not ({E},)")
        bias = bias.detach().contiguous()
    if selector is not None:
        if selector.numel() != T:
            raise RuntimeError(f"route_experts: selector has {selector.numel()} entries for {T} rows")
        selector = selector.detach().reshape(-1).contiguous()
        if selector.dtype == torch.bool:
            selector = selector.view(torch.uint8)
    cfg = (int(top_k), _SCORES[scores], int(n_groups), int(n_groups if top_groups is None else top_groups), int(group_top),
           int(bool(renormalise)), float(scale))
    if logits.requires_grad and torch.is_grad_enabled():
        return _RouteFn.apply(logits, bias, selector, cfg)
    x, stride = _rows_of(logits.detach(), 1)
    return _route(x, stride, bias, selector, *cfg)


# ------------------------------------------------------------------------------------------------
# plan
# ------------------------------------------------------------------------------------------------
def expert_plan(chosen: torch.Tensor, n_experts: int) -> ExpertPlan:
    """The plan of ``chosen`` [T, top_k] int32 (``route_experts``): a stable sort of its entries by expert.  Entries outside
    [0, n_experts) are not routed."""
    if chosen.dim() != 2 or chosen.dtype != torch.int32:
        raise RuntimeError(f"expert_plan: chosen is [T, top_k] int32 (got {tuple(chosen.shape)} {chosen.dtype})")
    chosen = chosen.contiguous()
    T, k = chosen.shape
    dev, n_experts = chosen.device, int(n_experts)
    need = int(lib().nsx_expert_plan_workspace(T * k, n_experts))
    if need < 0:
        check(need, "nsx_expert_plan_workspace")
    # one allocation: offsets | rows | positions | workspace (16-byte steps)
    o, r = -(-(n_experts + 1) // 4) * 4, -(-(T * k) // 4) * 4
    buf = torch.empty((o + 2 * r + need // 4,), dtype=torch.int32, device=dev)
    plan = ExpertPlan(buf[:n_experts + 1], buf[o:o + T * k], buf[o + r:o + r + T * k].view(T, k))
    check(lib().nsx_expert_plan(ptr(chosen), T, k, n_experts, ptr(plan.offsets), ptr(plan.rows), ptr(plan.positions),
                                ptr(buf[o + 2 * r:]), ndev(T), stream()), "nsx_expert_plan")
    return plan


# ------------------------------------------------------------------------------------------------
# products
# ------------------------------------------------------------------------------------------------
def _linear(x, x_stride, w16, plan, gather, relu):
    E, N, K = w16.shape
    R = plan.rows.shape[0]
    y = torch.empty((R, N), dtype=x.dtype, device=x.device)
    check(lib().nsx_expert_linear_fwd(_at(x), _DTYPE[x.dtype], x_stride, x.shape[0],
                                      ptr(plan.rows, torch.int32) if gather else None, plan.top_k, ptr(w16), K, N, E,
                                      ptr(plan.offsets, torch.int32), R, int(relu), ptr(y), stream()), "nsx_expert_linear_fwd")
    return y


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, w16, plan, gather, relu):
        xr, x_stride = _rows_of(x.detach(), 8)
        y = _linear(xr, x_stride, w16, plan, gather, relu)
        need_x, need_w = ctx.needs_input_grad[:2]
        ctx.save_for_backward(xr if need_w else None, w16 if need_x else None, y if relu else None,
                              plan.offsets, plan.rows, plan.positions)
        ctx.cfg = (x_stride, tuple(x.shape), tuple(w16.shape), gather, weight.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w16, y, offsets, rows, positions = ctx.saved_tensors
        x_stride, x_shape, (E, N, K), gather, w_dtype = ctx.cfg
        plan = ExpertPlan(offsets, rows, positions)
        R, code, dev = rows.shape[0], _DTYPE[dy.dtype], dy.device
        g, g_stride = _rows_of(dy, 8)
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = torch.empty((R, K), dtype=g.dtype, device=dev)
            check(lib().nsx_expert_linear_bwd_x(_at(g), code, g_stride, ptr(y), N, ptr(w16), K, N, E, ptr(offsets), R, ptr(dx),
                                                stream()), "nsx_expert_linear_bwd_x")
            if gather:
                # a row's choices summed in 32 bits; their gradients lie in 16 bits between the two launches (twice the
                # memory traffic otherwise): an error of at most half a step of each term beside the sum's own rounding
                dx = _combine(dx, K, None, positions)
        if ctx.needs_input_grad[1]:
            need = int(lib().nsx_expert_linear_bwd_w_workspace(R, E, K, N))
            if need < 0:
                check(need, "nsx_expert_linear_bwd_w_workspace")
            ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
            dw = torch.empty((E, N, K), dtype=w_dtype, device=dev)
            check(lib().nsx_expert_linear_bwd_w(_at(x), code, x_stride, x_shape[0], ptr(rows) if gather else None, plan.top_k,
                                                _at(g), g_stride, ptr(y), N, K, N, E, ptr(offsets), R,
                                                int(w_dtype == torch.float32), ptr(dw), ptr(ws), stream()),
                  "nsx_expert_linear_bwd_w")
        return dx, dw, None, None, None, None


def expert_linear(x: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan, gather: bool = True, relu: bool = False,
                  w16: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[T * top_k, n_out] in the plan's order: ordered row p of expert e is ``weight[e] @ x[row of p]`` (``relu``: its positive
    part), differentiable w.r.t. ``x`` and ``weight``; ordered rows behind the last segment are 0.

    x: fp16 or bf16, [T, n_in] rows (``gather``) or [T * top_k, n_in] in the plan's order.  weight [E, n_out, n_in]: of x's
    dtype, or fp32 parameters whose copy in x's dtype is ``w16`` (made here if it is not given); the gradient has the dtype of
    ``weight``.  n_in and n_out are multiples of 8."""
    _plan_check(plan, "expert_linear")
    if x.dim() != 2 or x.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"expert_linear: x is [rows, n_in] in fp16 or bf16 (got {tuple(x.shape)} {x.dtype})")
    if weight.dim() != 3 or weight.dtype not in (x.dtype, torch.float32):
        raise RuntimeError(f"expert_linear: weight is [E, n_out, n_in] in {x.dtype} or fp32 (got {tuple(weight.shape)} {weight.dtype})")
    E, N, K = weight.shape
    if E != plan.n_experts or x.shape[1] != K:
        raise RuntimeError(f"expert_linear: weight {tuple(weight.shape)} for rows of {x.shape[1]} and a plan of {plan.n_experts} experts")
    if x.shape[0] != (plan.positions.shape[0] if gather else plan.rows.shape[0]):
        raise RuntimeError(f"expert_linear: x has {x.shape[0]} rows for a plan of {tuple(plan.positions.shape)} entries "
                           f"(gather={bool(gather)})")
    if w16 is None:
        w16 = weight.detach() if weight.dtype == x.dtype else weight.detach().to(x.dtype)
    elif w16.shape != weight.shape or w16.dtype != x.dtype:
        raise RuntimeError(f"expert_linear: w16 is {tuple(w16.shape)} {w16.dtype}, not {tuple(weight.shape)} {x.dtype}")
    w16 = w16.detach().contiguous()
    if w16.data_ptr() % 16:
        w16 = w16.clone()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _LinearFn.apply(x, weight, w16, plan, bool(gather), bool(relu))
    xr, x_stride = _rows_of(x.detach(), 8)
    return _linear(xr, x_stride, w16, plan, bool(gather), bool(relu))


# ------------------------------------------------------------------------------------------------
# join
# ------------------------------------------------------------------------------------------------
def _combine(y, y_stride, weights, positions):
    T, k = positions.shape
    out = torch.empty((T, y.shape[1]), dtype=y.dtype, device=y.device)
    check(lib().nsx_expert_combine_fwd(_at(y), _DTYPE[y.dtype], y_stride, y.shape[0], y.shape[1], ptr(weights),
                                       ptr(positions, torch.int32), T, k, ptr(out), ndev(T), stream()), "nsx_expert_combine_fwd")
    return out


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, plan):
        yr, stride = _rows_of(y.detach(), 8)
        w = weights.detach().to(torch.float32).contiguous()
        ctx.save_for_backward(yr, w, plan.offsets, plan.positions)
        ctx.stride, ctx.w_dtype = stride, weights.dtype
        return _combine(yr, stride, w, plan.positions)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        y, w, offsets, positions = ctx.saved_tensors
        T, k = positions.shape
        R, n = y.shape
        dout = dout.contiguous()
        if dout.data_ptr() % 16:
            dout = dout.clone()
        dy = torch.empty((R, n), dtype=y.dtype, device=y.device)
        dw = torch.empty((T, k), dtype=torch.float32, device=y.device)
        check(lib().nsx_expert_combine_bwd(_at(y), _DTYPE[y.dtype], ctx.stride, R, n, ptr(w), ptr(positions), ptr(offsets[-1:]), T, k,
                                           ptr(dout), ptr(dy), ptr(dw), ndev(T), stream()), "nsx_expert_combine_bwd")
        return dy, dw.to(ctx.w_dtype), None


def expert_combine(y: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """[T, n]: sum over a row's choices of ``weights[t, j] * y[plan.positions[t, j]]``, differentiable w.r.t. ``y`` [T * top_k,
    n] (fp16 or bf16, n a multiple of 8) and ``weights`` [T, top_k]; choices that are not routed count nothing."""
    _plan_check(plan, "expert_combine")
    if y.dim() != 2 or y.dtype not in (torch.float16, torch.bfloat16) or y.shape[0] != plan.rows.shape[0]:
        raise RuntimeError(f"expert_combine: y is [{plan.rows.shape[0]}, n] in fp16 or bf16 (got {tuple(y.shape)} {y.dtype})")
    if weights.shape != plan.positions.shape or not weights.is_floating_point():
        raise RuntimeError(f"expert_combine: weights are {tuple(plan.positions.shape)} (got {tuple(weights.shape)} {weights.dtype})")
    if torch.is_grad_enabled() and (y.requires_grad or weights.requires_grad):
        return _CombineFn.apply(y, weights, plan)
    yr, stride = _rows_of(y.detach(), 8)
    return _combine(yr, stride, weights.detach().to(torch.float32).contiguous(), plan.positions)
