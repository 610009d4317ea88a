"""Routed experts: every row (a sample, a token) goes to ``top_k`` of E experts.

    weights, chosen = route_experts(logits, top_k)            # which experts, with what weight
    plan = expert_plan(chosen, n_experts)                     # the (row, choice) entries in the experts' order
    h = expert_linear(x, w1, plan, gather=True, relu=True)    # [T * top_k, n] in that order
    y = expert_linear(h, w2, plan, gather=False)
    out = expert_combine(y, weights, plan)                    # [T, n]

(The reference's only mixture is the dense blend of all hash grids, hash_ensemble.py:133-156; ``tcnn.RoutedNetwork`` is the
module built on these calls.)  All four launch on torch's current stream, keep nothing between calls, never read the device from
the host and can be captured into a graph.  Under
``_lib.device_count`` rows behind the device-side count are not routed, and not written by ``route_experts`` and
``expert_combine``.  A plan's numbers are bounded inside the kernels; equal inputs give equal bits.
"""
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check, lib, ndev, ptr

_DTYPE = {torch.float32: _lib.NSX_DTYPE_F32, torch.float16: _lib.NSX_DTYPE_F16, torch.bfloat16: _lib.NSX_DTYPE_BF16}
_SCORES = {"softmax": 0, "sigmoid": 1}
_F32, _I32 = torch.float32, torch.int32
_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_profiler = _lib.profiler


class _FastNotLoaded:
    """csrc/experts_torch.cpp before its first call."""

    def __getattr__(self, name):
        global _fast
        version = lib().nsx_version()
        try:
            from .csrc import _experts
        except ImportError as e:
            raise RuntimeError(f"nersemble_amd: the native binding csrc/_experts.so cannot be loaded ({e}). Build it with "
                               f"`python -c 'import __graft_entry__ as g; g.build()'`.") from e
        if _experts.nsx_version != version or _experts.torch_version != torch.__version__:
            raise RuntimeError(f"nersemble_amd: csrc/_experts.so was built against libnsx.so {_experts.nsx_version} and torch "
                               f"{_experts.torch_version}, not {version} and {torch.__version__}. Build it again with "
                               f"`python -c 'import __graft_entry__ as g; g.build()'`.")
        _fast = _experts
        return getattr(_fast, name)


# The calls whose arguments are plain (contiguous rows on the current device, no row count on the device, nobody profiling) run
# natively from end to end; every other goes through the Functions below, which copy, refuse and record what there is.
_fast = _FastNotLoaded()


class ExpertPlan:
    """Entries (row * top_k + choice) ordered by expert (``expert_plan``): int32 device tensors.

    offsets [E + 1]: the ordered rows of expert e are offsets[e] .. offsets[e + 1]; rows [T * top_k]: entry of every ordered
    row, -1 behind the last segment; positions [T, top_k]: ordered row of every entry, -1 for an entry that is not routed."""
    __slots__ = ("_offsets", "_rows", "_positions", "n_experts", "n_rows", "top_k", "n_entries", "device")
    offsets = property(lambda self: self._offsets)
    rows = property(lambda self: self._rows)
    positions = property(lambda self: self._positions)

    def __init__(self, offsets: torch.Tensor, rows: torch.Tensor, positions: torch.Tensor):
        o, r, p = offsets.shape, rows.shape, positions.shape
        if len(o) != 1 or o[0] < 2 or len(r) != 1 or len(p) != 2 or p[0] * p[1] != r[0] \
                or not offsets.dtype == rows.dtype == positions.dtype == _I32:
            raise RuntimeError(f"ExpertPlan: offsets [E + 1], rows [T * top_k] and positions [T, top_k] are int32 (got {tuple(o)} "
                               f"{offsets.dtype}, {tuple(r)} {rows.dtype}, {tuple(p)} {positions.dtype})")
        self.device = offsets.get_device()
        if not self.device == rows.get_device() == positions.get_device():
            raise RuntimeError(f"ExpertPlan: offsets, rows and positions are on {offsets.device}, {rows.device} and {positions.device}")
        if not (offsets.is_contiguous() and rows.is_contiguous() and positions.is_contiguous()):
            offsets, rows, positions = offsets.contiguous(), rows.contiguous(), positions.contiguous()
        self._offsets, self._rows, self._positions = offsets, rows, positions
        self.n_experts, self.n_entries = o[0] - 1, r[0]
        self.n_rows, self.top_k = p

    def _version(self):
        return self.offsets._version + self.rows._version + self.positions._version


def _plan_of(ctx) -> ExpertPlan:
    """The plan of a forward pass, which has to be as it was then."""
    plan, version = ctx.plan
    if plan._version() != version:
        raise RuntimeError("the plan that the forward pass used has been modified by an inplace operation")
    return plan


def _rows_of(t: torch.Tensor, align: int) -> Tuple[torch.Tensor, int]:
    """``t`` as rows of consecutive values whose distance is a multiple of ``align`` elements (and which start on 16 bytes if
    ``align`` > 1), and that distance; copied where it is laid out otherwise."""
    n, w = t.shape
    if t.is_contiguous() and w % align == 0 and (align == 1 or t.data_ptr() % 16 == 0):
        return t, w
    s = t.stride(0) if n > 1 else -(-w // align) * align
    if (w > 1 and t.stride(1) != 1) or s < w or s % align or (align > 1 and (t.data_ptr() % 16 or s > _lib.NSX_MAX_EXPERT_STRIDE)):
        t, s = t.contiguous(), w
        if align > 1 and t.data_ptr() % 16:
            t = t.clone()
    return t, s


def _here(t: torch.Tensor) -> int:
    """The current device, which has to be ``t``'s."""
    d = t.get_device()
    if d < 0 or d != _device():
        ptr(t)
    return d


def _at(t: torch.Tensor, dev: int) -> int:
    """Address of a tensor of the current device (``ptr`` says what is wrong with any other)."""
    if t.get_device() != dev:
        ptr(t)
    return t.data_ptr()


def _no_tangent(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Dual tensors (forward mode) have no ``requires_grad``: without this their tangents would be lost silently."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name}: forward-mode derivatives are not implemented")


# ------------------------------------------------------------------------------------------------
# choice
# ------------------------------------------------------------------------------------------------
def _route(x, stride, bias, selector, top_k, sigmoid, n_groups, top_groups, group_top, renorm, scale):
    T, E = x.shape
    dev = _here(x)
    weights = x.new_empty((T, top_k), dtype=_F32)
    chosen = x.new_empty((T, top_k), dtype=_I32)
    rc = lib().nsx_expert_route_fwd(x.data_ptr(), _DTYPE[x.dtype], T, E, stride, None if bias is None else _at(bias, dev),
                                    None if selector is None else _at(selector, dev), top_k, sigmoid, n_groups, top_groups, group_top,
                                    renorm, scale, weights.data_ptr(), chosen.data_ptr(),
                                    None if _lib._COUNT_SCOPE is None else ndev(T), _raw_stream(dev))
    if rc:
        check(rc, "nsx_expert_route_fwd")
    return weights, chosen


def _route_bwd(ctx, g, _):
    if g is None:
        return None, None, None, None
    x, weights, chosen = ctx.saved_tensors
    stride, top_k, sigmoid, renorm, scale = ctx.cfg
    T, E = x.shape
    if g.dtype != _F32 or not g.is_contiguous():
        g = g.to(_F32).contiguous()
    dev = x.get_device()
    d = torch.empty_like(x) if stride == E else x.new_empty((T, E))
    rc = lib().nsx_expert_route_bwd(x.data_ptr(), _DTYPE[x.dtype], T, E, stride, top_k, sigmoid, renorm, scale, weights.data_ptr(),
                                    chosen.data_ptr(), g.data_ptr(), d.data_ptr(),
                                    None if _lib._COUNT_SCOPE is None else ndev(T), _raw_stream(dev))
    if rc:
        check(rc, "nsx_expert_route_bwd")
    return d, None, None, None


class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, selector, cfg):
        x, stride = _rows_of(logits, 1)
        weights, chosen = _route(x, stride, bias, selector, *cfg)
        ctx.save_for_backward(x, weights, chosen)
        ctx.cfg = (stride, cfg[0], cfg[1], cfg[5], cfg[6])
        ctx.mark_non_differentiable(chosen)
        ctx.set_materialize_grads(False)
        return weights, chosen

    @staticmethod
    def backward(ctx, g, _):
        return (_route_bwd_once if torch.is_grad_enabled() else _route_bwd)(ctx, g, _)


_route_bwd_once = once_differentiable(_route_bwd)        # (under create_graph: a second differentiation raises)


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
    sigmoid = _SCORES.get(scores)
    groups = n_groups if top_groups is None else top_groups
    if sigmoid is not None and _lib._COUNT_SCOPE is None and not _profiler.enabled:
        out = _fast.route_experts(logits, int(top_k), sigmoid, bias, selector, int(n_groups), int(groups), int(group_top),
                                  int(bool(renormalise)), float(scale))
        if out is not None:
            return out
    _no_tangent("route_experts", logits)
    if logits.dim() != 2 or logits.dtype not in _DTYPE:
        raise RuntimeError(f"route_experts: logits are [T, E] in fp32, fp16 or bf16 (got {tuple(logits.shape)} {logits.dtype})")
    if sigmoid is None:
        raise RuntimeError(f"route_experts: scores are 'softmax' or 'sigmoid' (got {scores!r})")
    T, E = logits.shape
    if not 1 <= E <= _lib.NSX_MAX_EXPERTS:
        raise RuntimeError(f"route_experts: n_experts {E} not in [1,{_lib.NSX_MAX_EXPERTS}]")
    if not 1 <= int(top_k) <= min(E, _lib.NSX_MAX_TOP_K):
        raise RuntimeError(f"route_experts: top_k {top_k} not in [1,{_lib.NSX_MAX_TOP_K}] or more than the {E} experts")
    if bias is not None:
        if bias.shape != (E,) or bias.dtype != _F32:
            raise RuntimeError(f"route_experts: bias is {tuple(bias.shape)} {bias.dtype}, not ({E},) fp32")
        if bias.requires_grad or not bias.is_contiguous():
            bias = bias.detach().contiguous()
    if selector is not None:
        if selector.numel() != T:
            raise RuntimeError(f"route_experts: selector has {selector.numel()} entries for {T} rows")
        selector = selector.reshape(-1).contiguous()
        if selector.dtype == torch.bool:
            selector = selector.view(torch.uint8)
        if selector.dtype != torch.uint8:
            raise RuntimeError(f"route_experts: selector is uint8 or bool (got {selector.dtype})")
    cfg = (int(top_k), sigmoid, int(n_groups), int(groups), int(group_top), int(bool(renormalise)), float(scale))
    if logits.requires_grad and torch.is_grad_enabled():
        return _RouteFn.apply(logits, bias, selector, cfg)
    x, stride = _rows_of(logits, 1)
    return _route(x, stride, bias, selector, *cfg)


# ------------------------------------------------------------------------------------------------
# plan
# ------------------------------------------------------------------------------------------------
def _plan_bytes(n_entries, n_experts):
    n = lib().nsx_expert_plan_workspace(n_entries, n_experts)
    if n < 0:
        check(n, "nsx_expert_plan_workspace")
    return n


def expert_plan(chosen: torch.Tensor, n_experts: int) -> ExpertPlan:
    """The plan of ``chosen`` [T, top_k] int32 (``route_experts``): a stable sort of its entries by expert.  Entries outside
    [0, n_experts) are not routed."""
    if _lib._COUNT_SCOPE is None and not _profiler.enabled:
        out = _fast.plan(chosen, int(n_experts))
        if out is not None:
            plan = ExpertPlan.__new__(ExpertPlan)
            plan._offsets, plan._rows, plan._positions = out
            plan.n_rows, plan.top_k = chosen.shape
            plan.n_experts, plan.n_entries, plan.device = int(n_experts), plan.n_rows * plan.top_k, chosen.get_device()
            return plan
    if chosen.dim() != 2 or chosen.dtype != torch.int32:
        raise RuntimeError(f"expert_plan: chosen is [T, top_k] int32 (got {tuple(chosen.shape)} {chosen.dtype})")
    chosen = chosen.contiguous()
    T, k = chosen.shape
    n_experts = int(n_experts)
    need = _plan_bytes(T * k, n_experts)
    # one allocation: offsets | rows | positions | workspace (16-byte steps)
    o, r = -(-(n_experts + 1) // 4) * 4, -(-(T * k) // 4) * 4
    dev = _here(chosen)
    buf = chosen.new_empty((o + 2 * r + need // 4,))
    base = buf.data_ptr()
    rc = lib().nsx_expert_plan(chosen.data_ptr(), T, k, n_experts, base, base + 4 * o, base + 4 * (o + r), base + 4 * (o + 2 * r),
                                   None if _lib._COUNT_SCOPE is None else ndev(T), _raw_stream(dev))
    if rc:
        check(rc, "nsx_expert_plan")
    return ExpertPlan(buf[:n_experts + 1], buf[o:o + T * k], buf[o + r:o + r + T * k].view(T, k))


# ------------------------------------------------------------------------------------------------
# products
# ------------------------------------------------------------------------------------------------
def _linear(x, x_stride, w16, plan, gather, relu):
    E, N, K = w16.shape
    dev = _here(x)
    if w16.get_device() != dev or plan.device != dev:
        ptr(w16), ptr(plan.offsets)
    n = plan.n_entries
    y = x.new_empty((n, N))
    rc = lib().nsx_expert_linear_fwd(x.data_ptr(), _DTYPE[x.dtype], x_stride, x.shape[0], plan.rows.data_ptr() if gather else None,
                                     plan.top_k, w16.data_ptr(), K, N, E, plan.offsets.data_ptr(), n, relu, y.data_ptr(),
                                     _raw_stream(dev))
    if rc:
        check(rc, "nsx_expert_linear_fwd")
    return y


def _linear_bwd_bytes(R, E, K, N, need_x, choices, need_w, masked):
    n = lib().nsx_expert_linear_bwd_workspace(R, E, K, N, need_x, choices, need_w, masked)
    if n < 0:
        check(n, "nsx_expert_linear_bwd_workspace")
    return n


def _linear_bwd(ctx, dy):
    x, w16, y = ctx.saved_tensors
    x_stride, x_rows, (E, N, K), gather, w_dtype, need_x, need_w = ctx.cfg
    plan = _plan_of(ctx)
    R = plan.n_entries
    if dy.is_contiguous() and dy.data_ptr() % 16 == 0:
        g, g_stride = dy, N
    else:
        g, g_stride = _rows_of(dy, 8)
    dev = _here(g)
    need = _linear_bwd_bytes(R, E, K, N, need_x, plan.top_k if gather else 0, need_w, y is not None)
    ws = g.new_empty((need // 2,)) if need else None
    dx = g.new_empty((x_rows, K)) if need_x else None
    dw = None if not need_w else g.new_empty((E, N, K)) if w_dtype == g.dtype else g.new_empty((E, N, K), dtype=w_dtype)
    rc = lib().nsx_expert_linear_bwd(
        x.data_ptr() if need_w else None, _DTYPE[g.dtype], x_stride, x_rows, plan.rows.data_ptr() if gather else None,
        plan.positions.data_ptr(), plan.top_k, w16.data_ptr() if need_x else None, g.data_ptr(), g_stride,
        None if y is None else y.data_ptr(), N, K, N, E, plan.offsets.data_ptr(), R, dx.data_ptr() if need_x else None,
        w_dtype == _F32, dw.data_ptr() if need_w else None, ws.data_ptr() if need else None, _raw_stream(dev))
    if rc:
        check(rc, "nsx_expert_linear_bwd")
    return dx, dw, None, None, None, None


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, w16, plan, gather, relu):
        xr, x_stride = _rows_of(x, 8)
        y = _linear(xr, x_stride, w16, plan, gather, relu)
        need_x, need_w = ctx.needs_input_grad[:2]
        ctx.save_for_backward(xr if need_w else None, w16 if need_x else None, y if relu else None)
        ctx.plan = plan, plan._version()
        ctx.cfg = (x_stride, x.shape[0], w16.shape, gather, weight.dtype, need_x, need_w)
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_linear_bwd_once if torch.is_grad_enabled() else _linear_bwd)(ctx, dy)


_linear_bwd_once = once_differentiable(_linear_bwd)


def expert_linear(x: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan, gather: bool = True, relu: bool = False,
                  w16: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[T * top_k, n_out] in the plan's order: ordered row p of expert e is ``weight[e] @ x[row of p]`` (``relu``: its positive
    part), differentiable w.r.t. ``x`` and ``weight``; ordered rows behind the last segment are 0.

    x: fp16 or bf16, [T, n_in] rows (``gather``) or [T * top_k, n_in] in the plan's order.  weight [E, n_out, n_in]: of x's
    dtype, or fp32 parameters whose copy in x's dtype is ``w16`` (made here if it is not given); the gradient has the dtype of
    ``weight``.  n_in and n_out are multiples of 8."""
    if _lib._COUNT_SCOPE is None and not _profiler.enabled:
        out = _fast.expert_linear(x, weight, w16, plan._offsets, plan._rows, plan._positions, bool(gather), bool(relu))
        if out is not None:
            return out
    _no_tangent("expert_linear", x, weight, w16)
    xs, ws, xt, wt = x.shape, weight.shape, x.dtype, weight.dtype
    if len(xs) != 2 or xt not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"expert_linear: x is [rows, n_in] in fp16 or bf16 (got {tuple(xs)} {xt})")
    if len(ws) != 3 or (wt != xt and wt != _F32):
        raise RuntimeError(f"expert_linear: weight is [E, n_out, n_in] in {xt} or fp32 (got {tuple(ws)} {wt})")
    if ws[0] != plan.n_experts or xs[1] != ws[2]:
        raise RuntimeError(f"expert_linear: weight {tuple(ws)} for rows of {xs[1]} and a plan of {plan.n_experts} experts")
    if xs[0] != (plan.n_rows if gather else plan.n_entries):
        raise RuntimeError(f"expert_linear: x has {xs[0]} rows for a plan of {plan.n_rows} x {plan.top_k} entries (gather={bool(gather)})")
    if w16 is None:
        w16 = weight if wt == xt else weight.detach().to(xt)
    elif w16.shape != ws or w16.dtype != xt:
        raise RuntimeError(f"expert_linear: w16 is {tuple(w16.shape)} {w16.dtype}, not {tuple(ws)} {xt}")
    if not w16.is_contiguous():
        w16 = w16.contiguous()
    if w16.data_ptr() % 16:
        w16 = w16.clone()
    if (x.requires_grad or weight.requires_grad) and torch.is_grad_enabled():
        return _LinearFn.apply(x, weight, w16, plan, bool(gather), bool(relu))
    xr, x_stride = _rows_of(x, 8)
    return _linear(xr, x_stride, w16, plan, bool(gather), bool(relu))


# ------------------------------------------------------------------------------------------------
# join
# ------------------------------------------------------------------------------------------------
def _combine(y, y_stride, weights, plan):
    R, n = y.shape
    T = plan.n_rows
    dev = _here(y)
    if weights.get_device() != dev or plan.device != dev:
        ptr(weights), ptr(plan.positions)
    out = y.new_empty((T, n))
    rc = lib().nsx_expert_combine_fwd(y.data_ptr(), _DTYPE[y.dtype], y_stride, R, n, weights.data_ptr(), plan.positions.data_ptr(), T,
                                      plan.top_k, out.data_ptr(), None if _lib._COUNT_SCOPE is None else ndev(T), _raw_stream(dev))
    if rc:
        check(rc, "nsx_expert_combine_fwd")
    return out


def _combine_bwd(ctx, dout):
    y, w = ctx.saved_tensors
    stride, w_dtype = ctx.cfg
    plan = _plan_of(ctx)
    T, k = plan.n_rows, plan.top_k
    R, n = y.shape
    if not dout.is_contiguous():
        dout = dout.contiguous()
    if dout.data_ptr() % 16:
        dout = dout.clone()
    dev = y.get_device()
    dy = torch.empty_like(y) if stride == n else y.new_empty((R, n))
    dw = torch.empty_like(w)
    rc = lib().nsx_expert_combine_bwd(y.data_ptr(), _DTYPE[y.dtype], stride, R, n, w.data_ptr(), plan.positions.data_ptr(),
                                      plan.offsets.data_ptr() + 4 * plan.n_experts, T, k, dout.data_ptr(), dy.data_ptr(),
                                      dw.data_ptr(), None if _lib._COUNT_SCOPE is None else ndev(T), _raw_stream(dev))
    if rc:
        check(rc, "nsx_expert_combine_bwd")
    return dy, dw if w_dtype == _F32 else dw.to(w_dtype), None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, plan):
        yr, stride = _rows_of(y, 8)
        w = weights if weights.dtype == _F32 and weights.is_contiguous() else weights.to(_F32).contiguous()
        ctx.save_for_backward(yr, w)
        ctx.plan = plan, plan._version()
        ctx.cfg = (stride, weights.dtype)
        return _combine(yr, stride, w, plan)

    @staticmethod
    def backward(ctx, dout):
        return (_combine_bwd_once if torch.is_grad_enabled() else _combine_bwd)(ctx, dout)


_combine_bwd_once = once_differentiable(_combine_bwd)


def expert_combine(y: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """[T, n]: sum over a row's choices of ``weights[t, j] * y[plan.positions[t, j]]``, differentiable w.r.t. ``y`` [T * top_k,
    n] (fp16 or bf16, n a multiple of 8) and ``weights`` [T, top_k]; choices that are not routed count nothing."""
    if _lib._COUNT_SCOPE is None and not _profiler.enabled:
        out = _fast.expert_combine(y, weights, plan._offsets, plan._rows, plan._positions)
        if out is not None:
            return out
    _no_tangent("expert_combine", y, weights)
    ys = y.shape
    if len(ys) != 2 or ys[0] != plan.n_entries or y.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"expert_combine: y is [{plan.n_entries}, n] in fp16 or bf16 (got {tuple(ys)} {y.dtype})")
    if weights.shape != (plan.n_rows, plan.top_k) or not weights.is_floating_point():
        raise RuntimeError(f"expert_combine: weights are {(plan.n_rows, plan.top_k)} (got {tuple(weights.shape)} {weights.dtype})")
    if (y.requires_grad or weights.requires_grad) and torch.is_grad_enabled():
        return _CombineFn.apply(y, weights, plan)
    yr, stride = _rows_of(y, 8)
    return _combine(yr, stride, weights if weights.dtype == _F32 and weights.is_contiguous() else weights.to(_F32).contiguous(), plan)
