"""Mixtures of models: rows routed to experts, laid out by expert, and the experts' answers summed.

An additive model that is too stiff for a whole data set is replaced by several, each fitted and asked on its own rows: a router
gives every row a score for every expert (a gating model's outputs, distances to k-means centres, ...), :func:`route` picks each row's experts and
their weights, :func:`plan` and :func:`dispatch` lay the rows out so that every expert finds its own in one block, and
:func:`combine` sums the answers.  The ``*_grad`` functions are the closed-form adjoints, so that a router and its experts can be
trained against any loss on the mixture's output (:mod:`oak.distillation` has one).

All functions take NumPy arrays (float64, results are NumPy arrays) or torch tensors on a HIP device (float64, float32, bfloat16, float16;
results are tensors on the same device, computed on its current stream without waiting for them).  Sums, weights and
their gradients are float64 for float64 arrays and float32 otherwise.

>>> experts, weights = route(scores, top_k=2)                 # [N, 2], [N, 2]
>>> p = plan(experts, n_experts=scores.shape[1])
>>> rows = dispatch(X, p)                                      # expert e's rows: rows[p.offsets[e]:p.offsets[e + 1]]
>>> y = combine(answers, weights, p)                           # answers in the same layout
"""
from __future__ import annotations

from typing import NamedTuple

import numpy as np

from . import _arrays as A
from . import _capi

MAX_EXPERTS, MAX_PLAN_EXPERTS, MAX_TOP_K = 1024, 4096, 64
_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"max": 0, "top2": 1}


def _code(table, value, what):
    try:
        return table[value]
    except (KeyError, TypeError):
        raise ValueError(f"{what} must be one of {', '.join(map(repr, table))}, not {value!r}") from None


def _route_args(scores, top_k, score, n_groups, top_groups, group_score, renormalise, scale, code, ld):
    n, e = scores.shape
    if not 1 <= e <= MAX_EXPERTS:
        raise ValueError(f"scores has {e} columns; 1 .. {MAX_EXPERTS} experts are supported")
    n_groups = A.whole(n_groups, "n_groups", 1, 64)
    a = _capi.RouteArgs(n_rows=n, ld_scores=ld, n_experts=e, top_k=A.whole(top_k, "top_k", 1, min(e, MAX_TOP_K)), n_groups=n_groups,
                        top_groups=n_groups if top_groups is None else A.whole(top_groups, "top_groups", 1, n_groups), dtype=code,
                        score=_code(_SCORES, score, "score"), group_score=_code(_GROUP_SCORES, group_score, "group_score"),
                        renormalise=1 if renormalise else 0, scale=float(scale))
    a.scores = A.ptr(scores)
    return a


def _device_mask(d, mask, n, e, a):
    """Boolean (or uint8) [n, e] or [e] -> the tensor to keep alive."""
    if mask is None:
        return None
    mask = d.tensor(mask, "mask")
    if mask.dtype not in (d.torch.bool, d.torch.uint8):
        raise ValueError(f"mask is of type {mask.dtype}; bool is expected")
    if tuple(mask.shape) == (e,):
        mask, a.ld_mask = mask.contiguous(), 0
    else:
        mask = d.matrix(mask, "mask", (n, e))
        a.ld_mask = mask.stride(0)
    a.mask = A.ptr(mask)
    return mask


def _host_mask(mask, n, e, a):
    if mask is None:
        return None
    mask = np.ascontiguousarray(mask, dtype=bool).view(np.uint8)
    if mask.shape not in ((e,), (n, e)):
        raise ValueError(f"mask has shape {mask.shape}, expected {(n, e)} or {(e,)}")
    a.ld_mask = 0 if mask.ndim == 1 else e
    a.mask = A.ptr(mask)
    return mask


def route(scores, top_k: int, *, score: str = "softmax", bias=None, n_groups: int = 1, top_groups: int | None = None,
          group_score: str = "max", renormalise: bool = True, scale: float = 1.0, mask=None):
    """Each row's ``top_k`` experts and their weights: (experts [N, k] int32, weights [N, k]).

    ``scores`` [N, E] become probabilities p by ``score`` = "softmax" (over the row's open experts) or "sigmoid".  An expert is
    open to a row unless ``mask`` [N, E] or [E] is False there or its score is -inf.  The choice goes by p + ``bias`` [E] (a balance
    correction of size below 1e300: it moves the choice, not the weights; -inf closes its expert to the choice), highest
    first, ties to the lower index.  With ``n_groups`` > 1 the experts form groups of consecutive ones, of which the
    ``top_groups`` best stay open; ``group_score`` = "max" ranks them by their best expert, "top2" by the sum of their two
    best.  weights = ``scale`` * p, divided by the chosen experts' sum if ``renormalise``.

    Slots that no open expert is left for hold expert -1 and weight 0.  A row with a NaN or +inf among its open scores holds
    experts -1 and weights NaN.  A NaN or +inf in ``bias`` is refused in a NumPy array; on a device it counts like such a score of
    that expert.  At most 1024 experts, ``top_k`` at most 64.
    """
    if A.on_device(scores):
        d = A.Device(scores)
        scores = d.matrix(scores, "scores")
        n, e = scores.shape
        code = A.code_of(scores, "scores")
        a = _route_args(scores, top_k, score, n_groups, top_groups, group_score, renormalise, scale, code, scores.stride(0))
        mask = _device_mask(d, mask, n, e, a)
        if bias is not None:
            bias = d.dense(bias, "bias", (e,))
            if bias.dtype not in (d.torch.float32, d.torch.float64):
                bias = bias.to(d.torch.float32)
            a.bias_f64, a.bias = int(bias.dtype == d.torch.float64), A.ptr(bias)
        experts, weights = d.empty((n, a.top_k), d.torch.int32), d.empty((n, a.top_k), d.wide(code))
        a.experts, a.weights = A.ptr(experts), A.ptr(weights)
        _capi.call_device("route", d.ctx, d.stream, a)
        return experts, weights
    scores = A.host(scores, "scores")
    n, e = scores.shape
    a = _route_args(scores, top_k, score, n_groups, top_groups, group_score, renormalise, scale, A.F64, e)
    mask = _host_mask(mask, n, e, a)
    if bias is not None:
        bias = A.host(bias, "bias", (e,))
        if not (bias < np.inf).all():
            raise ValueError("bias holds NaN or +inf")
        a.bias_f64, a.bias = 1, A.ptr(bias)
    experts, weights = np.empty((n, a.top_k), dtype=np.int32), np.empty((n, a.top_k))
    a.experts, a.weights = A.ptr(experts), A.ptr(weights)
    _capi.default_context().call("route", a)
    return experts, weights


def route_grad(scores, experts, dweights, *, score: str = "softmax", renormalise: bool = True, scale: float = 1.0, mask=None):
    """Gradient with respect to ``scores`` from the gradient ``dweights`` [N, k] with respect to :func:`route`'s weights.

    ``experts`` are the ones :func:`route` chose (different ones in every row; -1: none), the other arguments those of its
    call; the choice itself is not differentiated.  A row without experts has gradient 0.
    """
    if A.on_device(scores):
        d = A.Device(scores)
        scores = d.matrix(scores, "scores")
        n, e = scores.shape
        code = A.code_of(scores, "scores")
        k = _columns(experts, n, "experts")
        experts = _device_experts(d, experts, (n, k), e)
        dweights = d.dense(dweights, "dweights", (n, k), d.wide(code))
        a = _route_args(scores, k, score, 1, 1, "max", renormalise, scale, code, scores.stride(0))
        mask = _device_mask(d, mask, n, e, a)
        out = d.empty((n, e), scores.dtype)
        a.experts, a.dweights, a.dscores, a.ld_dscores = A.ptr(experts), A.ptr(dweights), A.ptr(out), e
        _capi.call_device("route_grad", d.ctx, d.stream, a)
        return out
    scores = A.host(scores, "scores")
    n, e = scores.shape
    k = _columns(experts, n, "experts")
    experts = A.host_index(experts, "experts", -1, e)
    dweights = A.host(dweights, "dweights", (n, k))
    a = _route_args(scores, k, score, 1, 1, "max", renormalise, scale, A.F64, e)
    mask = _host_mask(mask, n, e, a)
    out = np.empty((n, e))
    a.experts, a.dweights, a.dscores, a.ld_dscores = A.ptr(experts), A.ptr(dweights), A.ptr(out), e
    _capi.default_context().call("route_grad", a)
    return out


def _columns(experts, n, what):
    shape = tuple(experts.shape) if hasattr(experts, "shape") else np.shape(experts)
    if len(shape) != 2 or shape[0] != n:
        raise ValueError(f"{what} has shape {shape}, expected {n} rows")
    return shape[1]


def _device_experts(d, experts, shape, n_experts):
    experts = d.tensor(experts, "experts")
    if experts.dtype == d.torch.int32:
        return d.dense(experts, "experts", shape)
    t = d.torch
    if experts.dtype == t.int64:                                        # what 32 bits cannot hold stays no expert's number
        return d.dense(experts.clamp(-1, n_experts), "experts", shape, t.int32)
    if experts.dtype not in (t.int16, t.int8, t.uint8):
        raise ValueError(f"experts is of type {experts.dtype}; int8, int16, int32, int64 and uint8 are supported")
    return d.dense(experts, "experts", shape, t.int32)


class Plan(NamedTuple):
    """Where every slot (row n's j-th expert) sits in the layout by expert.

    ``rows`` [N k]: the row at each place, -1 behind the last used one; ``positions``: the place of each slot, -1 for slots without an
    expert, in the shape of the experts; ``counts`` [E] and ``offsets`` [E + 1]: expert e has the places offsets[e] .. offsets[e + 1).
    All int32, of the kind (array or tensor) of the experts.
    """
    rows: object
    positions: object
    counts: object
    offsets: object
    n_rows: int
    top_k: int
    n_experts: int


def plan(experts, n_experts: int) -> Plan:
    """The layout by expert of ``experts`` [N, k], or of labels [N] (one expert a row, as k-means gives them).

    Slots keep their order within an expert, so the layout depends on nothing but its input.  A slot whose expert is -1 has no place.  On a device any
    other value outside 0 .. n_experts - 1 has none either; in a NumPy array it is refused.  At most 4096 experts.
    """
    n_experts = A.whole(n_experts, "n_experts", 1, MAX_PLAN_EXPERTS)
    shape = tuple(experts.shape) if hasattr(experts, "shape") else np.shape(experts)
    if len(shape) not in (1, 2):
        raise ValueError(f"experts has shape {shape}, expected [N, k] or [N]")
    n, k = shape[0], A.whole(shape[1], "k", 1, MAX_TOP_K) if len(shape) == 2 else 1
    if n * k >= 1 << 31:
        raise ValueError(f"{n} rows x {k} experts pass 2^31 slots")
    a = _capi.PlanArgs(n_rows=n, top_k=k, n_experts=n_experts)
    if A.on_device(experts):
        d = A.Device(experts)
        experts = _device_experts(d, experts, shape, n_experts)
        i32 = d.torch.int32
        out = d.empty((2 * n * k + 2 * n_experts + 1,), i32).split_with_sizes((n * k, n * k, n_experts, n_experts + 1))   # one allocation
        out = [out[0], out[1].view(shape), out[2], out[3]]
        a.workspace_ints = _capi.plan_workspace(d.ctx, n, k, n_experts)
        workspace = d.empty((a.workspace_ints,), i32) if a.workspace_ints else None
        a.workspace = A.ptr(workspace)
    else:
        experts = A.host_index(experts, "experts", -1, n_experts)
        out = [np.empty(s, dtype=np.int32) for s in ((n * k,), shape, (n_experts,), (n_experts + 1,))]
    a.experts = A.ptr(experts)
    a.rows, a.positions, a.counts, a.offsets = map(A.ptr, out)
    if A.on_device(experts):
        _capi.call_device("plan", d.ctx, d.stream, a)
    else:
        _capi.default_context().call("plan", a)
    return Plan(*out, n, k, n_experts)


def _mix(name, plan, first, what, slots_in, weights=None, dout=None):
    """Common body of dispatch (rows -> slots), combine (slots -> rows) and combine_grad."""
    if not isinstance(plan, Plan):
        raise ValueError("plan must come from oak.experts.plan")
    _, positions, _, offsets, n, k, n_experts = plan
    device = A.on_device(first)
    if device != A.on_device(positions) or device != A.on_device(offsets):
        raise ValueError(f"{what} and the plan must both be device arrays or both be host arrays")
    d = A.Device(first) if device else None
    if not device:
        first = np.asarray(first)
    shape = first.shape
    rows_in = n * k if slots_in else n
    flat = len(shape) == 1
    if len(shape) not in (1, 2) or shape[0] != rows_in:
        raise ValueError(f"{what} has shape {tuple(shape)}, the plan expects {rows_in} rows")
    if flat:
        first = first[:, None]
        dout = dout if dout is None else (dout if device else np.asarray(dout))[:, None]
    c = first.shape[1]
    if c > 1 << 30:
        raise ValueError(f"{what} has {c} columns; at most 2^30 are supported")
    if device:
        i32 = d.torch.int32
        altered = positions.dtype != i32 or offsets.dtype != i32 or positions.numel() != n * k or offsets.numel() != n_experts + 1
        if altered or not (positions.is_contiguous() and offsets.is_contiguous()):
            raise ValueError("plan has been altered: its arrays do not fit its sizes")
        d.tensor(positions, "the plan")
        d.tensor(offsets, "the plan")
        src = d.matrix(first, what)
        code = A.code_of(src, what)
        wide, row_stride, grad_stride = d.wide(code), src.stride(0), c
        if weights is not None:
            weights = d.dense(weights, "weights", (n, k), wide)
        if dout is not None:
            dout = d.matrix(dout, "dout", (n, c))
            if dout.dtype != src.dtype:
                dout = dout.to(src.dtype)
            grad_stride = dout.stride(0)
    else:
        positions, offsets = A.host_index(positions, "positions", -1, max(n * k, 1)), A.host_index(offsets, "offsets", 0, n * k + 1)
        if positions.size != n * k or offsets.size != n_experts + 1:
            raise ValueError("plan has been altered: its arrays do not fit its sizes")
        src = A.host(first, what)
        code, wide, row_stride, grad_stride = A.F64, np.float64, c, c
        if weights is not None:
            weights = A.host(weights, "weights", (n, k))
        if dout is not None:
            dout = A.host(dout, "dout", (n, c))

    def empty(rows, columns, dtype):
        return d.empty((rows, columns), dtype) if device else np.empty((rows, columns), dtype)

    out = empty(n if slots_in and dout is None else n * k, c, src.dtype)
    dweights = None if dout is None else empty(n, k, wide)
    a = _capi.MixArgs(n, c if slots_in else row_stride, row_stride if slots_in else c, grad_stride, k, n_experts, c, code,
                      A.ptr(positions), A.ptr(offsets), A.ptr(weights), A.ptr(src), None if dweights is not None else A.ptr(out), A.ptr(dout),
                      A.ptr(out) if dweights is not None else None, A.ptr(dweights))
    if c == 0:
        if dweights is not None:
            dweights[...] = 0
    elif device:
        _capi.call_device(name, d.ctx, d.stream, a)
    else:
        _capi.default_context().call(name, a)
    if flat:
        out = out[:, 0]
    return out if dweights is None else (out, dweights)


def dispatch(X, plan: Plan):
    """Rows ``X`` [N, C] (or [N]) laid out by expert: [N k, C], zeros behind the last used place."""
    return _mix("dispatch", plan, X, "X", False)


def dispatch_grad(dlaid, plan: Plan):
    """Gradient with respect to ``X`` of :func:`dispatch`: each row's sum over its places of ``dlaid`` [N k, C]."""
    return _mix("combine", plan, dlaid, "dlaid", True)


def combine(answers, weights, plan: Plan):
    """Sum over each row's experts of weight times answer, [N, C]; ``answers`` [N k, C] (or [N k]) in the plan's layout.

    The answer of a slot without a place is a row of zeros: its weight, if finite, leaves no trace, and one that is NaN or infinite makes the
    row NaN, so that the NaN weights which :func:`route` gives a row it cannot route show in the sum.  What stands behind the last used
    place is not read.
    """
    return _mix("combine", plan, answers, "answers", True, weights=_required(weights, "weights"))


def combine_grad(answers, weights, plan: Plan, dout):
    """Gradients of :func:`combine` from ``dout`` [N, C]: (danswers [N k, C], zeros behind the last used place; dweights [N, k], 0 for slots without one)."""
    return _mix("combine_grad", plan, answers, "answers", True, weights=_required(weights, "weights"), dout=_required(dout, "dout"))


def _required(a, what):
    if a is None:
        raise ValueError(f"{what} is missing")
    return a
