"""Training against another model's class probabilities of which only the highest logits are kept.

A black-box teacher (any classifier, whatever its number of classes) is distilled into a student: the teacher's ``k`` highest
logits of every row are stored once, and :func:`distill_grad` gives the divergence of the student's distribution from the teacher's
and its gradient with respect to the student's logits.  The caller chains that gradient into what made the logits: the weights of
features (a model's Gram matrix columns, say), or through :func:`oak.experts.combine_grad` and :func:`oak.experts.route_grad` a
mixture's answers and router.  The models' own kernel parameters are not reached: their gradients in this package are those of the
bound and of the log marginal likelihood.

Arrays are NumPy arrays (float64; results are NumPy arrays) or torch tensors on a HIP device (logits of type float64, float32, bfloat16 or float16;
results on the same device, computed on its current stream without waiting for them).  Losses are float64 for float64 logits
and float32 otherwise.
"""
from __future__ import annotations

import numpy as np

from . import _arrays as A
from . import _capi

MAX_CLASSES, MAX_TEACHER = 1 << 20, 1024
_DIRECTIONS = {"forward": 0, "reverse": 1}


def distill(logits, top, index, *, top_lse=None, temperature: float = 1.0, direction: str = "forward", row_weight=None):
    """Divergence of every row, [N].

    ``logits`` [N, V] are the student's, q = softmax(logits / temperature).  ``top`` and ``index`` [N, k] are the teacher's kept
    logits and their classes (int32 or int64); index -1 or a value of -inf is padding, entries of the same class add their probabilities.

    Without ``top_lse`` the teacher is softmax(top / temperature) over its kept classes.  With ``top_lse`` [N], log sum exp(logit / temperature) over
    ALL the teacher's classes, the kept ones have p = exp(top / temperature - top_lse) and what is left of 1 is one more outcome, held
    against the student's mass outside the kept classes.

    ``direction`` "forward" is KL(teacher || student), "reverse" KL(student || teacher), which needs ``top_lse`` and takes
    the mass left over as at least the resolution of ``top_lse`` (2^-24, float64: 2^-53).  The divergence is multiplied by temperature^2 and by
    ``row_weight`` [N]; rows of weight 0 are not read.  Rows whose teacher kept nothing have loss 0.  A student that rules out (-inf) what its
    teacher does not has an infinite loss.  An index outside -1 .. V - 1 is refused in a NumPy array and makes its row's loss
    NaN on a device.  V is at most 2^20, k at most 1024.
    """
    return _distill(logits, top, index, top_lse, temperature, direction, row_weight, False)[0]


def distill_grad(logits, top, index, *, top_lse=None, temperature: float = 1.0, direction: str = "forward", row_weight=None):
    """(loss [N], gradient of their sum with respect to ``logits`` [N, V]) in one call; arguments as for :func:`distill`.

    ``top_lse`` may be rounded: a kept mass above 1 stays what it is, in the loss and in its gradient (within 2^-18 of 1 it is taken for 1 in the
    gradient).  For the mean over rows, or any weighting of them, give ``row_weight``.
    """
    return _distill(logits, top, index, top_lse, temperature, direction, row_weight, True)


def _distill(logits, top, index, top_lse, temperature, direction, row_weight, grad):
    if direction not in _DIRECTIONS:
        raise ValueError(f"direction must be 'forward' or 'reverse', not {direction!r}")
    device = A.on_device(logits)
    if device:
        d = A.Device(logits)
        logits = d.matrix(logits, "logits")
        top = d.matrix(top, "top")
    else:
        logits, top = A.host(logits, "logits"), A.host(top, "top")
    n, v = logits.shape
    k = top.shape[1]
    if top.shape[0] != n:
        raise ValueError(f"top has {top.shape[0]} rows, logits {n}")
    if not (1 <= v <= MAX_CLASSES and 1 <= k <= MAX_TEACHER):
        raise ValueError(f"{v} classes and {k} entries; 1 .. {MAX_CLASSES} classes and 1 .. {MAX_TEACHER} entries are supported")
    a = _capi.DistillArgs(n_rows=n, n_classes=v, top_k=k, temperature=float(temperature), direction=_DIRECTIONS[direction])
    if device:
        a.dtype, a.top_dtype = A.code_of(logits, "logits"), A.code_of(top, "top")
        index = d.matrix(index, "index", (n, k))
        if index.dtype not in (d.torch.int32, d.torch.int64):
            raise ValueError(f"index is of type {index.dtype}; int32 or int64 is expected")
        a.index_64 = int(index.dtype == d.torch.int64)
        a.ld_logits, a.ld_top, a.ld_index = logits.stride(0), top.stride(0), index.stride(0)
        if top_lse is not None:
            top_lse = d.dense(top_lse, "top_lse", (n,))
            a.lse_dtype = A.code_of(top_lse, "top_lse")
        if row_weight is not None:
            row_weight = d.dense(row_weight, "row_weight", (n,))
            a.weight_dtype = A.code_of(row_weight, "row_weight")
        loss = d.empty((n,), d.wide(a.dtype))
        dlogits = d.empty((n, v), logits.dtype) if grad else None
    else:
        index = A.host_index(index, "index", -1, v)
        if index.shape != (n, k):
            raise ValueError(f"index has shape {index.shape}, expected {(n, k)}")
        a.ld_logits, a.ld_top, a.ld_index = v, k, k
        top_lse = None if top_lse is None else A.host(top_lse, "top_lse", (n,))
        row_weight = None if row_weight is None else A.host(row_weight, "row_weight", (n,))
        loss = np.empty(n)
        dlogits = np.empty((n, v)) if grad else None
    a.ld_dlogits = v
    a.logits, a.top, a.index, a.top_lse, a.row_weight = A.ptr(logits), A.ptr(top), A.ptr(index), A.ptr(top_lse), A.ptr(row_weight)
    a.loss, a.dlogits = A.ptr(loss), A.ptr(dlogits)
    if device:
        if n <= 128:                                                     # few rows may be cut into slices, whose sums are kept meanwhile
            a.workspace_doubles = _capi.distill_workspace(d.ctx, n, v, a.dtype)
            workspace = d.empty((a.workspace_doubles,), d.torch.float64) if a.workspace_doubles else None
            a.workspace = A.ptr(workspace)
        _capi.call_device("distill", d.ctx, d.stream, a)
    else:
        _capi.default_context().call("distill", a)
    return loss, dlogits
