"""Host and device arrays of the operators in ``oak.experts`` and ``oak.distillation``.

Host arrays are whatever ``numpy.asarray`` takes and become contiguous float64, as everywhere in this package.  Device arrays are
torch tensors on a HIP device; they stay where they are, in their own type, and the operators run on the tensor's device and that
device's current torch stream.  This module never imports torch itself: a caller who has a tensor has imported it.
"""
from __future__ import annotations

import sys

import numpy as np

from . import _capi

F64, F32, BF16, F16 = 0, 1, 2, 3
_codes = {}                 # torch dtype -> element type of the C interface
_contexts = {}              # contexts of the devices whose torch memory the library's HIP runtime is known to see


def on_device(a) -> bool:
    return getattr(a, "is_cuda", False) is True


def _torch():
    return sys.modules["torch"]


def code_of(t, what: str) -> int:
    if not _codes:
        torch = _torch()
        _codes.update({torch.float64: F64, torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16})
    code = _codes.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} is of type {t.dtype}; float64, float32, bfloat16 and float16 are supported")
    return code


class Device:
    """The device and stream of one call, with its checks of every tensor."""

    __slots__ = ("torch", "index", "ctx", "like", "dual")

    def __init__(self, t):
        self.torch, self.like = _torch(), t
        self.dual = getattr(self.torch.autograd.forward_ad, "_current_level", 0) >= 0        # a level of forward-mode differentiation is open
        self.index = t.get_device()
        self.ctx = _contexts.get(self.index)
        if self.ctx is None or self.ctx._h is None:
            self.ctx = self._first(t)

    def _first(self, t):
        """The first call on a device: its context, and whether the tensor's memory is the library's to see."""
        two = "torch and the OAK library hold different copies of the HIP runtime; import torch before the first use of the oak package"
        if len(_capi.hip_runtimes()) > 1:
            raise _capi.OakHipError(two)
        if self.torch.cuda.is_current_stream_capturing():
            raise _capi.OakHipError("the first call on a device makes its context, which a stream cannot capture: make one call before the capture")
        with self.torch.cuda.device(self.index):            # making a context changes the current device
            ctx = _capi.device_context(self.index)
        if t.data_ptr() != 0:
            try:
                _capi.check_device_pointer(ctx, t.data_ptr())
            except ValueError as e:
                raise _capi.OakHipError(f"{e}: {two}") from None
            _contexts[self.index] = ctx
        return ctx

    @property
    def stream(self) -> int:
        # the handle alone: building a torch.cuda.Stream around it takes as long as a small kernel
        try:
            return self.torch._C._cuda_getCurrentRawStream(self.index)
        except AttributeError:
            return self.torch.cuda.current_stream(self.index).cuda_stream

    def tensor(self, a, what: str):
        try:
            here = a.get_device() == self.index
        except AttributeError:
            here = False
        if not here:
            raise ValueError(f"{what} must be on {self.like.device} like the first array of the call")
        if a.requires_grad and self.torch.is_grad_enabled():
            raise ValueError(f"{what} requires grad: the operators record no graph, their gradients are calls of their own; pass {what}.detach()")
        if self.dual and self.torch.autograd.forward_ad.unpack_dual(a).tangent is not None:
            raise ValueError(f"{what} carries a forward-mode tangent, which the operators would drop; pass its primal")
        return a.resolve_neg() if a.is_neg() else a          # a view that negates when it is read

    def matrix(self, a, what: str, shape=None):
        """A 2-D tensor whose columns are consecutive (copied if they are not)."""
        a = self.tensor(a, what)
        if a.dim() != 2 or (shape is not None and a.shape != shape):
            raise ValueError(f"{what} has shape {tuple(a.shape)}, expected {'two dimensions' if shape is None else shape}")
        return a if a.stride(1) == 1 or a.shape[1] <= 1 else a.contiguous()

    def dense(self, a, what: str, shape, dtype=None):
        """A contiguous tensor of this shape (and type)."""
        a = self.tensor(a, what)
        if a.shape != shape:
            raise ValueError(f"{what} has shape {tuple(a.shape)}, expected {shape}")
        if dtype is not None and a.dtype != dtype:
            a = a.to(dtype)
        return a if a.is_contiguous() else a.contiguous()

    def wide(self, code: int):
        """Type of sums, weights and losses for arrays of this type."""
        return self.torch.float64 if code == F64 else self.torch.float32

    def empty(self, shape, dtype):
        return self.like.new_empty(shape, dtype=dtype)


def whole(value, what: str, low: int, high: int) -> int:
    """An integer in [low, high]; checked here, before it sizes an array or is cut to 32 bits on its way to the library."""
    number = int(value)
    if number != value or not low <= number <= high:
        raise ValueError(f"{what} = {value!r} is not an integer in {low} .. {high}")
    return number


def ptr(a) -> int | None:
    """Address of a tensor or array, None for None and for empty ones."""
    if a is None:
        return None
    if isinstance(a, np.ndarray):
        return a.ctypes.data if a.size else None
    address = a.data_ptr()
    if address == 0 and a.numel() > 0:                       # would be an array left out
        raise ValueError("an array is zeros without storage; pass its clone()")
    return address or None


def host(a, what: str, shape=None) -> np.ndarray:
    if on_device(a):
        raise ValueError(f"{what} is a device array, the call's first array is not")
    a = np.ascontiguousarray(a, dtype=np.float64)
    if (a.ndim != 2) if shape is None else (a.shape != shape):
        raise ValueError(f"{what} has shape {a.shape}, expected {'two dimensions' if shape is None else shape}")
    return a


def host_index(a, what: str, low: int, high: int, dtype=np.int32) -> np.ndarray:
    """Integers in [low, high)."""
    if on_device(a):
        raise ValueError(f"{what} is a device array, the call's first array is not")
    a = np.asarray(a)
    if a.dtype.kind not in "iu":
        raise ValueError(f"{what} must be integers, not {a.dtype}")
    if a.size and (a.min() < low or a.max() >= high):
        raise ValueError(f"{what} has values outside {low} .. {high - 1}")
    return np.ascontiguousarray(a, dtype=dtype)
