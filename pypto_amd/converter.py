"""``from_torch``: the tensor hand-over of the reference's legacy jit front end.

Reference: python/pypto/converter.py:35-112.  There the call returns a ``pypto.Tensor`` carrying
shape (with dynamic axes marked), dtype, name, data pointer, format and device.  Here the kernels
are pre-compiled and every shape is a launch argument, so ``dynamic_axis`` and ``tensor_format``
carry no information; the wrapper keeps the torch tensor and exposes the same attributes.
The error behaviour is the reference's: ``TypeError`` for anything that is not a torch tensor,
``RuntimeError`` for a non-contiguous one (converter.py:76-80).
"""
from __future__ import annotations

from typing import List, Optional

import torch


class Tensor:
    """Thin handle on a contiguous torch tensor (device memory stays owned by the caller)."""

    __slots__ = ("_t", "name", "dynamic_axis", "format")

    def __init__(self, t: torch.Tensor, name: str = "", dynamic_axis: Optional[List[int]] = None, fmt=None):
        self._t = t
        self.name = name
        self.dynamic_axis = list(dynamic_axis) if dynamic_axis is not None else None
        self.format = fmt

    @property
    def shape(self):
        return list(self._t.shape) if self._t.dim() else [1]

    @property
    def ori_shape(self):
        return list(self._t.shape)

    @property
    def dtype(self):
        return self._t.dtype

    @property
    def device(self):
        return self._t.device

    @property
    def data_ptr(self):
        return self._t.data_ptr()

    def torch(self) -> torch.Tensor:
        return self._t

    def __repr__(self):
        return f"pypto_amd.Tensor(name={self.name!r}, shape={self.shape}, dtype={self.dtype}, device={self.device})"


def from_torch(tensor, name: str = "", dynamic_axis: Optional[List[int]] = None, tensor_format=None) -> Tensor:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError("input type is not currently supported.")
    if not tensor.is_contiguous():
        raise RuntimeError("not all tensors are contiguous")
    return Tensor(tensor, name, dynamic_axis, tensor_format)


def as_torch(x, what: str) -> torch.Tensor:
    """Operator-side unwrapping: accepts the wrapper or a bare torch tensor."""
    if isinstance(x, Tensor):
        return x.torch()
    if isinstance(x, torch.Tensor):
        if not x.is_contiguous():
            raise RuntimeError(f"{what}: not all tensors are contiguous")
        return x
    raise TypeError(f"{what}: input type is not currently supported.")


def as_rows(x, what: str) -> torch.Tensor:
    """Unwrapping for the operators that take strided tensors: the last dimension alone has to be contiguous."""
    t = x.torch() if isinstance(x, Tensor) else x
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: input type is not currently supported.")
    if t.dim() and t.stride(-1) != 1 and t.shape[-1] > 1:
        raise RuntimeError(f"{what}: the last dimension must be contiguous")
    return t


def extent(t: torch.Tensor):
    """First and one past the last byte that a tensor's elements lie in."""
    if t.numel() == 0:
        return t.data_ptr(), t.data_ptr()
    return t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def same_rows(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one shape and type are the same memory, element by element."""
    return a.data_ptr() == b.data_ptr() and all(x == y for n, x, y in zip(a.shape, a.stride(), b.stride()) if n > 1)


def side_by_side(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors are different columns of rows that lie equally far apart, or different channels of such heads (slices of one
    tensor)."""
    x, y = a, b
    for d in range(min(a.dim(), b.dim()) - 1):
        pitch = x.stride(0) * a.element_size()
        if min(x.shape[0], y.shape[0]) < 2 or pitch <= 0 or y.stride(0) * b.element_size() != pitch:
            return False
        if d and (a.stride(0) % x.stride(0) or b.stride(0) % y.stride(0)):
            return False
        x, y = x[0], y[0]
        (lo, hi), (lo2, hi2) = extent(x), extent(y)
        at = (lo2 - lo) % pitch                            # where b's columns begin, seen from a's
        if at >= hi - lo and at + (hi2 - lo2) <= pitch:
            return True
    return False


def refuse_overlap(out: torch.Tensor, other: torch.Tensor, what: str) -> None:
    """Outputs have memory of their own.  Views that interleave in one allocation count as overlapping, but for different columns of the
    same rows."""
    (lo, hi), (lo2, hi2) = extent(out), extent(other)
    if lo < hi2 and lo2 < hi and not side_by_side(out, other):
        raise ValueError(f"{what} overlap in memory")


def check_writable(t: torch.Tensor, what: str) -> None:
    """No two elements of an output may share memory."""
    reach = 1
    for stride, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if stride < reach:
            raise ValueError(f"{what}: elements share memory")
        reach += (n - 1) * stride


def copy_unless_same(dst: torch.Tensor, src: torch.Tensor, what: str) -> None:
    """The cache-out arguments of the prolog operators: normally the very tensor passed as cache-in (the
    kernels then update the rows named by the cache index in place and nothing is copied).  A different
    tensor receives a copy of the whole cache first -- the reference's semantics, and gigabytes per call at
    real cache sizes, so in-place use is the intended path.  Two views that share memory without being the
    same range would be copied onto themselves: refused."""
    if dst.data_ptr() == src.data_ptr():
        return
    lo_d, lo_s = dst.data_ptr(), src.data_ptr()
    hi_d, hi_s = lo_d + dst.numel() * dst.element_size(), lo_s + src.numel() * src.element_size()
    if lo_d < hi_s and lo_s < hi_d:
        raise ValueError(f"{what} and {what}_out overlap in memory without being the same tensor")
    dst.copy_(src.reshape(dst.shape))
