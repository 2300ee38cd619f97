"""Argument checks shared by the prompt and draft operators."""

from __future__ import annotations

from typing import Tuple

import torch
from torch.autograd import forward_ad

HEAD_DIM = 128


def refuse_gradients(*tensors) -> None:
    """The kernels have no derivatives: say so rather than return outputs without a gradient or a tangent."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise NotImplementedError("TurboPolar kernels have no backward pass; call them under torch.no_grad()")
    if getattr(forward_ad, "_current_level", 0) >= 0:  # inside dual_level(), also under no_grad()
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("TurboPolar kernels have no forward-mode derivative; pass the primal tensors")


def raw_stream(device: torch.device) -> int:
    """The handle of ``device``'s current stream."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def launch(device: torch.device, fn, *args) -> int:
    """``fn(*args, stream)`` on ``device`` and its current stream."""
    i, stream = device.index, raw_stream(device)
    if i == torch.cuda.current_device():
        return fn(*args, stream)
    with torch.cuda.device(device):
        return fn(*args, stream)


def extent(x: torch.Tensor) -> Tuple[int, int]:
    """The byte range [lo, hi) that a non-empty tensor touches (strides are never negative)."""
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()


def _share_rows(a: torch.Tensor, b: torch.Tensor) -> bool:
    """True when ``a`` and ``b`` ``(..., T, H, 128)`` are slices of the same token rows with no common
    element: equal strides and, within a row, disjoint runs of heads (a fused projection's q and k).  Rows
    are ``row`` elements apart and every leading stride is a multiple of that, so an element's place within
    its row says which run it belongs to."""
    if a.dim() != b.dim() or a.stride() != b.stride() or a.shape[:-2] != b.shape[:-2]:
        return False
    leading = [s for s, n in zip(a.stride()[:-2], a.shape[:-2]) if n > 1]
    row = min(leading, default=0)  # none: one row, whose run is the extent
    size = a.element_size()
    if not row or size != b.element_size() or (b.data_ptr() - a.data_ptr()) % size or any(s % row for s in leading):
        return False
    off = (b.data_ptr() - a.data_ptr()) // size
    run_a, run_b = (a.shape[-2] - 1) * a.stride(-2) + HEAD_DIM, (b.shape[-2] - 1) * b.stride(-2) + HEAD_DIM
    return (run_a <= off and off + run_b <= row) or (run_b <= -off and -off + run_a <= row)


def disjoint(a: torch.Tensor, b: torch.Tensor) -> bool:
    """False when two tensors of rows may have an element in common."""
    if not a.numel() or not b.numel():
        return True
    (a0, a1), (b0, b1) = extent(a), extent(b)
    return a1 <= b0 or b1 <= a0 or _share_rows(a, b)


def check_out(out: torch.Tensor, shape, dtype, device, what: str) -> None:
    """``out`` is a tensor of this shape, type and device whose elements are all different places."""
    if not isinstance(out, torch.Tensor) or tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != device:
        raise ValueError(f"{what} must be a {tuple(shape)} tensor of {dtype} on {device}")
    axes = sorted((s, n) for s, n in zip(out.stride(), out.shape) if n > 1)
    reach = 0
    for s, n in axes:
        if s <= reach:
            raise ValueError(f"{what} must not overlap itself")
        reach += s * (n - 1)
