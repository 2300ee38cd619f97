"""Norms of the query and key heads with the position rotation, in one kernel (``tp_norm_rope``).

The step before every attention call: the reference leaves the rotation to MLX
(``benchmarks/turbopolar_fast_attention.py:247-278``, ``self.rope``); models with per-head norms
apply those first.  One call reads the rows of both projections (slices of a fused projection's
output are taken as they are) and writes rotated queries and keys.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._checks import HEAD_DIM, check_out, disjoint, launch, refuse_gradients

_CODES = {torch.float16: _lib.TP_F16, torch.float32: _lib.TP_F32, torch.bfloat16: _lib.TP_BF16}
_I64x2 = ctypes.c_int64 * 2
_I64x3 = ctypes.c_int64 * 3


def _strides(x: torch.Tensor):
    # The stride of an axis of one entry is arbitrary and never used.
    st = [s if n > 1 else 0 for s, n in zip(x.stride(), x.shape)]
    return _I64x3(0, st[0], st[1]) if len(st) == 3 else _I64x3(st[0], st[1], st[2])


def _aligned(x: torch.Tensor) -> bool:
    """Rows of 128 contiguous channels on boundaries of four elements."""
    return x.stride(-1) == 1 and not any(s & 3 for s, n in zip(x.stride()[:-1], x.shape) if n > 1) \
        and not x.data_ptr() & (4 * x.element_size() - 1)


def _check_rows_out(out, x, others, what: str) -> None:
    check_out(out, x.shape, x.dtype, x.device, what)
    if not _aligned(out):
        raise ValueError(f"{what} needs contiguous channels and strides that are multiples of 4 elements")
    same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
    if not (same or disjoint(out, x)) or not all(disjoint(out, y) for y in others if y is not None):
        raise ValueError(f"{what} overlaps an input; it may only be its own input, whole")


# Checked layouts by shapes, strides, types and devices (no data, no addresses): a model's layers call
# with few different ones, and checking them anew would cost more than the kernel takes.
_layouts: dict = {}


def _kind(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if _aligned(x) else x.clone(memory_format=torch.contiguous_format)


def _table(x: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if x is None else x.clone(memory_format=torch.contiguous_format)


def _checked(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved):
    """The layout of a call with outputs to be made and the alignment bits of its rows, or None where
    inputs have to be copied first.  Raises for everything that does not fit together."""
    dt = q.dtype
    if q.dim() not in (3, 4) or k.dim() != q.dim() or q.shape[:-2] != k.shape[:-2]:
        raise ValueError(f"q and k must be (T, H, 128) or (B, T, H, 128) of the same tokens, got {tuple(q.shape)} "
                         f"and {tuple(k.shape)}")
    if q.shape[-1] != HEAD_DIM or k.shape[-1] != HEAD_DIM:
        raise NotImplementedError("norm_rope only supports head_dim == 128")
    if dt not in _CODES or k.dtype != dt:
        raise ValueError(f"q and k must both be float16, bfloat16 or float32, got {dt} and {k.dtype}")
    if not q.is_cuda or k.device != q.device or cos.device != q.device or sin.device != q.device:
        raise ValueError("norm_rope needs q, k, cos and sin on one CUDA device")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != HEAD_DIM // 2 or cos.dtype != sin.dtype \
            or cos.dtype not in _CODES:
        raise ValueError("cos and sin must be (rows, 64) tables of one floating type")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.shape != (HEAD_DIM,) or w.dtype != weights[0].dtype or w.dtype not in _CODES or w.device != q.device:
            raise ValueError("norm weights must be (128,) floating tensors of one dtype on q's device")
    batch, tokens = (1, q.shape[0]) if q.dim() == 3 else (q.shape[0], q.shape[1])
    rows = cos.shape[0]
    pos_strides, pos64, batch_rows = (0, 0), 0, 0
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
            raise ValueError("positions must be an int32 or int64 tensor on q's device")
        if positions.shape == (tokens,):
            pos_strides = (0, positions.stride(0))
        elif q.dim() == 4 and positions.shape == (batch, tokens):
            pos_strides = (positions.stride(0), positions.stride(1))
        else:
            raise ValueError(f"positions must be ({tokens},) or ({batch}, {tokens}), got {tuple(positions.shape)}")
        pos64 = int(positions.dtype == torch.int64)
    elif batch > 1 and rows == batch * tokens:
        batch_rows = tokens
    elif rows < tokens:
        raise ValueError(f"cos and sin have {rows} rows for {tokens} tokens")
    packed = all(w.stride(0) == 1 for w in weights) and cos.stride(1) == 1 and cos.stride() == sin.stride() \
        and (rows < 2 or cos.stride(0) >= HEAD_DIM // 2)
    layout = _lib.RopeLayout(batch, tokens, q.shape[-2], k.shape[-2], _CODES[dt],
                             _CODES[weights[0].dtype] if weights else _lib.TP_F32, _CODES[cos.dtype], int(interleaved),
                             _strides(q), _strides(k), _fresh(q), _fresh(k), cos.stride(0), _I64x2(*pos_strides), rows,
                             batch_rows, pos64, eps)
    bits = 4 * q.element_size() - 1
    odd = any(s & 3 for s in (*layout.q_in, *layout.k_in)) or q.stride(-1) != 1 or k.stride(-1) != 1
    return (layout, bits) if packed and not odd else None


def _fresh(x: torch.Tensor):
    """Strides of a contiguous tensor of x's shape."""
    t, h = x.shape[-3], x.shape[-2]
    return _I64x3(t * h * HEAD_DIM, h * HEAD_DIM, HEAD_DIM)


def norm_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
              positions: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
              k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
              q_out: Optional[torch.Tensor] = None,
              k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Normalise each head of ``q`` and ``k`` and rotate it by its token's position.

    ``q`` is ``(T, H_q, 128)`` or ``(B, T, H_q, 128)``, ``k`` alike with ``H_kv`` heads, in float16,
    bfloat16 or float32; channels contiguous, any other strides.  For each row,
    ``y = x * rsqrt(mean(x^2) + eps) * weight`` (``y = x`` where that weight is ``None``), then the
    pairs ``(y[d], y[d + 64])``, or with ``interleaved`` ``(y[2d], y[2d + 1])``, turn by the angle
    of the token's position: ``(a cos - b sin, b cos + a sin)``.  The arithmetic is float32 and the
    result is rounded once.

    ``cos`` and ``sin`` hold 64 values per row, ``(rows, 64)``.  ``positions`` (int32 or int64,
    ``(T,)`` or ``(B, T)``) selects each token's row; a position outside the table gives NaN rows.
    Without it token ``t`` uses row ``t``, or row ``b * T + t`` of a table of ``B * T`` rows.

    Returns ``(q_out, k_out)``, new contiguous tensors unless given.  ``q_out`` may be ``q`` itself
    and ``k_out`` ``k`` itself (in place); other overlaps are refused.
    """
    refuse_gradients(q, k, cos, sin, q_weight, k_weight)
    key = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device, cos.shape, cos.stride(),
           cos.dtype, cos.device, sin.shape, sin.stride(), sin.dtype, sin.device, eps, interleaved, _kind(positions),
           _kind(q_weight), _kind(k_weight))
    layout = _layouts.get(key)
    if layout is None:
        layout = _checked(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved)
        if layout is None:  # rows or tables that the kernel cannot read in place
            return norm_rope(_rows(q), _rows(k), _table(cos), _table(sin), positions, _table(q_weight), _table(k_weight),
                             eps, interleaved, q_out, k_out)
        if len(_layouts) >= 1024:
            _layouts.clear()
        _layouts[key] = layout
    qp, kp = q.data_ptr(), k.data_ptr()
    if (qp | kp) & layout[1]:
        return norm_rope(_rows(q), _rows(k), cos, sin, positions, q_weight, k_weight, eps, interleaved, q_out, k_out)
    given = q_out is not None or k_out is not None
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_rows_out(q_out, q, (k, cos, sin, positions, q_weight, k_weight), "q_out")
    if k_out is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        _check_rows_out(k_out, k, (q, cos, sin, positions, q_weight, k_weight), "k_out")
    struct = layout[0]
    if given:
        if not disjoint(q_out, k_out):
            raise ValueError("q_out and k_out overlap")
        struct = _lib.RopeLayout.from_buffer_copy(struct)
        struct.q_out, struct.k_out = _strides(q_out), _strides(k_out)
    status = launch(q.device, _lib.lib().tp_norm_rope, struct, qp, kp, None if q_weight is None else q_weight.data_ptr(),
                    None if k_weight is None else k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                    None if positions is None else positions.data_ptr(), q_out.data_ptr(), k_out.data_ptr())
    if status:
        _lib.check(status)
    return q_out, k_out
