"""Causal attention of packed prompts with grouped query heads (``tp_prompt_attention``).

The reference's adapter runs MLX's dense attention over the decompressed history for every prompt
chunk (``benchmarks/turbopolar_fast_attention.py:56-86``); here the sequences of a batch are packed
row after row and one call attends all of them, each over its own keys.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _lib
from ._checks import HEAD_DIM, check_out, disjoint, launch, refuse_gradients

_CODES = {torch.float16: _lib.TP_F16, torch.bfloat16: _lib.TP_BF16}
_I64x2 = ctypes.c_int64 * 2


class PromptPlan:
    """Work list of :func:`prompt_attention` for sequences of given lengths.

    ``q_lens`` are the numbers of query tokens, ``k_lens`` those of key tokens (``q_lens`` if not
    given).  Query ``a`` of a sequence sees keys ``j <= a + k_len - q_len``: a whole prompt with
    equal lengths, the last rows of a history with ``k_len > q_len`` (one row: a decode step).
    Lengths of zero are allowed, and rows of a sequence with ``k_len < q_len`` that see nothing
    give 0.  A plan is made once and serves every layer; it owns the work list and the workspace, so calls
    that may run at the same time (on several streams) need a plan each, and a CUDA graph that captured calls
    needs the plan as long as it is replayed.  Making one takes 50 to 90 us of host time (a blocking copy and a
    cleared workspace), so a decode step of single tokens pays that once for its layers.
    """

    def __init__(self, q_lens: Sequence[int], k_lens: Optional[Sequence[int]] = None, *, num_q_heads: int,
                 num_kv_heads: int, device=None):
        self.q_lens = [int(n) for n in q_lens]
        self.k_lens = self.q_lens if k_lens is None else [int(n) for n in k_lens]
        if len(self.k_lens) != len(self.q_lens):
            raise ValueError(f"{len(self.q_lens)} query lengths and {len(self.k_lens)} key lengths")
        n = len(self.q_lens)
        lens = ctypes.c_int64 * max(1, n)
        args = (lens(*self.q_lens), lens(*self.k_lens), n, int(num_q_heads), int(num_kv_heads))
        self.struct = _lib.PromptPlan()
        lib = _lib.lib()
        _lib.check(lib.tp_prompt_plan_make(*args, self.struct, None, 0))
        words = torch.zeros(max(1, self.struct.words), dtype=torch.int32)
        _lib.check(lib.tp_prompt_plan_make(*args, self.struct, words.data_ptr(), words.numel()))
        self.num_q_heads, self.num_kv_heads = int(num_q_heads), int(num_kv_heads)
        self.device = torch.device("cuda" if device is None else device)
        if self.device.type != "cuda":
            raise ValueError("TurboPolar B200 kernels need a CUDA device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._workspace = torch.zeros(self.struct.workspace_bytes, dtype=torch.uint8, device=self.device)
        self._words = words.to(self.device)  # waits, so any stream may use both
        self._stream = torch.cuda.current_stream(self.device).cuda_stream
        self._ptrs = (self._words.data_ptr(), self._workspace.data_ptr(), self._workspace.numel())
        self._layouts: dict = {}  # checked row layouts, by strides and types

    @property
    def device_error(self) -> torch.Tensor:
        """The error word on the device, an int32 tensor ``(1,)``."""
        return self._workspace[:4].view(torch.int32)

    def read_device_error(self) -> int:
        """0, or 1 when a wait in a kernel of this plan ran out (outputs unusable); synchronises."""
        return int(self.device_error.item())

    def _layout(self, q, k, v) -> _lib.PromptRows:
        for name, x, tokens, heads in (("q", q, self.struct.q_tokens, self.num_q_heads),
                                       ("k", k, self.struct.k_tokens, self.num_kv_heads),
                                       ("v", v, self.struct.k_tokens, self.num_kv_heads)):
            if x.dim() == 3 and x.shape[2] != HEAD_DIM:
                raise NotImplementedError("prompt_attention only supports head_dim == 128")
            if tuple(x.shape) != (tokens, heads, HEAD_DIM):
                raise ValueError(f"{name} must be ({tokens}, {heads}, 128) for this plan, got {tuple(x.shape)}")
            if x.device != self.device:
                raise ValueError(f"{name} must be on the plan's device {self.device}")
            if x.dtype not in _CODES or x.dtype != q.dtype:
                raise ValueError(f"q, k and v must all be float16 or bfloat16, got {q.dtype}, {k.dtype} and {v.dtype}")
        return _lib.PromptRows(*(_I64x2(x.stride(0), x.stride(1)) for x in (q, k, v)), _CODES[q.dtype])


def _readable(x: torch.Tensor) -> bool:
    """Rows that tensor copies can fetch: contiguous channels, 16-byte boundaries, no broadcast axes."""
    return x.stride(2) == 1 and not x.data_ptr() & 15 and all(
        s % 8 == 0 and s >= HEAD_DIM for s, n in zip(x.stride()[:2], x.shape) if n > 1)


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if _readable(x) else x.clone(memory_format=torch.contiguous_format)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PromptPlan, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the plan's packed sequences.

    ``q`` is ``(sum of q_lens, H_q, 128)``, ``k`` and ``v`` ``(sum of k_lens, H_kv, 128)``, float16
    or bfloat16; query head ``h`` reads KV head ``h // (H_q // H_kv)``.  Token and head strides are
    free (multiples of 8 elements; other layouts are copied first).  Returns
    ``(sum of q_lens, H_q, 128)`` of the same type, in ``out`` if given (contiguous).  Scores,
    maxima, sums and outputs are float32; weights are rounded to the input type for the second
    product.  A key that a row does not see has no influence on it, whatever it holds.
    ``scale`` (positive) defaults to ``1 / sqrt(128)``.
    """
    refuse_gradients(q, k, v)
    key = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype,
           v.device)
    layout = plan._layouts.get(key)
    qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if layout is None or (qp | kp | vp) & 15:
        layout = plan._layout(q, k, v)
        if not (_readable(q) and _readable(k) and _readable(v)):
            return prompt_attention(_rows(q), _rows(k), _rows(v), plan, scale, out)
        if len(plan._layouts) >= 64:
            plan._layouts.clear()
        plan._layouts[key] = layout
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        check_out(out, q.shape, q.dtype, q.device, "out")
        if not out.is_contiguous() or out.data_ptr() & 15:
            raise ValueError("out must be contiguous and 16-byte aligned")
        if not (disjoint(out, q) and disjoint(out, k) and disjoint(out, v)):
            raise ValueError("out shares memory with an input")
    words, workspace, size = plan._ptrs
    if torch._C._cuda_getCurrentRawStream(plan.device.index) != plan._stream:
        here = torch.cuda.current_stream(plan.device)  # keep the plan's buffers until this stream is done with them
        plan._words.record_stream(here)
        plan._workspace.record_stream(here)
    status = launch(plan.device, _lib.lib().tp_prompt_attention, plan.struct, words, layout, qp, kp, vp,
                    HEAD_DIM ** -0.5 if scale is None else scale, out.data_ptr(), workspace, size)
    if status:
        _lib.check(status)
    return out
