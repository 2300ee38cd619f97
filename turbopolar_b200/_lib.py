"""ctypes binding of ``libturbopolar.so`` (declared in ``include/turbopolar.h``).

The library is loaded from this package folder.  There is no CPU fallback: a missing library
or a machine without CUDA raises on first use.
"""

from __future__ import annotations

import ctypes
import os
import threading

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libturbopolar.so")

TP_OK, TP_ERR_INVALID, TP_ERR_UNSUPPORTED, TP_ERR_CUDA = 0, 1, 2, 3
TP_F16, TP_F32, TP_BF16 = 0, 1, 2
PARTIAL_FLOATS = 130
STATE_WORDS = 6

EXPORTED = (
    "tp_row_bytes", "tp_unit_bytes", "tp_encode_pages", "tp_append", "tp_decode_attention_workspace_size",
    "tp_decode_attention", "tp_decode_attention_dense_v", "tp_decode_step", "tp_decode_attention_noalloc", "tp_noalloc_error", "tp_combine_partials", "tp_fused_scores", "tp_decode_pages",
    "tp_export_pages", "tp_import_pages", "tp_last_error", "tp_version",
    "tp_exchange_bytes", "tp_ipc_alloc", "tp_ipc_open", "tp_ipc_close", "tp_ipc_free",
    "tp_decode_attention_sharded", "tp_decode_step_sharded",
    "tp_norm_rope", "tp_prompt_plan_make", "tp_prompt_attention",
    "tp_tree_attention", "tp_tree_attention_workspace_size",
)
MAX_RANKS = 8


class Format(ctypes.Structure):
    _fields_ = [("l1_bits", ctypes.c_int32), ("deep_bits", ctypes.c_int32),
                ("split_dim", ctypes.c_int32), ("int8_radii", ctypes.c_int32)]


class PagePool(ctypes.Structure):
    """tp_page_pool: page blocks in the kernels' layout."""
    _fields_ = [("pages", ctypes.c_void_p), ("radii_scales", ctypes.c_void_p),
                ("num_kv_heads", ctypes.c_int32), ("page_capacity", ctypes.c_int32),
                ("fmt", Format)]


class BlockStore(ctypes.Structure):
    """tp_block_store: pages in the reference's block-storage layout."""
    _fields_ = [("radii", ctypes.c_void_p), ("radii_scales", ctypes.c_void_p),
                ("angle_codes_l1", ctypes.c_void_p), ("angle_codes_deep", ctypes.c_void_p),
                ("v_codes", ctypes.c_void_p), ("v_scales", ctypes.c_void_p),
                ("num_kv_heads", ctypes.c_int32), ("page_capacity", ctypes.c_int32),
                ("fmt", Format)]


def fmt_struct(fmt: dict) -> Format:
    return Format(fmt["l1_bits"], fmt["deep_bits"], fmt["split_dim"], fmt["int8_radii"])


def empty_pool(heads: int, fmt: dict) -> PagePool:
    """A pool of capacity 0 (attention over the dense tail only)."""
    return PagePool(None, None, heads, 0, fmt_struct(fmt))


class Tail(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("dtype", ctypes.c_int32)]


class State(ctypes.Structure):
    _fields_ = [("n_pages", ctypes.c_int32), ("tail_len", ctypes.c_int32),
                ("seq_len", ctypes.c_int32), ("first_page", ctypes.c_int32)]


class Exchange(ctypes.Structure):
    _fields_ = [("world", ctypes.c_int32), ("rank", ctypes.c_int32), ("buffers", ctypes.c_void_p * 8)]


class RopeLayout(ctypes.Structure):
    """tp_rope_layout: sizes, types and strides of a tp_norm_rope call."""
    _fields_ = [("batch", ctypes.c_int32), ("tokens", ctypes.c_int32), ("q_heads", ctypes.c_int32),
                ("k_heads", ctypes.c_int32), ("dtype", ctypes.c_int32), ("weight_dtype", ctypes.c_int32),
                ("table_dtype", ctypes.c_int32), ("interleaved", ctypes.c_int32), ("q_in", ctypes.c_int64 * 3),
                ("k_in", ctypes.c_int64 * 3), ("q_out", ctypes.c_int64 * 3), ("k_out", ctypes.c_int64 * 3),
                ("row_stride", ctypes.c_int64), ("pos_strides", ctypes.c_int64 * 2), ("table_rows", ctypes.c_int32),
                ("batch_rows", ctypes.c_int32), ("pos64", ctypes.c_int32), ("eps", ctypes.c_float)]


class PromptPlan(ctypes.Structure):
    """tp_prompt_plan: the sizes of a prompt-attention work list."""
    _fields_ = [("num_q_heads", ctypes.c_int32), ("num_kv_heads", ctypes.c_int32), ("q_tokens", ctypes.c_int64),
                ("k_tokens", ctypes.c_int64), ("items", ctypes.c_int32), ("merges", ctypes.c_int32),
                ("block_tokens", ctypes.c_int32), ("words", ctypes.c_size_t), ("workspace_bytes", ctypes.c_size_t)]


class PromptRows(ctypes.Structure):
    """tp_prompt_rows: token and head strides of packed q, k and v, and their type."""
    _fields_ = [("q", ctypes.c_int64 * 2), ("k", ctypes.c_int64 * 2), ("v", ctypes.c_int64 * 2),
                ("dtype", ctypes.c_int32)]


class Drafts(ctypes.Structure):
    """tp_drafts: sizes, types and strides of a tp_tree_attention call."""
    _fields_ = [("batch", ctypes.c_int32), ("num_q_heads", ctypes.c_int32), ("n_drafts", ctypes.c_int32),
                ("q_dtype", ctypes.c_int32), ("kv_dtype", ctypes.c_int32), ("q", ctypes.c_int64 * 3),
                ("k", ctypes.c_int64 * 3), ("v", ctypes.c_int64 * 3), ("mask", ctypes.c_int64 * 2), ("d_state", ctypes.c_void_p)]


_lib = None
_lock = threading.Lock()


def _declare(lib):
    P, I32, I64, SZ, F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float
    sig = {
        "tp_row_bytes": (ctypes.c_int, [ctypes.POINTER(Format), ctypes.POINTER(I32), ctypes.POINTER(I32)]),
        "tp_unit_bytes": (ctypes.c_int, [ctypes.POINTER(Format), ctypes.POINTER(I32)]),
        "tp_encode_pages": (ctypes.c_int, [ctypes.POINTER(PagePool), P, P, I32, I64, I64, I64, I32, I32, P, P]),
        "tp_append": (ctypes.c_int, [ctypes.POINTER(PagePool), ctypes.POINTER(Tail), P, P, P, I32, I64, I64, I32, P]),
        "tp_decode_attention_workspace_size": (SZ, [I32, I32]),
        "tp_decode_attention": (ctypes.c_int, [ctypes.POINTER(PagePool), ctypes.POINTER(Tail), State, P, P, I32, I32,
                                               F, P, P, P, SZ, P]),
        "tp_decode_attention_dense_v": (ctypes.c_int, [ctypes.POINTER(PagePool), State, P, I64, I64, P, I32, I32, F,
                                                       P, P, P, SZ, P]),
        "tp_decode_step": (ctypes.c_int, [ctypes.POINTER(PagePool), ctypes.POINTER(Tail), P, P, P, I32, I64, P, I32,
                                          I32, F, P, P, P, SZ, P]),
        "tp_decode_attention_noalloc": (ctypes.c_int, [ctypes.POINTER(PagePool), ctypes.POINTER(Tail), State, P, P,
                                                       I32, I32, F, P, P, P]),
        "tp_noalloc_error": (ctypes.c_int, [ctypes.POINTER(I32), P]),
        "tp_combine_partials": (ctypes.c_int, [P, I32, I32, P, P]),
        "tp_fused_scores": (ctypes.c_int, [ctypes.POINTER(PagePool), I32, P, I32, I32, F, P, P]),
        "tp_decode_pages": (ctypes.c_int, [ctypes.POINTER(PagePool), I32, I32, P, P, P]),
        "tp_export_pages": (ctypes.c_int, [ctypes.POINTER(PagePool), I32, I32, ctypes.POINTER(BlockStore), P]),
        "tp_import_pages": (ctypes.c_int, [ctypes.POINTER(PagePool), I32, I32, ctypes.POINTER(BlockStore), P]),
        "tp_exchange_bytes": (SZ, [I32, I32]),
        "tp_ipc_alloc": (ctypes.c_int, [SZ, ctypes.POINTER(ctypes.c_void_p), P]),
        "tp_ipc_open": (ctypes.c_int, [P, ctypes.POINTER(ctypes.c_void_p)]),
        "tp_ipc_close": (ctypes.c_int, [P]),
        "tp_ipc_free": (ctypes.c_int, [P]),
        "tp_decode_attention_sharded": (ctypes.c_int, [ctypes.POINTER(PagePool), ctypes.POINTER(Tail), State, P, P,
                                                       I32, I32, F, P, ctypes.POINTER(Exchange), P, SZ, P]),
        "tp_decode_step_sharded": (ctypes.c_int, [ctypes.POINTER(PagePool), ctypes.POINTER(Tail), P, P, P, I32, I64, P,
                                                  I32, I32, F, P, ctypes.POINTER(Exchange), P, SZ, P]),
        "tp_norm_rope": (ctypes.c_int, [ctypes.POINTER(RopeLayout), P, P, P, P, P, P, P, P, P, P]),
        "tp_prompt_plan_make": (ctypes.c_int, [P, P, I32, I32, I32, ctypes.POINTER(PromptPlan), P, SZ]),
        "tp_prompt_attention": (ctypes.c_int, [ctypes.POINTER(PromptPlan), P, ctypes.POINTER(PromptRows), P, P, P, F,
                                               P, P, SZ, P]),
        "tp_tree_attention_workspace_size": (SZ, [I32, I32, I32]),
        "tp_tree_attention": (ctypes.c_int, [ctypes.POINTER(PagePool), ctypes.POINTER(Tail), State,
                                             ctypes.POINTER(Drafts), P, P, P, P, F, P, P, SZ, P]),
        "tp_last_error": (ctypes.c_char_p, []),
        "tp_version": (ctypes.c_int, []),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args


def lib():
    """The loaded library (loaded once).  Raises RuntimeError when it has not been built."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                if not os.path.exists(LIB_PATH):
                    raise RuntimeError(
                        f"libturbopolar.so not found at {LIB_PATH}; build it with "
                        "`python -m turbopolar_b200.build` (CUDA 12.9 nvcc, sm_100a)")
                handle = ctypes.CDLL(LIB_PATH)
                _declare(handle)
                _lib = handle
    return _lib


def check(status: int) -> None:
    """Map a tp_status to the reference's exception types."""
    if status == TP_OK:
        return
    msg = lib().tp_last_error().decode(errors="replace")
    if status == TP_ERR_INVALID:
        raise ValueError(msg)
    if status == TP_ERR_UNSUPPORTED:
        raise NotImplementedError(msg)
    raise RuntimeError(msg)
