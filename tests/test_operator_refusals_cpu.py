"""Arguments that tp_norm_rope and tp_tree_attention refuse, each before any CUDA call.

The pointers are addresses that nothing dereferences on the host."""

import ctypes

import pytest

P = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    from turbopolar_b200 import _lib, build
    build.build()
    return _lib.lib()


def _rope(**change):
    from turbopolar_b200 import _lib
    heads = {"q": change.get("q_heads", 8), "k": change.get("k_heads", 4)}
    fields = dict(batch=1, tokens=3, q_heads=8, k_heads=4, dtype=_lib.TP_F16, weight_dtype=_lib.TP_F32,
                  table_dtype=_lib.TP_F32, interleaved=0, row_stride=64, table_rows=16, batch_rows=0, pos64=0, eps=1e-6)
    for side in ("q", "k"):
        n = heads[side] * 128
        for way in ("in", "out"):
            fields[f"{side}_{way}"] = (ctypes.c_int64 * 3)(3 * n, n, 128)
    fields["pos_strides"] = (ctypes.c_int64 * 2)(0, 1)
    fields.update(change)
    return _lib.RopeLayout(**fields)


@pytest.mark.parametrize("change, pointers, pattern", [
    (dict(dtype=17), {}, "dtype"),
    (dict(weight_dtype=17), {}, "dtype"),
    (dict(table_dtype=-1), {}, "dtype"),
    (dict(tokens=-1), {}, "negative"),
    (dict(batch=-1), {}, "negative"),
    (dict(q_heads=0), {}, "at least one head"),
    (dict(k_heads=0), {}, "at least one head"),
    (dict(q_in=(ctypes.c_int64 * 3)(3072, 1022, 128)), {}, "rows of q must start"),
    (dict(k_out=(ctypes.c_int64 * 3)(1536, 512, 130)), {}, "rows of k_out must start"),
    ({}, dict(q=P(4100)), "rows of q must start"),
    ({}, dict(k=None), "NULL k"),
    ({}, dict(q_out=None), "NULL q_out"),
    ({}, dict(cos=None), "NULL angle table"),
    ({}, dict(sin=None), "NULL angle table"),
    (dict(row_stride=63), {}, "64 elements apart"),
    (dict(table_rows=-1), {}, "64 elements apart"),
    (dict(table_rows=2), {}, "fewer rows than tokens"),
    (dict(batch=2, batch_rows=14), {}, "fewer rows than tokens"),
    (dict(batch=1 << 20, tokens=1 << 20, table_rows=1 << 30), {}, "2\\^31 rows"),
])
def test_norm_rope_refuses(lib, change, pointers, pattern):
    from turbopolar_b200 import _lib
    p = dict(q=P(4096), k=P(8192), q_weight=None, k_weight=None, cos=P(4096), sin=P(4096), positions=None,
             q_out=P(1 << 20), k_out=P(1 << 21))
    p.update(pointers)
    with pytest.raises(ValueError, match=pattern):
        _lib.check(lib.tp_norm_rope(_rope(**change), *p.values(), None))


def test_norm_rope_needs_a_layout_and_accepts_no_tokens(lib):
    from turbopolar_b200 import _lib
    with pytest.raises(ValueError, match="NULL layout"):
        _lib.check(lib.tp_norm_rope(None, *[None] * 9, None))
    for empty in (dict(tokens=0), dict(batch=0)):  # nothing to do, whatever the pointers
        assert lib.tp_norm_rope(_rope(**empty), *[None] * 9, None) == _lib.TP_OK


def _drafts(**change):
    from turbopolar_b200 import _lib
    fields = dict(batch=1, num_q_heads=8, n_drafts=5, q_dtype=_lib.TP_F16, kv_dtype=_lib.TP_F16,
                  q=(ctypes.c_int64 * 3)(5120, 640, 128), k=(ctypes.c_int64 * 3)(2560, 640, 128),
                  v=(ctypes.c_int64 * 3)(2560, 640, 128), mask=(ctypes.c_int64 * 2)(0, 5))
    fields.update(change)
    return _lib.Drafts(**fields)


@pytest.mark.parametrize("change, call, pattern", [
    (dict(batch=0), {}, "batch does not divide"),
    (dict(batch=3), {}, "batch does not divide"),
    (dict(num_q_heads=6), {}, "divisible"),
    (dict(num_q_heads=0), {}, "divisible"),
    (dict(n_drafts=0), {}, "\\[1, 256\\]"),
    (dict(n_drafts=257), {}, "\\[1, 256\\]"),
    (dict(q_dtype=2), {}, "float16 or float32"),
    (dict(kv_dtype=9), {}, "float16 or float32"),
    (dict(q=(ctypes.c_int64 * 3)(5120, 640, 124)), {}, "16-byte boundaries"),
    (dict(v=(ctypes.c_int64 * 3)(2560, 636, 128)), {}, "16-byte boundaries"),
    ({}, dict(k=P(4104)), "16-byte boundaries"),
    ({}, dict(out=P(4104)), "16-byte boundaries"),
    ({}, dict(q=None), "NULL argument"),
    ({}, dict(mask=None), "NULL argument"),
    ({}, dict(out=None), "NULL argument"),
    ({}, dict(scale=0.0), "scale must be positive"),
    ({}, dict(scale=-1.0), "scale must be positive"),
    ({}, dict(scale=float("nan")), "scale must be positive"),
    ({}, dict(scale=float("inf")), "scale must be positive"),
    ({}, dict(state=(-1, 0, 0, 0)), "cache state"),
    ({}, dict(state=(5, 0, 320, 0)), "cache state"),
    ({}, dict(state=(2, 64, 192, 0)), "cache state"),
    ({}, dict(state=(2, 0, 128, 1)), "cache state"),
    ({}, dict(state=(2, 3, 132, 0)), "seq_len"),
    ({}, dict(state=(2, 0, -1, 0)), "seq_len"),
    ({}, dict(tail=False), "tail buffers"),
    ({}, dict(tail_dtype=2), "tail dtype"),
    ({}, dict(workspace=None), "workspace too small"),
    ({}, dict(workspace_bytes=1024), "workspace too small"),
])
def test_tree_attention_refuses(lib, change, call, pattern):
    from turbopolar_b200 import _lib
    pool = _lib.PagePool(P(1 << 20), None, 4, 4, _lib.Format(4, 4, 64, 0))
    a = dict(state=(2, 3, 131, 0), q=P(4096), k=P(4096), v=P(4096), mask=P(4096), scale=0.1, out=P(1 << 22), workspace=P(1 << 24),
             workspace_bytes=1 << 30, tail=True, tail_dtype=_lib.TP_F16)
    a.update(call)
    tail = _lib.Tail(k=P(4096), v=P(8192), dtype=a["tail_dtype"]) if a["tail"] else None
    with pytest.raises(ValueError, match=pattern):
        _lib.check(lib.tp_tree_attention(pool, tail, _lib.State(*a["state"]), _drafts(**change), a["q"], a["k"], a["v"],
                                         a["mask"], a["scale"], a["out"], a["workspace"], a["workspace_bytes"], None))


def test_tree_attention_workspace_size_of_impossible_sizes_is_zero(lib):
    size = lib.tp_tree_attention_workspace_size
    for sizes in ((0, 8, 5), (4, 0, 5), (4, 6, 5), (4, 8, 0), (4, 8, 257), (-4, 8, 5)):
        assert size(*sizes) == 0
    assert 0 < size(4, 8, 1) <= size(4, 8, 5) <= size(4, 8, 256)
