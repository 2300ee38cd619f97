"""Host logic of prompt attention: the work list covers every (query row, visible key) pair once."""

import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from turbopolar_b200 import _lib, build
    build.build()
    return _lib.lib()


def _plan(lib, q_lens, k_lens, hq, hkv):
    from turbopolar_b200 import _lib
    n = len(q_lens)
    arr = ctypes.c_int64 * max(1, n)
    plan = _lib.PromptPlan()
    args = (arr(*q_lens), arr(*k_lens), n, hq, hkv, plan)
    _lib.check(lib.tp_prompt_plan_make(*args, None, 0))
    words = (ctypes.c_int32 * max(1, plan.words))()
    _lib.check(lib.tp_prompt_plan_make(*args, words, plan.words))
    w = list(words)
    items = [w[8 * i:8 * i + 8] for i in range(plan.items)]
    rest = w[8 * plan.items:]
    return plan, items, [rest[4 * i:4 * i + 4] for i in range(plan.merges)]


CASES = [
    ([1], [1]), ([37], [37]), ([16384], [16384]), ([2000, 0, 5, 129], [2000, 0, 5, 129]),
    ([1, 1, 1, 1], [8192, 5001, 3001, 8001]), ([1], [100000]), ([300], [20]), ([7, 0, 4], [0, 9, 3]),
    ([512], [9000]), ([1] * 70, list(range(1, 7001, 100))), ([0], [0]), ([], []), ([255, 257, 31], [600, 257, 31]),
]


@pytest.mark.parametrize("heads", [(32, 8), (8, 8), (12, 4), (14, 2), (128, 1)])
@pytest.mark.parametrize("q_lens,k_lens", CASES)
def test_items_cover_every_visible_pair_once(lib, q_lens, k_lens, heads):
    hq, hkv = heads
    plan, items, merges = _plan(lib, q_lens, k_lens, hq, hkv)
    tile = 128 // (hq // hkv)
    q_off, k_off = 0, 0
    seqs = []
    for q, k in zip(q_lens, k_lens):
        seqs.append((q_off, q, k_off, k))
        q_off, k_off = q_off + q, k_off + k
    assert (plan.q_tokens, plan.k_tokens) == (q_off, k_off)
    seen = {}
    cost = []
    for q_row, q_tokens, sees, k_row, k_begin, k_end, slot, _ in items:
        assert 1 <= q_tokens <= plan.block_tokens <= 2 * tile
        qa, q, ka, k = next(s for s in seqs if s[0] <= q_row < s[0] + s[1])
        assert q_row + q_tokens <= qa + q and k_row == ka and 0 <= k_begin <= k_end <= k
        assert k_begin % 128 == 0
        a = q_row - qa
        assert sees == a + k - q + 1
        seen.setdefault((q_row, q_tokens), []).append((k_begin, k_end, slot))
        cost.append(-(-(k_end - k_begin) // 128))
        # Keys of the tiles that some row does not see whole fit the kernel's list.
        whole = min(sees, k_end) - k_begin
        assert k_end - k_begin - (0 if whole <= 0 else whole // 128 * 128) <= 384
    assert cost == sorted(cost, reverse=True)
    assert sum(n for _, n in seen) == q_off
    by_slot = {}
    for (q_row, q_tokens), parts in seen.items():
        parts.sort()
        qa, q, ka, k = next(s for s in seqs if s[0] <= q_row < s[0] + s[1])
        last = max(0, q_row - qa + k - q + q_tokens)
        assert parts[0][0] == 0 and parts[-1][1] == last
        assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
        if len(parts) == 1:
            assert parts[0][2] == -1
        else:
            by_slot[(q_row, q_tokens)] = sorted(p[2] for p in parts)
    assert {(m[0], m[1]): list(range(m[2], m[2] + m[3])) for m in merges} == by_slot
    slots = sorted(s for v in by_slot.values() for s in v)
    assert slots == list(range(len(slots)))
    assert plan.workspace_bytes == 256 + len(slots) * hkv * 256 * (512 + 8)


def test_few_rows_over_long_keys_fill_one_wave(lib):
    plan, items, merges = _plan(lib, [1, 1, 1, 1], [8192, 5001, 3001, 8001], 32, 8)
    assert 100 <= plan.items * 8 <= 148 and plan.merges == 4
    plan, items, _ = _plan(lib, [1], [131072], 32, 8)
    assert 100 <= plan.items * 8 <= 148


def test_plan_refusals(lib):
    from turbopolar_b200 import _lib
    plan = _lib.PromptPlan()
    one = (ctypes.c_int64 * 1)(5)
    neg = (ctypes.c_int64 * 1)(-1)
    big = (ctypes.c_int64 * 1)(2 ** 31)
    for args in ((neg, one, 1, 8, 4), (one, neg, 1, 8, 4), (one, one, 1, 7, 4), (one, one, 1, 8, 0), (big, one, 1, 8, 4),
                 (None, one, 1, 8, 4), (one, one, -1, 8, 4)):
        assert lib.tp_prompt_plan_make(*args, plan, None, 0) == _lib.TP_ERR_INVALID
    assert lib.tp_prompt_plan_make(one, one, 1, 129, 1, plan, None, 0) == _lib.TP_ERR_UNSUPPORTED
    words = (ctypes.c_int32 * 4)()
    assert lib.tp_prompt_plan_make(one, one, 1, 8, 4, plan, words, 4) == _lib.TP_ERR_INVALID
    # Arguments of the call itself, before any launch.
    _lib.check(lib.tp_prompt_plan_make(one, one, 1, 8, 4, plan, None, 0))
    rows = _lib.PromptRows(dtype=_lib.TP_F32)
    p = ctypes.c_void_p(4096)
    assert lib.tp_prompt_attention(plan, p, rows, p, p, p, 0.1, p, p, 1 << 20, None) == _lib.TP_ERR_INVALID
    rows.dtype = _lib.TP_F16
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert lib.tp_prompt_attention(plan, p, rows, p, p, p, scale, p, p, 1 << 20, None) == _lib.TP_ERR_INVALID
    assert lib.tp_prompt_attention(plan, p, rows, p, p, p, 0.1, ctypes.c_void_p(8), p, 1 << 20, None) == _lib.TP_ERR_INVALID
    assert lib.tp_prompt_attention(plan, p, rows, p, p, p, 0.1, p, p, 8, None) == _lib.TP_ERR_INVALID
