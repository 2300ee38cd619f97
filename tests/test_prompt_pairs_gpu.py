"""prompt_attention on batches whose items are pairs of query tiles (enough rows and heads to fill the GPU):
masked non-finite keys and values, rows that see nothing, moving maxima, and split key ranges.  Tolerances are those
of the formula's tests."""

import pytest
import torch

from test_prompt_gpu import U, _check, _inputs

pytestmark = pytest.mark.gpu


def _pairs(q_lens, k_lens, hq, hkv):
    from turbopolar_b200 import PromptPlan
    plan = PromptPlan(q_lens, k_lens, num_q_heads=hq, num_kv_heads=hkv)
    assert plan.struct.block_tokens == 2 * (128 // (hq // hkv))
    return plan


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(64, 64), (64, 32)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_keys_have_no_influence(bad, heads, dtype):
    from turbopolar_b200 import prompt_attention
    q_lens, k_lens = [70, 333, 290, 1], [70, 333, 600, 150]
    starts = [0, 70, 403, 1003]
    q, k, v = _inputs(q_lens, k_lens, *heads, dtype)
    plan = _pairs(q_lens, k_lens, *heads)
    clean = prompt_attention(q, k, v, plan)
    kb, vb = k.clone(), v.clone()
    kb[70:403], vb[70:403] = bad, bad   # the whole second sequence
    out = prompt_attention(q, kb, vb, plan)
    assert torch.equal(out[:70], clean[:70]) and torch.equal(out[403:], clean[403:])
    vb = v.clone()
    first_bad = {0: 69, 70: 200, 403: 399}   # (first key of a sequence): its first key with a bad value
    for first, j in first_bad.items():
        vb[first + j, :, 5] = bad
    vb[70 + 290, :, 5] = bad
    out = prompt_attention(q, k, vb, plan)
    assert plan.read_device_error() == 0
    qa = 0
    for nq, nk, first in zip(q_lens, k_lens, starts):
        rows = max(0, first_bad.get(first, nk) - (nk - nq))   # rows that see no bad key
        assert torch.equal(out[qa:qa + rows], clean[qa:qa + rows])
        if rows < nq:
            later = out[qa + rows:qa + nq]
            assert not torch.isfinite(later[:, :, 5]).any()
            rest = [c for c in range(128) if c != 5]
            err = (later[:, :, rest].double() - clean[qa + rows:qa + nq][:, :, rest].double()).abs()
            assert (err <= 4 * U[dtype] * 6).all()   # values are below 6; weights rounded or not
        qa += nq


@pytest.mark.parametrize("heads", [(64, 64), (64, 32), (96, 32)])
def test_rows_that_see_nothing_give_zero(heads):
    from turbopolar_b200 import prompt_attention
    q_lens, k_lens = [700, 4, 9, 0, 300], [20, 0, 9, 50, 300]
    q, k, v = _inputs(q_lens, k_lens, *heads, torch.float16)
    out = prompt_attention(q, k, v, _pairs(q_lens, k_lens, *heads))
    _check(out, q, k, v, q_lens, k_lens, 128 ** -0.5)
    assert (out[:680] == 0).all() and (out[700:704] == 0).all()


def test_large_scores_and_moving_maxima():
    from turbopolar_b200 import prompt_attention
    n = 1500
    q, k, v = _inputs([n], [n], 32, 16, torch.float16)
    k = (k * torch.linspace(0.1, 6, n, device="cuda")[:, None, None]).half()
    out = prompt_attention(q, k, v, _pairs([n], [n], 32, 16), scale=1.0)
    _check(out, q, k, v, [n], [n], 1.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_split_key_ranges(dtype):
    # One block with far more keys than the others: its pair of tiles is split over several items.
    from turbopolar_b200 import prompt_attention
    q_lens, k_lens = [200] + [9] * 11, [9000] + [9] * 11
    q, k, v = _inputs(q_lens, k_lens, 32, 32, dtype)
    plan = _pairs(q_lens, k_lens, 32, 32)
    assert plan.struct.merges > 0
    out = prompt_attention(q, k, v, plan)
    assert plan.read_device_error() == 0
    _check(out, q, k, v, q_lens, k_lens, 128 ** -0.5)
    assert torch.equal(out, prompt_attention(q, k, v, plan))
