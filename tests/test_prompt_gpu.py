"""prompt_attention against its formula in float64.

Tolerance per element, u = 2^-11 (float16) or 2^-8 (bfloat16), W = sum_j w_j |v_j| with the exact weights:
  u |out|                      the output's rounding
  u W                          each weight's rounding to 16 bits
  2 eps W, eps = 2^-18 scale max_j sum_d |q_d k_jd| + 2^-20
                               scores: 8 accumulations of 16 products, each off by at most 2^-22 of the sum's
                               size, and as much inside a product group; the exponential and its argument;
                               once in the numerator and once in the sum
  n 2^-25 max|v|               weights below the normal range of float16 (the row's largest is at least 1)
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _expect(q, k, v, q_lens, k_lens, scale):
    """(out, bound) in float64."""
    hq, hkv = q.shape[1], k.shape[1]
    g = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    u = U[q.dtype]
    qa = ka = 0
    for nq, nk in zip(q_lens, k_lens):
        if nq and nk:
            for h in range(hq):
                qq = q[qa:qa + nq, h].double()
                kk, vv = k[ka:ka + nk, h // g].double(), v[ka:ka + nk, h // g].double()
                hidden = torch.arange(nk, device="cuda") > torch.arange(nq, device="cuda")[:, None] + (nk - nq)
                s = (qq @ kk.T * scale).masked_fill(hidden, -torch.inf)
                w = torch.nan_to_num(torch.softmax(s, -1))
                o = w @ vv
                big = w @ vv.abs()
                eps = 2.0 ** -18 * scale * (qq.abs() @ kk.abs().T).amax(-1, keepdim=True) + 2.0 ** -20
                out[qa:qa + nq, h] = o
                bound[qa:qa + nq, h] = u * o.abs() + (u + 2 * eps) * big + nk * 2.0 ** -25 * vv.abs().max()
        qa, ka = qa + nq, ka + nk
    return out, bound


def _inputs(q_lens, k_lens, hq, hkv, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tq, tk = sum(q_lens), sum(k_lens)
    q = torch.randn(tq, hq, 128, generator=g, device="cuda").to(dtype)
    k = (torch.randn(tk, hkv, 128, generator=g, device="cuda") * torch.rand(128, generator=g, device="cuda") * 4).to(dtype)
    return q, k, torch.randn(tk, hkv, 128, generator=g, device="cuda").to(dtype)


def _check(out, q, k, v, q_lens, k_lens, scale):
    want, bound = _expect(q, k, v, q_lens, k_lens, scale)
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= bound).all(), float((err / bound.clamp_min(1e-30)).max())


LENGTHS = [
    ([1], [1]), ([2], None), ([37], None), ([127], None), ([128], None), ([129], None), ([1000], None),
    ([2049], None), ([1, 300, 0, 77, 128, 1, 5], None), ([64, 64, 64], None),
    ([1], [4097]), ([1, 1, 1], [300, 1, 5000]), ([17, 200], [1000, 333]), ([5], [128]), ([300], [300 + 256]),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(32, 8), (4, 4), (12, 4), (7, 1)])
@pytest.mark.parametrize("q_lens,k_lens", LENGTHS)
def test_formula(q_lens, k_lens, heads, dtype):
    from turbopolar_b200 import PromptPlan, prompt_attention
    k_lens = k_lens or q_lens
    q, k, v = _inputs(q_lens, k_lens, *heads, dtype, seed=len(q_lens) + sum(k_lens))
    plan = PromptPlan(q_lens, k_lens, num_q_heads=heads[0], num_kv_heads=heads[1])
    out = prompt_attention(q, k, v, plan)
    assert plan.read_device_error() == 0
    _check(out, q, k, v, q_lens, k_lens, 128 ** -0.5)
    assert torch.equal(out, prompt_attention(q, k, v, plan))


@pytest.mark.parametrize("heads", [(16, 2), (10, 2), (128, 1), (2, 1), (33, 3)])
def test_head_groups(heads):
    from turbopolar_b200 import PromptPlan, prompt_attention
    q_lens, k_lens = [50, 3, 131], [50, 400, 200]
    q, k, v = _inputs(q_lens, k_lens, *heads, torch.float16)
    plan = PromptPlan(q_lens, k_lens, num_q_heads=heads[0], num_kv_heads=heads[1])
    out = prompt_attention(q, k, v, plan, scale=0.2)
    _check(out, q, k, v, q_lens, k_lens, 0.2)


def test_rows_that_see_nothing_give_zero():
    from turbopolar_b200 import PromptPlan, prompt_attention
    q_lens, k_lens = [300, 4, 9, 0], [20, 0, 9, 50]
    q, k, v = _inputs(q_lens, k_lens, 8, 4, torch.float16)
    out = prompt_attention(q, k, v, PromptPlan(q_lens, k_lens, num_q_heads=8, num_kv_heads=4))
    _check(out, q, k, v, q_lens, k_lens, 128 ** -0.5)
    assert (out[:280] == 0).all() and (out[300:304] == 0).all()
    none = prompt_attention(q[:4], k[:0], v[:0], PromptPlan([4], [0], num_q_heads=8, num_kv_heads=4))
    assert (none == 0).all()
    empty = prompt_attention(q[:0], k[:5], v[:5], PromptPlan([0], [5], num_q_heads=8, num_kv_heads=4))
    assert empty.shape == (0, 8, 128)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_keys_have_no_influence(bad, dtype):
    # Non-finite keys and values: of other sequences, and of later tokens of the same tile.
    from turbopolar_b200 import PromptPlan, prompt_attention
    q_lens, k_lens = [70, 333, 40, 1], [70, 333, 300, 150]
    q, k, v = _inputs(q_lens, k_lens, 8, 4, dtype)
    plan = PromptPlan(q_lens, k_lens, num_q_heads=8, num_kv_heads=4)
    clean = prompt_attention(q, k, v, plan)
    kb, vb = k.clone(), v.clone()
    kb[70:403], vb[70:403] = bad, bad   # the whole second sequence
    out = prompt_attention(q, kb, vb, plan)
    assert torch.equal(out[:70], clean[:70]) and torch.equal(out[403:], clean[403:])
    # Values of single later tokens: rows before them are as without, rows from them on see them.
    kb, vb = k.clone(), v.clone()
    at = [(0, 69), (70, 200), (70, 290), (403, 280)]   # (first key, token)
    for first, j in at:
        vb[first + j, :, 5] = bad
    out = prompt_attention(q, kb, vb, plan)
    assert plan.read_device_error() == 0
    qa = ka = 0
    for nq, nk in zip(q_lens, k_lens):
        first_bad = min([j for first, j in at if first == ka] + [nk])
        rows = max(0, first_bad - (nk - nq))   # rows that see no bad key
        assert torch.equal(out[qa:qa + rows], clean[qa:qa + rows])
        later = out[qa + rows:qa + nq]
        if rows < nq:
            assert not torch.isfinite(later[:, :, 5]).any()
            rest = [c for c in range(128) if c != 5]
            err = (later[:, :, rest].double() - clean[qa + rows:qa + nq][:, :, rest].double()).abs()
            assert (err <= 4 * U[dtype] * 6).all()   # values are below 6; weights rounded or not
            if bad == bad and (first_bad, nk) != (200, 333):
                assert (later[:, :, 5] == bad).all()
        qa, ka = qa + nq, ka + nk
    # A key that only masked rows would meet.
    kb = k.clone()
    kb[69, :, 7] = bad
    out = prompt_attention(q, kb, v, plan)
    assert torch.equal(out[:69], clean[:69]) and torch.equal(out[70:], clean[70:])


def test_strided_inputs_and_given_output():
    from turbopolar_b200 import PromptPlan, prompt_attention
    q_lens = [200, 65]
    q, k, v = _inputs(q_lens, q_lens, 8, 2, torch.bfloat16)
    plan = PromptPlan(q_lens, num_q_heads=8, num_kv_heads=2)
    want = prompt_attention(q, k, v, plan)
    fused = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    parts = [t.unflatten(1, (-1, 128)) for t in fused.split([1024, 256, 256], 1)]
    out = torch.empty_like(q)
    assert prompt_attention(*parts, plan, out=out) is out and torch.equal(out, want)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(prompt_attention(*heads_first, plan), want)
    odd = torch.zeros(265, 8 * 128 + 3, dtype=torch.bfloat16, device="cuda")
    odd[:, 1:1025] = q.flatten(1)
    assert torch.equal(prompt_attention(odd[:, 1:1025].unflatten(1, (8, 128)), k, v, plan), want)
    one = k[:, :1].expand(265, 2, 128)   # a broadcast head
    same = prompt_attention(q, one, one, plan)
    assert torch.equal(same, prompt_attention(q, one.contiguous(), one.contiguous(), plan))


def test_large_scores_and_moving_maxima():
    # Scores of hundreds, growing along the keys: the running reference moves in every tile.
    from turbopolar_b200 import PromptPlan, prompt_attention
    n = 1500
    q, k, v = _inputs([n], [n], 4, 2, torch.float16)
    k = (k * torch.linspace(0.1, 6, n, device="cuda")[:, None, None]).half()
    out = prompt_attention(q, k, v, PromptPlan([n], num_q_heads=4, num_kv_heads=2), scale=1.0)
    _check(out, q, k, v, [n], [n], 1.0)


def test_other_streams_and_graphs():
    from turbopolar_b200 import PromptPlan, prompt_attention
    q, k, v = _inputs([1, 130], [3000, 130], 8, 2, torch.float16)
    plan = PromptPlan([1, 130], [3000, 130], num_q_heads=8, num_kv_heads=2)
    want = prompt_attention(q, k, v, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = prompt_attention(q, k, v, plan)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prompt_attention(q, k, v, plan, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert plan.read_device_error() == 0


def test_refusals():
    from turbopolar_b200 import PromptPlan, prompt_attention
    q, k, v = _inputs([20], [20], 8, 4, torch.float16)
    plan = PromptPlan([20], num_q_heads=8, num_kv_heads=4)
    for bad in (dict(q=q[:19]), dict(k=k[:, :2]), dict(v=v.bfloat16()), dict(q=q.float(), k=k.float(), v=v.float()),
                dict(q=q[0]), dict(k=k.cpu()), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(out=torch.empty(20, 8, 128, device="cuda")), dict(out=q), dict(out=q.new_empty(20, 8, 256)[..., :128])):
        with pytest.raises(ValueError):
            prompt_attention(**{**dict(q=q, k=k, v=v, plan=plan), **bad})
    with pytest.raises(NotImplementedError):
        prompt_attention(q[..., :64], k[..., :64], v[..., :64], plan)
    with pytest.raises(NotImplementedError, match="backward"):
        prompt_attention(q.clone().requires_grad_(), k, v, plan)
    for bad in (dict(q_lens=[-1]), dict(q_lens=[1], k_lens=[1, 2]), dict(q_lens=[1], num_q_heads=7),
                dict(q_lens=[1], device="cpu")):
        with pytest.raises(ValueError):
            PromptPlan(**{**dict(num_q_heads=8, num_kv_heads=4), **bad})
