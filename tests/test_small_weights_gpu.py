"""Weights far below a row's largest: 2^-20 to 2^-30 of it each, all of the output together.

Tolerance per element, u = 2^-11 (2^-8 for bfloat16), W = sum_j w_j |v_j| with the exact weights: u |out| (output),
u W (weights), 2 eps W with eps = 2^-18 S + 2^-20, S = scale max_j sum_d |q_d k_jd| (scores, exponential), and
2^-32 max|v| for each of the n keys (float16 weights are multiples of 2^-24 or so with the largest at 2^7 or more)."""

import pytest
import torch

pytestmark = pytest.mark.gpu
LN2 = 0.6931471805599453


def _rows(n, strong, g):
    """Scores' exponents of n keys, 0 at `strong`."""
    x = -20 - 10 * torch.rand(n, generator=g, device="cuda")
    x[strong] = 0
    return x


def _near(out, s, sees, v, u, size):
    w = torch.softmax(s.masked_fill(~sees, -torch.inf), -1)
    want, big = w @ v, w @ v.abs()
    bound = u * want.abs() + (u + 2 * (2.0 ** -18 * size + 2.0 ** -20)) * big + sees.sum(-1, keepdim=True) * 2.0 ** -32 * v.abs().max()
    err = (out.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("strong", [0, 1, 700, 5000])
@pytest.mark.parametrize("queries, keys, hq, hkv", [(1, 6000, 8, 2), (100, 6000, 4, 1), (4000, 6000, 8, 8)])
def test_prompt_attention(queries, keys, hq, hkv, strong, dtype):
    from turbopolar_b200 import PromptPlan, prompt_attention
    g = torch.Generator(device="cuda").manual_seed(strong)
    x = _rows(keys, strong, g)
    q, k = torch.zeros(queries, hq, 128, device="cuda"), torch.zeros(keys, hkv, 128, device="cuda")
    q[..., 3], k[..., 3] = 8.0, (x * LN2 / 0.8)[:, None]
    v = 500 + 500 * torch.rand(keys, hkv, 128, generator=g, device="cuda")
    v[strong] = 0
    q, k, v = (y.to(dtype) for y in (q, k, v))
    plan = PromptPlan([queries], [keys], num_q_heads=hq, num_kv_heads=hkv)
    out = prompt_attention(q, k, v, plan, scale=0.1)
    rows = torch.tensor(sorted({0, queries // 2, queries - 1}), device="cuda")
    sees = torch.arange(keys, device="cuda")[None] <= rows[:, None] + keys - queries
    for h in (0, hq - 1):
        kv = h * hkv // hq
        s = 0.1 * (q[rows, h].double() @ k[:, kv].double().t())
        _near(out[rows, h], s, sees, v[:, kv].double(), 2.0 ** (-11 if dtype == torch.float16 else -8), 22.0)


@pytest.mark.parametrize("batch, cached, drafts", [(1, 130, 3), (1, 130, 70), (40, 640, 10), (1, 6000, 40)])
def test_tree_attention(batch, cached, drafts):
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(cached)
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=8, num_kv_heads=4))
    k = torch.zeros(batch, 4, cached, 128, device="cuda")   # the background: stored keys of zero are exact
    k[:, :, 5, 3] = 26 * LN2 / 0.8                           # one strong key, as far above as its code decodes
    v = 500 + 500 * torch.rand(batch, 4, cached, 128, generator=g, device="cuda")
    v[:, :, 5] = 0
    rt.append(k.half(), v.half())
    q, kd, vd = (torch.zeros(batch, h, drafts, 128, device="cuda").half() for h in (8, 4, 4))
    q[..., 3] = 8.0
    mask = torch.eye(drafts, dtype=torch.bool, device="cuda")
    out = rt.tree_attention(q, kd, vd, mask, scale=0.1)
    stored_k, stored_v = rt.decompress(padded_tail=False)
    keys, values = (torch.cat(x, 2).double() for x in ((stored_k, kd), (stored_v, vd)))
    sees = torch.cat([torch.ones(drafts, cached, dtype=torch.bool, device="cuda"), mask], 1)
    for b, h in ((0, 0), (batch - 1, 7)):
        s = 0.1 * (q[b, h].double() @ keys[b, h // 2].t())
        assert s[0].max() > 24 * LN2
        _near(out[b, h], s, sees, values[b, h // 2], 2.0 ** -11, 22.0)
