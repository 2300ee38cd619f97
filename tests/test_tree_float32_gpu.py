"""tree_attention of float32 queries, tails and drafts: nothing of the inputs is rounded to float16 but the output and
the weights.

Tolerance per element, u = 2^-11, W = sum_j w_j |v_j| with the exact weights, S = scale max_j sum_d |q_d k_jd|:
u |out| (output), u W (weights), 2 eps W with eps = 2^-17 S + 2^-20 (scores: queries and keys in two float16 parts,
22 bits each, the product of the two small parts left out, accumulation, the exponential), 2^-21 W (values in two
parts) and n 2^-25 max|v| (weights below the normal range of float16)."""

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


@pytest.mark.parametrize("cached, drafts, heads, batch", [(6, 24, (8, 2), 4), (10, 1, (32, 8), 1), (1, 33, (4, 4), 1), (63, 64, (32, 8), 1),
                                                          (33, 97, (7, 1), 2), (32, 256, (4, 2), 1)])
def test_float32_inputs_are_not_rounded(cached, drafts, heads, batch):
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    hq, hkv = heads
    g = torch.Generator(device="cuda").manual_seed(cached + drafts)
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=hq, num_kv_heads=hkv))
    def normal(h, n, size=1.0):
        return size * torch.randn(batch, h, n, 128, generator=g, device="cuda")
    tail_k, tail_v = normal(hkv, cached, 2.0), normal(hkv, cached)
    rt.append(tail_k, tail_v)   # fewer than a page: the dense tail
    q, k, v = normal(hq, drafts), normal(hkv, drafts, 2.0), normal(hkv, drafts)
    mask = (torch.rand(drafts, drafts, generator=g, device="cuda") < 0.5) | torch.eye(drafts, dtype=torch.bool, device="cuda")
    out = rt.tree_attention(q, k, v, mask).double()
    keys = torch.cat([tail_k, k], 2).double().repeat_interleave(hq // hkv, 1)
    values = torch.cat([tail_v, v], 2).double().repeat_interleave(hq // hkv, 1)
    sees = torch.cat([torch.ones(drafts, cached, dtype=torch.bool, device="cuda"), mask], 1)
    scale = 128 ** -0.5
    w = torch.softmax((q.double() @ keys.transpose(-1, -2) * scale).masked_fill(~sees, -torch.inf), -1)
    want, big = w @ values, w @ values.abs()
    size = scale * (q.double().abs() @ keys.abs().transpose(-1, -2)).amax(-1, keepdim=True)
    eps = 2.0 ** -17 * size + 2.0 ** -20
    bound = U * want.abs() + (U + 2 * eps + 2.0 ** -21) * big + keys.shape[2] * 2.0 ** -25 * values.abs().max()
    err = (out - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    # Far closer than rounded inputs would be.
    assert err.norm() / want.norm() < 3.2e-4


def test_float32_values_that_float16_cannot_hold_stay_with_the_rows_that_see_them():
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(1)
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=8, num_kv_heads=4))
    rt.append(torch.randn(1, 4, 5, 128, generator=g, device="cuda"), torch.randn(1, 4, 5, 128, generator=g, device="cuda"))
    q = torch.randn(1, 8, 40, 128, generator=g, device="cuda")
    k, v = (torch.randn(1, 4, 40, 128, generator=g, device="cuda") for _ in range(2))
    mask = torch.ones(40, 40, dtype=torch.bool, device="cuda").tril()
    clean = rt.tree_attention(q, k, v, mask).clone()
    v[:, :, 35, 3] = float("inf")
    out = rt.tree_attention(q, k, v, mask)
    assert torch.equal(out[:, :, :35], clean[:, :, :35])
    assert not torch.isfinite(out[:, :, 35:, 3]).any()
