"""A mask byte other than 0 means seen, as it does to torch: masks made by viewing bytes as bool hold any value."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [0, 1, 4])   # aligned words of four, and single bytes
@pytest.mark.parametrize("t", [1, 6, 64, 67, 256])
def test_any_byte(t, offset):
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(t)
    rand = lambda h, n: torch.randn(1, h, n, 128, generator=g, device="cuda").half()
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=4, num_kv_heads=2))
    rt.append(rand(2, 3), rand(2, 3))
    q, k, v = rand(4, t), rand(2, t), rand(2, t)
    values = torch.tensor([0, 0, 1, 2, 64, 127, 128, 254, 255], dtype=torch.uint8, device="cuda")
    wide = values[torch.randint(0, 9, (t, 264), generator=g, device="cuda")].view(torch.bool)
    mask = wide[:, offset:offset + t]
    seen = mask.view(torch.uint8) != 0
    assert torch.equal(rt.tree_attention(q, k, v, mask), rt.tree_attention(q, k, v, seen))
