"""Outputs that share memory with the smaller inputs or with the cache are refused."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["cos", "sin", "positions", "q_weight", "k_weight"])
@pytest.mark.parametrize("side", ["q", "k"])
def test_norm_rope(what, side):
    from turbopolar_b200 import norm_rope
    dev = "cuda"
    buf = torch.zeros(1 << 16, device=dev)
    q, k = torch.randn(4, 8, 128, device=dev), torch.randn(4, 4, 128, device=dev)
    heads = 8 if side == "q" else 4
    args = dict(cos=torch.ones(4, 64, device=dev), sin=torch.zeros(4, 64, device=dev),
                positions=torch.arange(4, device=dev), q_weight=torch.ones(128, device=dev), k_weight=torch.ones(128, device=dev))
    shared = buf[128:128 + args[what].numel() * (2 if what == "positions" else 1)]
    view = (shared.view(torch.int64) if what == "positions" else shared).view(args[what].shape)
    view.copy_(args[what])
    out = buf[:4 * heads * 128].view(4, heads, 128)
    with pytest.raises(ValueError, match="overlaps"):
        norm_rope(q, k, **{**args, what: view}, **{f"{side}_out": out})
    apart = buf[1 << 15:][:4 * heads * 128].view(4, heads, 128)
    norm_rope(q, k, **{**args, what: view}, **{f"{side}_out": apart})


@pytest.mark.parametrize("what", ["mask", "tail", "pages"])
def test_tree_attention(what):
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda h, n: torch.randn(1, h, n, 128, generator=g, device="cuda").half()
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=2, num_kv_heads=2))
    rt.append(rand(2, 70), rand(2, 70))
    mask = torch.ones(4, 4, dtype=torch.bool, device="cuda").tril()
    if what == "mask":
        buf = torch.zeros(1 << 12, dtype=torch.float16, device="cuda")
        shared = buf[:8].view(torch.uint8).view(torch.bool).view(4, 4)
        shared.copy_(mask)
        mask, out = shared, buf[:1024].view(1, 4, 2, 128)
    elif what == "tail":
        out = rt.tail_k.view(-1)[:1024].view(1, 4, 2, 128)
    else:
        out = rt.pool.pages.view(-1).view(torch.float16)[:1024].view(1, 4, 2, 128)
    with pytest.raises(ValueError, match="shares memory"):
        rt.tree_attention(rand(2, 4), rand(2, 4), rand(2, 4), mask, out=out)
