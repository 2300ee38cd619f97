"""Replays on a changed cache in the key formats whose decoders read more than the pages (int8 radii: a scale per page)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [dict(use_int8_radii=True, k_angle_bits_deep=8, split_dim=0),
                                 dict(k_angle_bits_level1=8, k_angle_bits_deep=2, split_dim=32)])
@pytest.mark.parametrize("cached, drafts, dtype", [(130, 5, torch.float16), (2000, 70, torch.float32)])
def test_nan_and_then_the_new_answer(fmt, cached, drafts, dtype):
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(drafts)
    rand = lambda h, n: torch.randn(1, h, n, 128, generator=g, device="cuda").to(dtype)
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=8, num_kv_heads=4, **fmt), max_seq_len=4096)
    rt.append(rand(4, cached), rand(4, cached))
    q, k, v = rand(8, drafts), rand(4, drafts), rand(4, drafts)
    mask = torch.ones(drafts, drafts, dtype=torch.bool, device="cuda").tril()
    out = torch.empty(1, drafts, 8, 128, dtype=torch.float16, device="cuda")
    want = rt.tree_attention(q, k, v, mask).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.tree_attention(q, k, v, mask, out=out)
    graph.replay()
    assert torch.equal(out.transpose(1, 2), want)
    rt.append(rand(4, 64), rand(4, 64))
    graph.replay()
    assert out.isnan().all() and rt.read_device_error() == 4
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.tree_attention(q, k, v, mask, out=out)
    graph.replay()
    assert torch.equal(out.transpose(1, 2), rt.tree_attention(q, k, v, mask))
