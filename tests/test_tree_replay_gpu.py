"""A captured tree_attention answers for the cache that it was captured on, or not at all."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cached, drafts", [(40, 4), (100, 5), (3000, 30), (640, 200)])
def test_a_replay_on_a_changed_cache_gives_nan(cached, drafts):
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(cached)
    rand = lambda h, n: torch.randn(2, h, n, 128, generator=g, device="cuda").half()
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=8, num_kv_heads=4), max_seq_len=4096)
    rt.append(rand(4, cached), rand(4, cached))
    q, k, v = rand(8, drafts), rand(4, drafts), rand(4, drafts)
    mask = torch.ones(drafts, drafts, dtype=torch.bool, device="cuda").tril()
    want = rt.tree_attention(q, k, v, mask).clone()
    out = torch.empty(2, drafts, 8, 128, dtype=torch.float16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.tree_attention(q, k, v, mask, out=out)

    def replayed():
        out.zero_()
        graph.replay()
        return out.transpose(1, 2).clone()

    assert torch.equal(replayed(), want) and rt.read_device_error() == 0
    rt.append(rand(4, 1), rand(4, 1))
    assert replayed().isnan().all()
    assert rt.read_device_error() == 4
    new = rt.tree_attention(q, k, v, mask)          # eager calls are not affected
    assert torch.isfinite(new).all() and not torch.equal(new, want)
    rt.reset()
    assert replayed().isnan().all()
    rt.append(rand(4, cached), rand(4, cached))     # of the old size, in new buffers
    assert replayed().isnan().all()
    assert torch.isfinite(rt.tree_attention(q, k, v, mask)).all() and rt.read_device_error() == 0


def test_appending_and_verifying_in_one_graph():
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda h, n: torch.randn(1, h, n, 128, generator=g, device="cuda").half()
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=8, num_kv_heads=4), max_seq_len=1024, check_finite=False)
    rt.append(rand(4, 300), rand(4, 300))
    q, k, v, kn, vn = rand(8, 6), rand(4, 6), rand(4, 6), rand(4, 1), rand(4, 1)
    mask = torch.ones(6, 6, dtype=torch.bool, device="cuda").tril()
    out = torch.empty(1, 6, 8, 128, dtype=torch.float16, device="cuda")
    rt.tree_attention(q, k, v, mask)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.append(kn, vn)
        rt.tree_attention(q, k, v, mask, out=out)
    graph.replay()   # the append that the host has counted
    assert torch.equal(out.transpose(1, 2), rt.tree_attention(q, k, v, mask))
    graph.replay()   # one more
    assert out.isnan().all()
