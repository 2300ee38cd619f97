"""Scratch of tree_attention: a captured call keeps the address it was captured with, so that memory may not go
back to the allocator while the runtime exists, and calls on two streams have a piece each.

The CPU tests stand in for the launch and look at the addresses that calls pass."""

import weakref

import pytest
import torch


@pytest.fixture
def host_runtime(monkeypatch):
    """A runtime with a tail of 3 tokens on the CPU whose launches record their scratch; ``stream`` sets the stream."""
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime, _checks, build, cache
    build.build()
    stream, calls = [7], []
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: stream[0])
    monkeypatch.setattr(cache, "launch", lambda device, fn, *args: calls.append(args[-2:]) or 0)
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=8, num_kv_heads=4))

    def start():
        rt._batch_size, rt._num_kv_heads, rt._head_dim, rt._input_dtype = 1, 4, 128, torch.float16
        rt.device, rt._initialized, rt.tail_len, rt.actual_seq_len = torch.device("cpu"), True, 3, 3
        rt._allocate_tail()

    start()

    def call(drafts, on=7, heads=8):
        stream[0] = on
        half = lambda h: torch.zeros(1, h, drafts, 128, dtype=torch.float16)
        rt.tree_attention(half(heads), half(4), half(4), torch.ones(drafts, drafts, dtype=torch.bool))
        return calls[-1]

    return rt, start, call


def _held(rt):
    return {t.data_ptr() for t in [*rt._tree_scratch.values(), *rt._tree_replaced]}


def test_a_larger_call_keeps_the_scratch_of_a_captured_one(host_runtime):
    rt, start, call = host_runtime
    first, size = call(4)
    old = weakref.ref(rt._tree_workspace)
    second, larger = call(200)
    assert larger > size and second != first
    assert old() is not None and old().data_ptr() == first   # a graph may still write there
    assert call(4) == (second, larger)                       # later calls use the larger one
    call(200, heads=16)
    rt.reset()
    start()
    call(3)
    assert {first, second} <= _held(rt)


def test_scratch_is_replaced_a_few_times_only(host_runtime):
    rt, _, call = host_runtime
    for drafts in range(1, 257):
        call(drafts)
    assert len(rt._tree_replaced) <= 5
    total = sum(t.numel() for t in [*rt._tree_scratch.values(), *rt._tree_replaced])
    assert total < 3 * rt._tree_workspace.numel()


def test_streams_do_not_share_scratch(host_runtime):
    rt, _, call = host_runtime
    a, b = call(16, on=7)[0], call(16, on=8)[0]
    assert a != b and call(16, on=7)[0] == a and call(5, on=8)[0] == b
    call(256, on=8)
    assert call(16, on=7)[0] == a and {a, b} <= _held(rt)


@pytest.mark.gpu
def test_a_captured_call_is_right_after_a_larger_one():
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda h, n: torch.randn(1, h, n, 128, generator=g, device="cuda").half()
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=8, num_kv_heads=4), max_seq_len=4096)
    rt.append(rand(4, 3000), rand(4, 3000))
    small, large = (rand(8, 4), rand(4, 4), rand(4, 4)), (rand(8, 250), rand(4, 250), rand(4, 250))
    masks = [torch.ones(n, n, dtype=torch.bool, device="cuda").tril() for n in (4, 250)]
    want = rt.tree_attention(*small, masks[0]).clone()
    out = torch.empty(1, 4, 8, 128, dtype=torch.float16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.tree_attention(*small, masks[0], out=out)
        captured = rt._tree_workspace.data_ptr()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):   # the larger call of the same stream
        rt.tree_attention(*large, masks[1])
    want_large = rt.tree_attention(*large, masks[1]).clone()
    assert captured in _held(rt) and captured != rt._tree_workspace.data_ptr()
    others = [torch.full((1 << 18,), 5.0, device="cuda") for _ in range(64)]   # what the allocator hands out now
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out.transpose(1, 2), want)
        assert torch.equal(rt.tree_attention(*large, masks[1]), want_large)
    assert all(bool((x == 5.0).all()) for x in others)


@pytest.mark.gpu
def test_calls_on_two_streams_at_the_same_time():
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda h, n: torch.randn(1, h, n, 128, generator=g, device="cuda").half()
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=8, num_kv_heads=4))
    rt.append(rand(4, 5000), rand(4, 5000))
    sets = [(rand(8, n), rand(4, n), rand(4, n), torch.ones(n, n, dtype=torch.bool, device="cuda").tril()) for n in (9, 130)]
    want = [rt.tree_attention(*x).clone() for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(rt.tree_attention(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
