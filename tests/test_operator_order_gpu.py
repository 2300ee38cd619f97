"""Calls that follow an attention of prompts or drafts on one stream see its results.

Decode attention may start before the previous decode attention has completed when it reads nothing
that one writes.  It has to wait for a prompt or tree attention launched in between, whose buffers it does
not compare: here its query is that call's output."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cache(tokens, seed):
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(seed)
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=32, num_kv_heads=8))
    rt.append(torch.randn(1, 8, tokens, 128, generator=g, device="cuda").half(),
              torch.randn(1, 8, tokens, 128, generator=g, device="cuda").half())
    return rt, g


@pytest.mark.parametrize("tokens", [64, 700, 2048])
def test_decode_attention_waits_for_prompt_attention(tokens):
    from turbopolar_b200 import PromptPlan, prompt_attention
    rt, g = _cache(1000, 1)
    q = torch.randn(tokens, 32, 128, generator=g, device="cuda").half()
    k, v = (3 * torch.randn(tokens, 8, 128, generator=g, device="cuda").half() for _ in range(2))
    plan = PromptPlan([tokens], num_q_heads=32, num_kv_heads=8)
    want_q = prompt_attention(q, k, v, plan)[:1].clone()
    want = rt.attention(want_q).clone()
    first = torch.randn(1, 32, 128, generator=g, device="cuda").half()
    for _ in range(20):
        out = torch.full((tokens, 32, 128), 7.0, dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        rt.attention(first)  # lets a later, independent call start early
        prompt_attention(q, k, v, plan, out=out)
        got = rt.attention(out[:1])
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("cached, drafts", [(100, 5), (130, 64), (1000, 16)])
def test_decode_attention_waits_for_tree_attention(cached, drafts):
    rt, g = _cache(cached, 2)
    other, _ = _cache(1000, 3)
    q = torch.randn(1, 32, drafts, 128, generator=g, device="cuda").half()
    k, v = (torch.randn(1, 8, drafts, 128, generator=g, device="cuda").half() for _ in range(2))
    mask = torch.ones(drafts, drafts, dtype=torch.bool, device="cuda").tril()
    want_q = rt.tree_attention(q, k, v, mask)[:, :, 0].clone()
    want = other.attention(want_q).clone()
    first = torch.randn(1, 32, 128, generator=g, device="cuda").half()
    out = torch.empty(1, drafts, 32, 128, dtype=torch.float16, device="cuda")
    for _ in range(20):
        out.fill_(7.0)
        torch.cuda.synchronize()
        other.attention(first)
        rt.tree_attention(q, k, v, mask, out=out)
        got = other.attention(out[:, 0])
        torch.cuda.synchronize()
        assert torch.equal(got, want)
