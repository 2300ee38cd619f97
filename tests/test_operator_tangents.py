"""Inputs that carry a tangent of forward-mode differentiation are refused: the kernels would drop it."""

import pytest
import torch
from torch.autograd import forward_ad


def test_the_check_itself():
    from turbopolar_b200._checks import refuse_gradients
    t = torch.zeros(3)
    refuse_gradients(t, None)
    with forward_ad.dual_level():
        refuse_gradients(t, None)
        dual = forward_ad.make_dual(t, torch.ones(3))
        for x in (dual, dual * 2):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                refuse_gradients(t, x)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            refuse_gradients(dual)
        refuse_gradients(forward_ad.unpack_dual(dual).primal)
    refuse_gradients(dual)   # the level has ended, and the tangent with it


@pytest.mark.gpu
def test_operators():
    from turbopolar_b200 import PromptPlan, TurboPolarConfig, TurboPolarKVCacheRuntime, norm_rope, prompt_attention
    rand = lambda *shape: torch.randn(*shape, device="cuda").half()
    q, k, v = rand(4, 8, 128), rand(4, 4, 128), rand(4, 4, 128)
    cos, sin = torch.ones(4, 64, device="cuda"), torch.zeros(4, 64, device="cuda")
    plan = PromptPlan([4], num_q_heads=8, num_kv_heads=4)
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=8, num_kv_heads=4))
    rt.append(rand(1, 4, 9, 128), rand(1, 4, 9, 128))
    mask = torch.ones(4, 4, dtype=torch.bool, device="cuda").tril()
    heads_first = lambda x: x.transpose(0, 1)[None]
    with forward_ad.dual_level(), torch.no_grad():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: norm_rope(dual(q), k, cos, sin), lambda: norm_rope(q, k, dual(cos), sin),
                     lambda: norm_rope(q, k, cos, sin, q_weight=dual(torch.ones(128, device="cuda"))),
                     lambda: prompt_attention(q, dual(k), v, plan),
                     lambda: rt.tree_attention(heads_first(q), heads_first(k), heads_first(dual(v)), mask)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        norm_rope(q, k, cos, sin)
        prompt_attention(q, k, v, plan)
        rt.tree_attention(heads_first(q), heads_first(k), heads_first(v), mask)
