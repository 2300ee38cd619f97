"""tree_attention and one-token steps on the key format of the Llama adapter, whose steps keep their softmax weights in
two float16 parts where the tree keeps one.

Both round their output to float16 (relative errors spread evenly over +-2^-11 / 2 at the least, 2^-11 at the most: 0.0002 of
the norm) and the tree its weights as well: 0.0003 of the norm each at most, 0.0005 between the two allowed; per element
2 u |out| + (u + 2^-9 S) W, u = 2^-11, W = sum_j w_j |v_j|, S as in the formula's own test (int8 radii round to
either neighbour in each)."""

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


@pytest.mark.parametrize("cached", [100, 1000, 4096])
def test_a_tree_agrees_with_steps(cached):
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    t = 24
    g = torch.Generator(device="cuda").manual_seed(cached)
    rand = lambda h, n: torch.randn(1, h, n, 128, generator=g, device="cuda").half()
    config = TurboPolarConfig(num_q_heads=32, num_kv_heads=8, use_int8_radii=True, k_angle_bits_deep=8, split_dim=0)
    rt = TurboPolarKVCacheRuntime(config, max_seq_len=cached + 64)
    rt.append(rand(8, cached), rand(8, cached))
    q, k, v = rand(32, t), rand(8, t), rand(8, t)
    chain = torch.ones(t, t, dtype=torch.bool, device="cuda").tril()
    tree = rt.tree_attention(q, k, v, chain).double()
    stored_k, stored_v = (x.double() for x in rt.decompress(padded_tail=False))
    steps = []
    for i in range(t):
        if rt.tail_len == 63:   # the next step would store a page, whose keys are no longer the drafts'
            break
        steps.append(rt.decode_step(k[:, :, i:i + 1], v[:, :, i:i + 1], q[:, :, i]).double())
    steps, tree = torch.stack(steps, 2), tree[:, :, :len(steps)]
    n = steps.shape[2]
    assert n > 10
    keys, values = (torch.cat([x, y[:, :, :n].double()], 2).repeat_interleave(4, 1) for x, y in ((stored_k, k), (stored_v, v)))
    scale = 128 ** -0.5
    sees = torch.cat([torch.ones(n, cached, dtype=torch.bool, device="cuda"), chain[:n, :n]], 1)
    w = torch.softmax((q[:, :, :n].double() @ keys.transpose(-1, -2) * scale).masked_fill(~sees, -torch.inf), -1)
    big = w @ values.abs()
    size = scale * (q[:, :, :n].double().abs() @ keys.abs().transpose(-1, -2)).amax(-1, keepdim=True)
    assert ((tree - steps).abs() <= 2 * U * steps.abs() + (U + 2.0 ** -9 * size) * big).all()
    assert (tree - steps).norm() / steps.norm() < 5e-4
