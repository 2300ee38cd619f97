"""tree_attention against its formula in float64 on the decoded cache.

Tolerance per element, u = 2^-11, W = sum_j w_j |v_j| with the exact weights:
  u |out|       the output's rounding to float16
  u W           each weight's rounding to float16
  2 eps W       eps = 2^-18 S + 2^-20 + delta, S = scale max_j sum_d |q_d k_jd|: scores (eight accumulations of 16
                products) and the exponential, once in the numerator and once in the sum; delta = 2^-11 S
                where the kernel's radius 2^(code * s) may round to the other neighbour of the float16 key
                than tp_decode_pages' (int8 radii), and 3 * 2^-11 S where float32 inputs are rounded to float16
                (the query, and the tail's and drafts' keys)
  u W           float32 values rounded to float16 (float32 inputs)
  n 2^-25 max|v|  weights below the normal range of float16
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -11

FORMATS = {
    "default": {},
    "adapter": dict(use_int8_radii=True, k_angle_bits_deep=8, split_dim=0),
    "mixed": dict(k_angle_bits_level1=8, k_angle_bits_deep=2, split_dim=32),
    "odd": dict(k_angle_bits_level1=4, k_angle_bits_deep=2, split_dim=6, use_int8_radii=True),
    "wide": dict(k_angle_bits_level1=8, k_angle_bits_deep=8, split_dim=128),
}


def _runtime(fmt, hq, hkv, batch, cached, dtype=torch.float16, seed=0, **kw):
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(seed + cached)
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=hq, num_kv_heads=hkv, **FORMATS[fmt]), **kw)
    k = torch.randn(batch, hkv, cached, 128, generator=g, device="cuda") * (0.5 + 3.5 * torch.rand(128, generator=g, device="cuda"))
    v = torch.randn(batch, hkv, cached, 128, generator=g, device="cuda")
    rt.append(k.to(dtype), v.to(dtype))
    return rt, g


def _drafts(g, batch, hq, hkv, t, dtype=torch.float16):
    q = torch.randn(batch, hq, t, 128, generator=g, device="cuda").to(dtype)
    k = (2 * torch.randn(batch, hkv, t, 128, generator=g, device="cuda")).to(dtype)
    return q, k, torch.randn(batch, hkv, t, 128, generator=g, device="cuda").to(dtype)


def _tree_mask(t, seed=0):
    g = torch.Generator().manual_seed(seed)
    mask = torch.zeros(t, t, dtype=torch.bool)
    for i in range(t):
        p = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
        if p >= 0:
            mask[i] = mask[p]
        mask[i, i] = True
    return mask.cuda()


def _check(out, rt, q, kd, vd, mask, scale=128 ** -0.5):
    k, v = rt.decompress(padded_tail=False)
    f32 = q.dtype == torch.float32 or kd.dtype == torch.float32 or rt.tail_k.dtype == torch.float32
    if rt.tail_len:   # the tail itself, not its float16 copy
        k, v = k.double(), v.double()
        k[:, :, -rt.tail_len:] = rt.partial_k.double()
        v[:, :, -rt.tail_len:] = rt.partial_v.double()
    b, hq, t, _ = q.shape
    g = hq // k.shape[1]
    kk = torch.cat([k.double(), kd.double()], 2).repeat_interleave(g, 1)
    vv = torch.cat([v.double(), vd.double()], 2).repeat_interleave(g, 1)
    n = k.shape[2]
    m = mask if mask.dim() == 3 else mask[None]
    sees = torch.cat([torch.ones(m.shape[0], t, n, dtype=torch.bool, device="cuda"), m], 2)[:, None]
    s = (q.double() @ kk.transpose(-1, -2) * scale).masked_fill(~sees, -torch.inf)
    w = torch.softmax(s, -1)
    want = w @ vv
    big = w @ vv.abs()
    size = scale * (q.double().abs() @ kk.abs().transpose(-1, -2)).amax(-1, keepdim=True)
    eps = 2.0 ** -18 * size + 2.0 ** -20
    if rt.fmt["int8_radii"]:
        eps = eps + U * size
    if f32:
        eps = eps + 3 * U * size
    bound = U * want.abs() + (U * (2 if f32 else 1) + 2 * eps) * big + (n + t) * 2.0 ** -25 * vv.abs().max()
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all() and out.dtype == torch.float16 and out.shape == q.shape
    assert (err <= bound).all(), float((err / bound).max())
    assert int(rt._tree_workspace[:4].view(torch.int32)) == 0


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("cached", [1, 63, 64, 100, 128, 1000, 4096 + 17])
@pytest.mark.parametrize("hq,hkv,t", [(8, 4, 5), (32, 8, 1), (32, 8, 64), (4, 4, 17)])
def test_formula(fmt, cached, hq, hkv, t):
    rt, g = _runtime(fmt, hq, hkv, 1, cached)
    q, kd, vd = _drafts(g, 1, hq, hkv, t)
    mask = _tree_mask(t)
    out = rt.tree_attention(q, kd, vd, mask)
    _check(out, rt, q, kd, vd, mask)
    assert torch.equal(out, rt.tree_attention(q, kd, vd, mask))
    assert rt.actual_seq_len == cached


@pytest.mark.parametrize("hq,hkv,t", [(4, 2, 64), (4, 2, 65), (4, 1, 33), (8, 1, 100), (7, 1, 256), (6, 2, 129), (16, 1, 48)])
def test_row_tiles_and_draft_tiles(hq, hkv, t):
    rt, g = _runtime("default", hq, hkv, 1, 700)
    q, kd, vd = _drafts(g, 1, hq, hkv, t)
    mask = _tree_mask(t, seed=t)
    _check(rt.tree_attention(q, kd, vd, mask, scale=0.05), rt, q, kd, vd, mask, 0.05)


@pytest.mark.parametrize("batch,hq,hkv,cached,t", [(3, 8, 2, 300, 9), (40, 4, 4, 70, 3), (20, 32, 8, 130, 40), (200, 2, 1, 65, 2)])
def test_batches_and_masks_per_sequence(batch, hq, hkv, cached, t):
    rt, g = _runtime("adapter", hq, hkv, batch, cached)
    q, kd, vd = _drafts(g, batch, hq, hkv, t)
    mask = torch.stack([_tree_mask(t, seed=i) for i in range(batch)])
    _check(rt.tree_attention(q, kd, vd, mask), rt, q, kd, vd, mask)
    _check(rt.tree_attention(q, kd, vd, mask[1]), rt, q, kd, vd, mask[1])


@pytest.mark.parametrize("cached", [40, 64, 333])
def test_float32(cached):
    rt, g = _runtime("default", 8, 2, 1, cached, torch.float32)
    mask = _tree_mask(12)
    for dts in ((torch.float32, torch.float32), (torch.float16, torch.float32), (torch.float32, torch.float16)):
        q = _drafts(g, 1, 8, 2, 12, dts[0])[0]
        _, kd, vd = _drafts(g, 1, 8, 2, 12, dts[1])
        _check(rt.tree_attention(q, kd, vd, mask), rt, q, kd, vd, mask)


def test_long_context_and_single_drafts_agree_with_decode_steps():
    rt, g = _runtime("default", 32, 8, 1, 32768 + 5)
    q, kd, vd = _drafts(g, 1, 32, 8, 3)
    mask = torch.eye(3, dtype=torch.bool, device="cuda")   # three alternatives for the next token
    out = rt.tree_attention(q, kd, vd, mask)
    _check(out, rt, q, kd, vd, mask)
    import copy
    for t in range(3):
        state = rt.d_state.clone()
        n = rt.tail_len
        step = rt.decode_step(kd[:, :, t:t + 1], vd[:, :, t:t + 1], q[:, :, t])
        assert (step.float() - out[:, :, t].float()).abs().max() < 2e-3
        rt.d_state.copy_(state)   # drop the token again
        rt.tail_len, rt.actual_seq_len = n, rt.actual_seq_len - 1


def test_a_chain_of_drafts_equals_appending_them():
    rt, g = _runtime("default", 8, 4, 1, 150)
    q, kd, vd = _drafts(g, 1, 8, 4, 6)
    chain = torch.ones(6, 6, dtype=torch.bool, device="cuda").tril()
    out = rt.tree_attention(q, kd, vd, chain)
    path = torch.arange(6, device="cuda")
    for t in range(6):
        rt.append(kd[:, :, path[t:t + 1]], vd[:, :, path[t:t + 1]])
        got = rt.attention(q[:, :, t])
        assert (got.float() - out[:, :, t].float()).abs().max() < 2e-3


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_drafts_have_no_influence(bad):
    rt, g = _runtime("default", 8, 4, 1, 200)
    t = 70
    q, kd, vd = _drafts(g, 1, 8, 4, t)
    mask = _tree_mask(t, seed=3)
    clean = rt.tree_attention(q, kd, vd, mask).clone()
    for d in (0, 5, 69):
        k2, v2 = kd.clone(), vd.clone()
        k2[:, :, d] = bad
        hidden = ~mask[:, d]
        out = rt.tree_attention(q, k2, vd, mask)
        assert torch.equal(out[:, :, hidden], clean[:, :, hidden])
        v2[:, :, d, 9] = bad
        out = rt.tree_attention(q, kd, v2, mask)
        assert torch.equal(out[:, :, hidden], clean[:, :, hidden])
        seen = out[:, :, ~hidden]
        assert (seen[..., 9].isnan().all() if bad != bad else (seen[..., 9] == bad).all())
        rest = [c for c in range(128) if c != 9]
        assert (seen[..., rest] - clean[:, :, ~hidden][..., rest]).abs().max() < 4 * U * 6
    # A draft that sees itself only, and one that sees the cache only.
    mask = torch.zeros(t, t, dtype=torch.bool, device="cuda")
    mask[3, 3] = True
    _check(rt.tree_attention(q, kd, vd, mask), rt, q, kd, vd, mask)


def test_stale_tail_and_pool_memory_is_not_read():
    rt, g = _runtime("default", 8, 4, 1, 130, max_seq_len=512)
    q, kd, vd = _drafts(g, 1, 8, 4, 4)
    mask = _tree_mask(4)
    want = rt.tree_attention(q, kd, vd, mask).clone()
    rt.tail_k[:, rt.tail_len:] = float("nan")
    rt.tail_v[:, rt.tail_len:] = float("nan")
    rt.pool.pages[:, rt.n_pages:] = 0xff
    assert torch.equal(rt.tree_attention(q, kd, vd, mask), want)


def test_layouts_streams_and_graphs():
    rt, g = _runtime("adapter", 8, 2, 2, 777, max_seq_len=1024)
    q, kd, vd = _drafts(g, 2, 8, 2, 10)
    mask = _tree_mask(10)
    want = rt.tree_attention(q, kd, vd, mask).clone()
    alt = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, kd, vd)]   # (B, T, H, 128) storage
    assert torch.equal(rt.tree_attention(*alt, mask), want)
    odd = torch.zeros(2, 8, 10, 131, dtype=torch.float16, device="cuda")
    odd[..., 1:129] = q
    assert torch.equal(rt.tree_attention(odd[..., 1:129], kd, vd, mask.t().contiguous().t()), want)
    wide = torch.zeros(10, 33, dtype=torch.bool, device="cuda")
    wide[:, 3:13] = mask
    assert torch.equal(rt.tree_attention(q, kd, vd, wide[:, 3:13]), want)
    buf = torch.empty(2, 10, 8, 128, dtype=torch.float16, device="cuda")
    got = rt.tree_attention(q, kd, vd, mask, out=buf)
    assert got.data_ptr() == buf.data_ptr() and torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rt.tree_attention(q, kd, vd, mask)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.tree_attention(q, kd, vd, mask, out=buf)
    for _ in range(3):
        buf.zero_()
        graph.replay()
        assert torch.equal(buf.transpose(1, 2), want)


def test_mixed_with_decode_steps_on_one_stream():
    # The page pass of a decode step may start early behind a call it does not depend on; a tree
    # call in between reads and precedes what the steps write.
    rt, g = _runtime("default", 32, 8, 1, 2000, max_seq_len=4096, check_finite=False)
    q, kd, vd = _drafts(g, 1, 32, 8, 8)
    mask = _tree_mask(8)
    for i in range(70):
        rt.decode_step(kd[:, :, i % 8:i % 8 + 1], vd[:, :, i % 8:i % 8 + 1], q[:, :, i % 8])
        out = rt.tree_attention(q, kd, vd, mask)
        if i % 23 == 0:
            _check(out, rt, q, kd, vd, mask)
    _check(out, rt, q, kd, vd, mask)


def test_refusals():
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    rt, g = _runtime("default", 8, 4, 1, 100)
    q, kd, vd = _drafts(g, 1, 8, 4, 5)
    mask = _tree_mask(5)
    base = dict(q=q, k_draft=kd, v_draft=vd, mask=mask)
    for bad in (dict(q=q[:, :7]), dict(q=q[0]), dict(q=q[..., :64]), dict(k_draft=kd[:, :, :4]), dict(v_draft=vd.float()),
                dict(q=q.bfloat16()), dict(mask=mask.float()), dict(mask=mask[:4]), dict(mask=mask.cpu()), dict(scale=0.0),
                dict(scale=-0.1), dict(scale=float("nan")), dict(out=torch.empty(1, 8, 5, 128, device="cuda").half()),
                dict(out=torch.empty(1, 5, 8, 128, device="cuda")), dict(q=q[:, :, :0], k_draft=kd[:, :, :0], v_draft=vd[:, :, :0], mask=mask[:0, :0])):
        with pytest.raises(ValueError):
            rt.tree_attention(**{**base, **bad})
    q2, k2, v2 = _drafts(g, 1, 8, 4, 257)
    with pytest.raises(ValueError, match="256"):
        rt.tree_attention(q2, k2, v2, torch.ones(257, 257, dtype=torch.bool, device="cuda"))
    with pytest.raises(NotImplementedError, match="backward"):
        rt.tree_attention(q.clone().requires_grad_(), kd, vd, mask)
    with pytest.raises(RuntimeError, match="no blocks"):
        TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=8, num_kv_heads=4)).tree_attention(q, kd, vd, mask)
    rt.set_global_length(500)
    with pytest.raises(NotImplementedError, match="shard"):
        rt.tree_attention(q, kd, vd, mask)
