"""tree_attention of float32 inputs that float16 cannot hold: large, small, and of mixed sizes.

Tolerance per element, u = 2^-11, W = sum_j w_j |v_j| over values that float16 can hold, B the same over all values,
S = scale max_j sum_d |q_d k_jd|: u |out| (output), u W (weights of the product; values beyond float16 are multiplied in
float32), (2 eps + 2^-20) B with eps = 2^-17 S + 2^-20 (scores: queries and keys in two float16 parts of 22 bits, the
product of the small parts left out, accumulation, the exponential), 2^-21 W (values in two parts, each to 22 bits) and
2^-25 (values' smallest step) and 2^-32 max|v| for each of the n keys (smallest weights)."""

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


def _runtime(batch, hq, hkv, cached, seed, **change):
    from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda h, n: torch.randn(batch, h, n, 128, generator=g, device="cuda")
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=hq, num_kv_heads=hkv))
    k, v = rand(hkv, cached), rand(hkv, cached)
    for f in change.get("tail", ()):
        f(k, v)
    rt.append(k, v)
    return rt, rand


def _mask(n):
    return (torch.rand(n, n, generator=torch.Generator().manual_seed(n)) < 0.5).cuda() | torch.eye(n, dtype=torch.bool, device="cuda")


def _check(out, rt, q, kd, vd, mask, scale):
    k, v = (x.double() for x in rt.decompress(padded_tail=False))
    if rt.tail_len:
        k[:, :, -rt.tail_len:], v[:, :, -rt.tail_len:] = rt.partial_k.double(), rt.partial_v.double()
    g = q.shape[1] // kd.shape[1]
    keys, values = (torch.cat([x, y.double()], 2).repeat_interleave(g, 1) for x, y in ((k, kd), (v, vd)))
    sees = torch.cat([torch.ones(mask.shape[0], k.shape[2], dtype=torch.bool, device="cuda"), mask], 1)
    s = q.double() @ keys.transpose(-1, -2) * scale
    w = torch.softmax(s.masked_fill(~sees, -torch.inf), -1)
    want, every = w @ values, w @ values.abs()
    held = (values.abs() < 65504).all(-1, keepdim=True)
    small = w @ (values.abs() * held)
    size = scale * (q.double().abs() @ keys.abs().transpose(-1, -2)).amax(-1, keepdim=True)
    eps = 2.0 ** -17 * size + 2.0 ** -20
    n = keys.shape[2]
    bound = U * want.abs() + (U + 2.0 ** -21) * small + (2 * eps + 2.0 ** -20) * every + 2.0 ** -25 + n * 2.0 ** -32 * (values * held).abs().max()
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("cached, drafts, heads, batch", [(10, 6, (8, 2), 2), (50, 70, (4, 4), 1), (40, 200, (4, 1), 1)])
@pytest.mark.parametrize("a, b", [(0, 20), (17, 0), (-20, 20), (-24, -24), (40, -20), (100, -24), (30, 30), (-10, -10)])
def test_queries_and_keys_of_any_size(cached, drafts, heads, batch, a, b):
    hq, hkv = heads
    grow = lambda k, v: k.mul_(2.0 ** b)
    rt, rand = _runtime(batch, hq, hkv, cached, 10 * a + b, tail=[grow])   # fewer than a page: the dense tail
    q, k, v = rand(hq, drafts) * 2.0 ** a, rand(hkv, drafts) * 2.0 ** b, rand(hkv, drafts)
    mask, scale = _mask(drafts), 128 ** -0.5 * 2.0 ** -(a + b)
    _check(rt.tree_attention(q, k, v, mask, scale=scale), rt, q, k, v, mask, scale)


@pytest.mark.parametrize("a", [-20, 17, 60])
@pytest.mark.parametrize("cached", [200, 64 * 50 + 33])
def test_queries_of_any_size_over_pages(cached, a):
    rt, rand = _runtime(1, 8, 2, cached, a)
    q, k, v = rand(8, 40) * 2.0 ** a, rand(2, 40), rand(2, 40)
    mask, scale = _mask(40), 128 ** -0.5 * 2.0 ** -a
    _check(rt.tree_attention(q, k, v, mask, scale=scale), rt, q, k, v, mask, scale)


@pytest.mark.parametrize("q_dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("cached, drafts, heads, batch", [(20, 6, (4, 2), 1), (63, 80, (8, 2), 2), (133, 250, (4, 1), 1), (64 * 50 + 40, 70, (8, 2), 1)])
@pytest.mark.parametrize("size", [66000.0, 1e6])
def test_values_beyond_float16(cached, drafts, heads, batch, size, q_dtype):
    hq, hkv = heads

    def some(k, v):
        v[:, :, 64 * (v.shape[2] // 64) + 2, 5] = size        # in the tail: stored pages are float16
        v[:, :, -1, 100:] = -size
        k[:, :, -1] = -0.1                                      # and a weight that is small, not 0
    rt, rand = _runtime(batch, hq, hkv, cached, int(size), tail=[some])
    q, k, v = (0.3 * rand(hq, drafts)).to(q_dtype), rand(hkv, drafts), rand(hkv, drafts)
    for d in {1, 3, drafts // 2, drafts - 1}:
        v[:, :, d, d % 128] = size * (1 if d % 2 else -1)
    mask = torch.ones(drafts, drafts, dtype=torch.bool, device="cuda")
    mask[0, 1:] = False
    if size > 1e5 and cached < 100:
        q *= 0.1 if q_dtype == torch.float32 else 0.125         # flat weights: the outputs stay within float16
        v[:, :, drafts // 2:] = v[:, :, drafts // 2:].clamp(-3e5, 3e5)
        rt.tail_v.clamp_(-3e5, 3e5)
    _check(rt.tree_attention(q, k, v, mask), rt, q, k, v, mask, 128 ** -0.5)


def test_one_key_beyond_float16_beside_ordinary_ones():
    def some(k, v):
        k[:, :, 4, 7] = 1e6                  # where queries have nothing
    rt, rand = _runtime(1, 8, 2, 30, 3, tail=[some])
    q, k, v = rand(8, 40), rand(2, 40), rand(2, 40)
    q[..., 7] = 0
    k[:, :, 9, 7], k[:, :, 33, 7] = -3e38, 1e5
    mask = _mask(40)
    out = rt.tree_attention(q, k, v, mask)
    assert torch.isfinite(out).all()
    k[:, :, [9, 33], 7] = 0                  # the same scores, in sizes that the bound is tight for
    rt.tail_k[:, 4, 7] = 0
    _check(out, rt, q, k, v, mask, 128 ** -0.5)


def test_masked_drafts_beyond_float16_have_no_influence():
    rt, rand = _runtime(1, 8, 4, 20, 8)
    q, k, v = rand(8, 40), rand(4, 40), rand(4, 40)
    mask = torch.ones(40, 40, dtype=torch.bool, device="cuda").tril()
    clean = rt.tree_attention(q, k, v, mask).clone()
    v[:, :, 35], k[:, :, 36] = 1e30, -1e30
    out = rt.tree_attention(q, k, v, mask)
    assert torch.equal(out[:, :, :35], clean[:, :, :35])
