"""norm_rope against its formula in float64.

Tolerance per element: one rounding to the output type (half an ulp, relative 2^-11 float16,
2^-8 bfloat16, 2^-24 float32; half of the smallest subnormal below the normal range) plus the float32
arithmetic: at most 16 roundings of 2^-24 on the two products that make the element (sum of 8 terms per
lane and 4 shuffles, reciprocal square root of two ulps, three products, one sum)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}


def _table(rows, theta=500000.0, dtype=torch.float32):
    ang = np.arange(rows)[:, None] * theta ** (-np.arange(64) / 64)
    return torch.tensor(np.cos(ang), dtype=dtype, device="cuda"), torch.tensor(np.sin(ang), dtype=dtype, device="cuda")


def _expect(x, w, cos, sin, eps, interleaved):
    """(value, size of the two products) in float64; cos, sin (..., 64) of each row's token."""
    x = x.double().cpu().numpy()
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.double().cpu().numpy()
    c, s = (t.double().cpu().numpy()[..., None, :] for t in (cos, sin))
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :64], x[..., 64:])
    parts = (a * c - b * s, b * c + a * s)
    sizes = (np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s))
    join = (lambda p: np.stack(p, -1).reshape(x.shape)) if interleaved else (lambda p: np.concatenate(p, -1))
    return join(parts), join(sizes)


def _check(got, x, w, cos, sin, eps, interleaved):
    want, size = _expect(x, w, cos, sin, eps, interleaved)
    bound = HALF_ULP[x.dtype] * (np.abs(want) + 16 * 2.0 ** -24 * size) + 16 * 2.0 ** -24 * size + TINY[x.dtype]
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weights", ["none", "both", "q"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hkv", [(1, 32, 8), (3, 5, 1), (130, 8, 4), (1001, 12, 4)])
def test_formula(tokens, hq, hkv, dtype, weights, interleaved):
    from turbopolar_b200 import norm_rope
    g = torch.Generator(device="cuda").manual_seed(tokens)
    fused = (2 * torch.randn(tokens, (hq + 2 * hkv) * 128, generator=g, device="cuda")).to(dtype)
    q = fused[:, :hq * 128].view(tokens, hq, 128)
    k = fused[:, hq * 128:(hq + hkv) * 128].view(tokens, hkv, 128)
    cos, sin = _table(4096)
    pos = torch.randint(0, 4096, (tokens,), generator=g, device="cuda")
    qw = torch.randn(128, generator=g, device="cuda").to(dtype) if weights != "none" else None
    kw = torch.randn(128, generator=g, device="cuda").to(dtype) if weights == "both" else None
    for p in (pos, pos.int()):
        qo, ko = norm_rope(q, k, cos, sin, positions=p, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved)
        assert qo.is_contiguous() and ko.is_contiguous()
        _check(qo, q, qw, cos[pos], sin[pos], 1e-5, interleaved)
        _check(ko, k, kw, cos[pos], sin[pos], 1e-5, interleaved)


@pytest.mark.parametrize("table", [torch.float16, torch.bfloat16])
def test_batched_layouts_and_full_width_tables(table):
    # Rotary embeddings as Hugging Face models pass them: (B, T, 128), both halves alike.
    from turbopolar_b200 import norm_rope
    g = torch.Generator(device="cuda").manual_seed(5)
    B, T, hq, hkv = 3, 17, 8, 2
    ang = torch.rand(B, T, 64, generator=g, device="cuda") * 6
    cos, sin = (torch.cat([f(ang), f(ang)], -1).to(table) for f in (torch.cos, torch.sin))
    q = torch.randn(B, hq, T, 128, generator=g, device="cuda").half().transpose(1, 2)
    k = torch.randn(B, hkv, T, 128, generator=g, device="cuda").half().transpose(1, 2)
    q_out = torch.empty(B, hq, T, 128, dtype=torch.float16, device="cuda").transpose(1, 2)
    half = [t.view(B * T, 128)[:, :64] for t in (cos, sin)]
    qo, ko = norm_rope(q, k, *half, q_out=q_out)
    assert qo is q_out
    _check(qo, q, None, cos[..., :64], sin[..., :64], 0, False)
    _check(ko, k, None, cos[..., :64], sin[..., :64], 0, False)
    # One row per token shared by the batch, and positions per sequence.
    c, s = _table(64)
    qo, ko = norm_rope(q, k, c, s)
    _check(qo, q, None, c[:T], s[:T], 0, False)
    pos = torch.randint(0, 64, (B, T), generator=g, device="cuda")
    qo, ko = norm_rope(q, k, c, s, positions=pos)
    _check(ko, k, None, c[pos], s[pos], 0, False)


def test_in_place_and_unaligned_inputs():
    from turbopolar_b200 import norm_rope
    g = torch.Generator(device="cuda").manual_seed(6)
    T, hq, hkv = 33, 4, 2
    c, s = _table(64)
    w = torch.randn(128, generator=g, device="cuda")
    fused = torch.randn(T, (hq + 2 * hkv) * 128, generator=g, device="cuda").half()
    q, k, v = (t.view(T, -1, 128) for t in fused.split([hq * 128, hkv * 128, hkv * 128], 1))
    want = norm_rope(q, k, c, s, q_weight=w, k_weight=w)
    kept = v.clone()
    got = norm_rope(q, k, c, s, q_weight=w, k_weight=w, q_out=q, k_out=k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, kept)
    # Rows that start off the boundaries, odd strides, and one token with an arbitrary token stride.
    flat = torch.randn(1 + T * (hq * 128 + 3), generator=g, device="cuda").half()
    q = flat[1:].view(T, hq * 128 + 3)[:, :hq * 128].unflatten(1, (hq, 128))
    qo, _ = norm_rope(q, k, c, s)
    _check(qo, q, None, c[:T], s[:T], 0, False)
    one = torch.randn(hq * 128, generator=g, device="cuda").half().as_strided((1, hq, 128), (13, 128, 1))
    qo, _ = norm_rope(one, k[:1], c, s)
    _check(qo, one, None, c[:1], s[:1], 0, False)


def test_other_stream_and_empty_inputs():
    from turbopolar_b200 import norm_rope
    c, s = _table(8)
    q = torch.randn(8, 4, 128, device="cuda")
    want = norm_rope(q, q.clone(), c, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = norm_rope(q, q.clone(), c, s)
    side.synchronize()
    assert torch.equal(got[0], want[0])
    qo, ko = norm_rope(q[:0], q[:0], c, s)
    assert qo.shape == (0, 4, 128) and ko.shape == (0, 4, 128)


def test_extreme_rows():
    from turbopolar_b200 import norm_rope
    c, s = _table(8)
    q = torch.zeros(4, 1, 128, device="cuda", dtype=torch.bfloat16)
    q[1] = 1e18           # the sum of squares stays inside float32
    q[2] = float("inf")
    q[3, 0, 3] = float("nan")
    qo, _ = norm_rope(q, q.clone(), c, s, q_weight=torch.ones(128, device="cuda"), eps=1e-6)
    assert torch.equal(qo[0], torch.zeros_like(qo[0]))
    assert torch.isfinite(qo[1]).all() and qo[2].isnan().all() and qo[3].isnan().all()
    # A position outside the table gives NaN rows and reads nothing.
    pos = torch.tensor([0, -1, 8, 2 ** 40], device="cuda")
    qo, ko = norm_rope(q[:1].expand(4, 1, 128), q[:1].expand(4, 1, 128), c, s, positions=pos)
    assert torch.isfinite(qo[0]).all() and qo[1:].isnan().all() and ko[1:].isnan().all()


def test_refusals():
    from turbopolar_b200 import norm_rope
    c, s = _table(8)
    q = torch.randn(8, 4, 128, device="cuda", dtype=torch.float16)
    k = torch.randn(8, 2, 128, device="cuda", dtype=torch.float16)
    bad = [
        dict(q=q[0]), dict(k=k[:7]), dict(k=k.float()), dict(q=q.double(), k=k.double()), dict(q=q.cpu()),
        dict(cos=c[:7], sin=s[:7]), dict(cos=c[:, :32], sin=s[:, :32]), dict(sin=s.half()), dict(cos=c.cpu()),
        dict(positions=torch.zeros(7, dtype=torch.int32, device="cuda")), dict(positions=torch.zeros(8, device="cuda")),
        dict(q_weight=torch.ones(64, device="cuda")), dict(k_weight=torch.ones(128)),
        dict(q_weight=torch.ones(128, device="cuda"), k_weight=torch.ones(128, device="cuda").half()),
        dict(q_out=torch.empty(8, 4, 128, device="cuda")), dict(q_out=torch.empty(1, 4, 128, device="cuda").half().expand(8, 4, 128)),
        dict(k_out=k.flip(0)[:4]), dict(q_out=q[:, :, :].as_strided((8, 4, 128), (512, 128, 1), 0)[:, [0, 1, 2, 3]][:7]),
    ]
    base = dict(q=q, k=k, cos=c, sin=s)
    for change in bad:
        with pytest.raises(ValueError):
            norm_rope(**{**base, **change})
    buf = torch.empty(9, 4, 128, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError, match="overlaps"):
        norm_rope(buf[:8], k, c, s, q_out=buf[1:])
    with pytest.raises(ValueError, match="overlaps"):
        norm_rope(q, k, c, s, q_out=k.new_empty(8, 4, 128), k_out=q[:, :2])
    with pytest.raises(NotImplementedError):
        norm_rope(q[..., :64], k[..., :64], c, s)
    with pytest.raises(NotImplementedError, match="backward"):
        norm_rope(q.clone().requires_grad_(), k, c, s)
    with torch.no_grad():
        norm_rope(q.clone().requires_grad_(), k, c, s)
