"""What the prompt and draft operators do, in plain torch operations, and the cases they are timed on.

Three operators make one attention layer of a prompt chunk or of a tree of drafted tokens over the
compressed cache:

* ``rope``   -- norms of the query and key heads with the position rotation, in one pass;
* ``prompt`` -- causal attention of packed sequences with grouped heads, also over a history;
* ``tree``   -- attention of drafted tokens over the compressed pages, the dense tail and each other.

``run`` computes them in float32 with elementary operations where ``own`` is false, and calls the
package where it is true.  ``exact`` computes them from their definitions in float64.
"""

import math

import torch

own = False

D = 128
PAGE = 64
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# Key formats: level-1 bits, deep bits, channels coded at level 1, int8 log radii.
FORMATS = {"default": (4, 4, 64, 0), "adapter": (4, 8, 0, 1), "mixed": (8, 2, 32, 0)}


def listed():
    return [
        # One new token in one sequence: every decode step rotates one row per layer (no norm weights).
        {"name": "rope 1 token", "op": "rope", "dtype": "f16", "hq": 32, "hkv": 8, "tokens": 1, "start": 4095,
         "weights": False, "interleaved": False, "table": "f32"},
        # The drafts of one verification step, with norm weights and adjacent pairs, float32 activations.
        {"name": "rope 48 drafts f32", "op": "rope", "dtype": "f32", "hq": 32, "hkv": 8, "tokens": 48, "start": 8000,
         "weights": True, "interleaved": True, "table": "f32"},
        # One 8K prompt, bfloat16, q and k as slices of the fused projection's rows.
        {"name": "rope 8K bf16", "op": "rope", "dtype": "bf16", "hq": 32, "hkv": 8, "tokens": 8192, "start": 0,
         "weights": True, "interleaved": False, "table": "f32"},
        # One short question on a small head layout: launch latency.
        {"name": "prompt 37", "op": "prompt", "dtype": "f16", "hq": 8, "hkv": 4, "q_lens": "37", "past": "0"},
        # A batch of requests of very different lengths, packed.
        {"name": "prompt ragged bf16", "op": "prompt", "dtype": "bf16", "hq": 32, "hkv": 8,
         "q_lens": "1,613,2048,77,1301,5,333,129,2500,1000,64,1", "past": "0,0,0,0,0,0,0,0,0,0,0,0"},
        # Single tokens of four sequences over dense histories, as a decode step of a batch.
        {"name": "prompt 4 tokens on 8K", "op": "prompt", "dtype": "f16", "hq": 32, "hkv": 8, "q_lens": "1,1,1,1",
         "past": "8191,5000,3000,8000"},
        # One 16K prompt.
        {"name": "prompt 16K", "op": "prompt", "dtype": "f16", "hq": 32, "hkv": 8, "q_lens": "16384", "past": "0"},
        # A short conversation on a small head layout, a handful of drafts: launch latency.
        {"name": "tree 100 x 5", "op": "tree", "dtype": "f16", "hq": 8, "hkv": 4, "batch": 1, "fmt": "default",
         "cached": 100, "drafts": 5},
        # An ordinary verification step over a 4K context in the adapter's key format.
        {"name": "tree 4K x 8 adapter", "op": "tree", "dtype": "f16", "hq": 32, "hkv": 8, "batch": 1, "fmt": "adapter",
         "cached": 4096 + 17, "drafts": 8},
        # A wide tree over a 32K context.
        {"name": "tree 32K x 32", "op": "tree", "dtype": "f16", "hq": 32, "hkv": 8, "batch": 1, "fmt": "default",
         "cached": 32768 + 41, "drafts": 32},
        # Eight sequences of 4K verified together.
        {"name": "tree 8 x 4K x 16", "op": "tree", "dtype": "f16", "hq": 32, "hkv": 8, "batch": 8, "fmt": "default",
         "cached": 4096 + 5, "drafts": 16},
        # The longest context with the widest tree.
        {"name": "tree 128K x 64", "op": "tree", "dtype": "f16", "hq": 32, "hkv": 8, "batch": 1, "fmt": "default",
         "cached": 131072, "drafts": 64},
    ]


HEADS = [(32, 8), (32, 8), (8, 4), (8, 2), (4, 4), (16, 2), (12, 4), (14, 2), (8, 8), (5, 1)]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "prompt", "prompt", "tree", "tree"])
    hq, hkv = rng.choice(HEADS)
    if op == "rope":
        tokens = _log_int(rng, 1, 8192)
        return {"op": op, "dtype": rng.choice(["f16", "bf16", "f32"]) if tokens <= 4096 else "bf16", "hq": hq, "hkv": hkv,
                "tokens": tokens, "start": _log_int(rng, 1, 32768) - 1, "weights": rng.random() < 0.6,
                "interleaved": rng.random() < 0.4, "table": rng.choice(["f32", "same"])}
    if op == "prompt":
        n = _log_int(rng, 1, 24)
        top = 8000 // n + 8
        lens, past = [], []
        chunked = rng.random() < 0.4
        for _ in range(n):
            lens.append(_log_int(rng, 1, top) if rng.random() > 0.05 else 0)
            past.append(_log_int(rng, 1, 8192 // n + 8) if chunked and rng.random() < 0.7 else 0)
        if not any(lens):
            lens[0] = 33
        return {"op": op, "dtype": rng.choice(["f16", "bf16"]), "hq": hq, "hkv": hkv,
                "q_lens": ",".join(map(str, lens)), "past": ",".join(map(str, past))}
    batch = _log_int(rng, 1, 8)
    return {"op": op, "dtype": rng.choice(["f16", "f16", "f32"]), "hq": hq, "hkv": hkv, "batch": batch,
            "fmt": rng.choice(["default", "adapter", "default", "adapter", "mixed"]),
            "cached": _log_int(rng, 1, 131072 // batch), "drafts": _log_int(rng, 1, 64)}


def _ints(text):
    return [int(x) for x in text.split(",")]


def work(case):
    hq, hkv = case["hq"], case["hkv"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        t = case["tokens"]
        table = 2 * 64 * (4 if case["table"] == "f32" else size)
        return {"bytes": t * ((hq + hkv) * D * 2 * size + table + 4), "flops": t * (hq + hkv) * D * (7 if case["weights"] else 3)}
    if case["op"] == "prompt":
        lens, past = _ints(case["q_lens"]), _ints(case["past"])
        pairs = sum(q * p + q * (q + 1) // 2 for q, p in zip(lens, past))
        keys = sum(q + p for q, p in zip(lens, past) if q)
        return {"bytes": size * D * (2 * sum(lens) * hq + 2 * keys * hkv), "flops": 4 * D * hq * pairs}
    l1, deep, split, int8 = FORMATS[case["fmt"]]
    row = (64 if int8 else 128) + (split // 2 * l1 + 7) // 8 + ((64 - split // 2) * deep + 7) // 8 + D + 8
    b, n, t = case["batch"], case["cached"], case["drafts"]
    pages = n // PAGE * PAGE
    per_head = pages * row + (n - pages) * 2 * D * size + t * 2 * D * size
    return {"bytes": b * (hkv * per_head + t * hq * D * (size + 2) + t * t), "flops": 4 * D * hq * b * t * (n + 1)}


# ------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _channel_scale():
    # Keys differ in size from channel to channel, as keys of trained models do.
    return torch.linspace(0.5, 4.0, D, device="cuda")[torch.randperm(D, generator=_generator(1), device="cuda")]


def _rope_inputs(case, gen):
    t, hq, hkv, dt = case["tokens"], case["hq"], case["hkv"], DTYPES[case["dtype"]]
    fused = _normal(gen, t, (hq + 2 * hkv) * D).to(dt)  # rows of the fused q, k, v projection
    positions = torch.arange(case["start"], case["start"] + t, device="cuda", dtype=torch.int32)
    freq = 500000.0 ** (-torch.arange(0, 64, device="cuda", dtype=torch.float64) / 64)
    angle = torch.arange(case["start"] + t, device="cuda", dtype=torch.float64)[:, None] * freq
    tdt = torch.float32 if case["table"] == "f32" else dt
    s = {"q": fused[:, :hq * D].view(t, hq, D), "k": fused[:, hq * D:(hq + hkv) * D].view(t, hkv, D),
         "cos": angle.cos().to(tdt), "sin": angle.sin().to(tdt), "positions": positions, "qw": None, "kw": None,
         "interleaved": case["interleaved"]}
    if case["weights"]:
        s["qw"] = (1 + 0.2 * _normal(gen, D)).to(dt)
        s["kw"] = (1 + 0.2 * _normal(gen, D)).to(dt)
    return s


def _prompt_inputs(case, gen):
    hq, hkv, dt = case["hq"], case["hkv"], DTYPES[case["dtype"]]
    lens, past = _ints(case["q_lens"]), _ints(case["past"])
    k_lens = [q + p for q, p in zip(lens, past)]
    tq, tk = sum(lens), sum(k_lens)
    fused = _normal(gen, tk, 2 * hkv * D).to(dt)  # the values stay where the fused projection wrote them
    return {"q": _normal(gen, tq, hq, D).to(dt), "k": (_normal(gen, tk, hkv, D) * _channel_scale()).to(dt),
            "v": fused[:, hkv * D:].view(tk, hkv, D), "q_lens": lens, "k_lens": k_lens}


def _tree_inputs(case, gen):
    b, hq, hkv, n, t = case["batch"], case["hq"], case["hkv"], case["cached"], case["drafts"]
    dt = DTYPES[case["dtype"]]
    scale = _channel_scale()
    k = (_normal(gen, b, hkv, n, D) * scale).to(dt)
    v = _normal(gen, b, hkv, n, D).to(dt)
    # A tree: each draft's parent is an earlier draft or the last cached token (-1); a draft sees
    # its ancestors and itself.
    parent = (torch.rand(t, generator=gen, device="cuda") * (torch.arange(t, device="cuda") + 1)).long() - 1
    parents = parent.tolist()
    mask = torch.zeros(t, t, dtype=torch.bool)
    for i in range(t):
        if parents[i] >= 0:
            mask[i] = mask[parents[i]]
        mask[i, i] = True
    return {"q": _normal(gen, b, hq, t, D).to(dt), "kd": (_normal(gen, b, hkv, t, D) * scale).to(dt),
            "vd": _normal(gen, b, hkv, t, D).to(dt), "mask": mask.cuda()}, k, v


def _angle_codes(k, l1, deep, split):
    """The cache's angle codes of key pairs, one byte per pair (64 pairs a row)."""
    x, y = k[..., 0::2], k[..., 1::2]
    a = torch.atan2(y.double(), x.double()).float()
    if k.dtype == torch.float16:
        a = ((a.half() + 3.140625) / 6.28125).clamp(0, 1).float()
    else:
        a = ((a + math.pi) / (2 * math.pi)).clamp(0, 1)
        a = torch.where(a > 1.0 - 1e-6, torch.zeros_like(a), a)
    levels = torch.full((64,), float(2 ** deep - 1), device="cuda")
    levels[:split // 2] = float(2 ** l1 - 1)
    return (a * levels).round().to(torch.uint8)


def _encode(k, v, fmt):
    """The cached pages of dense keys and values (B, H, n * 64, 128): what the page store holds."""
    l1, deep, split, int8 = FORMATS[fmt]
    b, h, n, _ = k.shape
    x, y = k[..., 0::2], k[..., 1::2]
    radii = (x * x + y * y).sqrt().half().view(b, h, n // PAGE, PAGE, 64)
    page = {"codes": _angle_codes(k, l1, deep, split).view(b, h, n // PAGE, PAGE, 64), "radii": radii, "scales": None}
    if int8:
        log = radii.clamp_min(torch.tensor(1e-6, dtype=torch.float16, device="cuda")).double().log().float().half().float()
        scale = (log.abs().amax((-1, -2), keepdim=True) / 127.0).half()
        page["radii"] = (log / scale.float()).round().clamp(-128, 127).to(torch.int8)
        page["scales"] = scale
    g = v.reshape(b, h, n // PAGE, PAGE, 4, 32)
    vs = (g.abs().amax(-1, keepdim=True).float() / 127.0).half()
    vs = torch.where(vs == 0, torch.full_like(vs, 1e-4), vs)
    ratio = g.float() / vs.float()
    if v.dtype == torch.float16:
        ratio = ratio.half().float()
    page["v"] = ratio.round().clamp(-128, 127).to(torch.int8)
    page["vs"] = vs
    return page


def prepare(case, seed):
    gen = _generator(seed)
    if case["op"] == "rope":
        return {"case": case, **_rope_inputs(case, gen)}
    if case["op"] == "prompt":
        s = {"case": case, **_prompt_inputs(case, gen)}
        if own:  # the plan of these lengths, which all layers of a model share
            from turbopolar_b200 import PromptPlan
            s["plan"] = PromptPlan(s["q_lens"], s["k_lens"], num_q_heads=case["hq"], num_kv_heads=case["hkv"], device="cuda")
        return s
    inputs, k, v = _tree_inputs(case, gen)
    s = {"case": case, **inputs}
    if own:  # the cache as a program has it: filled by appends
        from turbopolar_b200 import TurboPolarConfig, TurboPolarKVCacheRuntime
        l1, deep, split, int8 = FORMATS[case["fmt"]]
        config = TurboPolarConfig(k_angle_bits_level1=l1, k_angle_bits_deep=deep, split_dim=split, use_int8_radii=bool(int8),
                                  num_q_heads=case["hq"], num_kv_heads=case["hkv"])
        s["cache"] = TurboPolarKVCacheRuntime(config, max_seq_len=case["cached"] + 1, check_finite=False)
        s["cache"].append(k, v)
        return s
    full = case["cached"] // PAGE * PAGE
    s["pages"] = _encode(k[:, :, :full], v[:, :, :full], case["fmt"]) if full else None
    s["tail_k"], s["tail_v"] = k[:, :, full:].clone(), v[:, :, full:].clone()
    return s


# ------------------------------------------------------------------------------------------- passes
def run(state):
    op = state["case"]["op"]
    if op == "rope":
        return _rope_own(state) if own else _rope_plain(state)
    if op == "prompt":
        return _prompt_own(state) if own else _prompt_plain(state)
    return _tree_own(state) if own else _tree_plain(state)


def _rope_own(s):
    from turbopolar_b200 import norm_rope
    return norm_rope(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], q_weight=s["qw"], k_weight=s["kw"],
                     eps=1e-6, interleaved=s["interleaved"])


def _prompt_own(s):
    from turbopolar_b200 import prompt_attention
    return prompt_attention(s["q"], s["k"], s["v"], s["plan"])


def _tree_own(s):
    return s["cache"].tree_attention(s["q"], s["kd"], s["vd"], s["mask"])


def _rope_one(x, w, cos, sin, interleaved):
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
    if interleaved:
        a, b = y[..., 0::2], y[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2).to(x.dtype)
    a, b = y[..., :64], y[..., 64:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _rope_plain(s):
    cos = s["cos"][s["positions"]].float()[:, None]
    sin = s["sin"][s["positions"]].float()[:, None]
    return _rope_one(s["q"], s["qw"], cos, sin, s["interleaved"]), _rope_one(s["k"], s["kw"], cos, sin, s["interleaved"])


def _softmax_values(scores, v):
    """softmax over the last axis (rows with nothing visible give 0) times v; the scores are overwritten."""
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return (p @ v) / total.clamp_min(torch.finfo(torch.float32).tiny)


def _prompt_plain(s):
    q, k, v = s["q"], s["k"], s["v"]
    hq, hkv = q.shape[1], k.shape[1]
    out = torch.empty_like(q)
    qa = ka = 0
    for nq, nk in zip(s["q_lens"], s["k_lens"]):  # each sequence by itself: the packed mask of all would do more work
        if nq:
            qs = (q[qa:qa + nq].float() * D ** -0.5).transpose(0, 1).reshape(hkv, hq // hkv * nq, D)
            ks = k[ka:ka + nk].float().permute(1, 2, 0)
            vs = v[ka:ka + nk].float().transpose(0, 1)
            scores = qs @ ks
            hidden = torch.arange(nk, device="cuda") > torch.arange(nq, device="cuda")[:, None] + (nk - nq)
            scores.view(hkv, hq // hkv, nq, nk).masked_fill_(hidden, float("-inf"))
            out[qa:qa + nq] = _softmax_values(scores, vs).view(hq, nq, D).transpose(0, 1).to(q.dtype)
        qa, ka = qa + nq, ka + nk
    return out


def _decoded(page, fmt):
    """float32 keys and values (B, H, tokens, 128) of cached pages; each is a float16 number."""
    l1, deep, split, int8 = FORMATS[fmt]
    levels = torch.full((64,), float(2 ** deep - 1), device="cuda")
    levels[:split // 2] = float(2 ** l1 - 1)
    angle = page["codes"].float() / levels * (2 * math.pi) - math.pi
    r = page["radii"].float()
    if int8:
        r = (r * page["scales"].float()).exp()
    k = torch.stack([r * angle.cos(), r * angle.sin()], -1).flatten(-2).half().float()
    v = (page["v"].float() * page["vs"].float()).half().float()
    b, h = k.shape[:2]
    return k.view(b, h, -1, D), v.view(b, h, -1, D)


def _tree_plain(s):
    q, mask = s["q"], s["mask"]
    b, hq, t, _ = q.shape
    hkv = s["kd"].shape[1]
    k, v = [s["tail_k"].float(), s["kd"].float()], [s["tail_v"].float(), s["vd"].float()]
    if s["pages"] is not None:
        pk, pv = _decoded(s["pages"], s["case"]["fmt"])
        k, v = [pk] + k, [pv] + v
    k, v = torch.cat(k, 2), torch.cat(v, 2)
    qs = (q.float() * D ** -0.5).reshape(b, hkv, hq // hkv * t, D)
    scores = qs @ k.transpose(-1, -2)
    scores.view(b, hkv, hq // hkv, t, -1)[..., -t:].masked_fill_(~mask, float("-inf"))
    return _softmax_values(scores, v).view(b, hq, t, D).half()


# ------------------------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    gen = _generator(seed)
    if case["op"] == "rope":
        s = _rope_inputs(case, gen)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()].unsqueeze(1)
        return tuple(_turned(s[x].double(), s[w], turn, s["interleaved"]) for x, w in (("q", "qw"), ("k", "kw")))
    if case["op"] == "prompt":
        s = _prompt_inputs(case, gen)
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        q0 = k0 = 0
        for nq, nk in zip(s["q_lens"], s["k_lens"]):
            last = torch.arange(nk - nq, nk, device="cuda").unsqueeze(1)  # the last key that each row sees
            for h in range(case["hq"]):
                g = h // (case["hq"] // case["hkv"])
                for r in range(0, nq, 4096):
                    rows = slice(r, min(r + 4096, nq))
                    seen = torch.arange(nk, device="cuda") <= last[rows]
                    out[q0 + r:q0 + rows.stop, h] = _attended(s["q"][q0 + r:q0 + rows.stop, h], s["k"][k0:k0 + nk, g],
                                                              s["v"][k0:k0 + nk, g], seen)
            q0, k0 = q0 + nq, k0 + nk
        return out
    s, k, v = _tree_inputs(case, gen)
    full = case["cached"] // PAGE * PAGE
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    seen = torch.cat([torch.ones(case["drafts"], case["cached"], dtype=torch.bool, device="cuda"), s["mask"]], 1)
    for i in range(case["batch"]):
        for g in range(case["hkv"]):
            kk, vv = k[i, g].double(), v[i, g].double()
            if full:
                kk[:full], vv[:full] = _stored(k[i, g, :full], v[i, g, :full], case["fmt"])
            kk, vv = torch.cat([kk, s["kd"][i, g].double()]), torch.cat([vv, s["vd"][i, g].double()])
            for h in range(case["hq"] // case["hkv"] * g, case["hq"] // case["hkv"] * (g + 1)):
                out[i, h] = _attended(s["q"][i, h], kk, vv, seen)
    return out


def _turned(x, w, turn, interleaved):
    if w is not None:
        x = x / (x.square().sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
    pairs = x.unflatten(-1, (64, 2)) if interleaved else x.unflatten(-1, (2, 64)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    return z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)


def _attended(q, k, v, seen):
    if not k.shape[0]:
        return torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    w = torch.where(seen, q.double() @ k.double().T / math.sqrt(D), -math.inf).softmax(-1)
    return torch.where(seen.any(-1, keepdim=True), torch.nan_to_num(w) @ v.double(), 0.0)


def _stored(k, v, fmt):
    """What one head's full pages hold for keys and values (n, 128), as the float16 numbers they decode to."""
    l1, deep, split, int8 = FORMATS[fmt]
    n = k.shape[0]
    page = _encode(k[None, None], v[None, None], fmt)
    steps = torch.where(torch.arange(64, device="cuda") < split // 2, 2 ** l1 - 1, 2 ** deep - 1).double()
    theta = (page["codes"].double() / steps - 0.5) * (2 * math.pi)
    r = page["radii"].double()
    if int8:
        r = torch.exp(r * page["scales"].double())
    kk = torch.view_as_real(torch.polar(r, theta)).reshape(n, D)
    vv = (page["v"].double() * page["vs"].double()).reshape(n, D)
    return kk.half().double(), vv.half().double()
