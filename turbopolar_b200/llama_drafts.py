"""Prompts and drafted tokens of a Hugging Face Llama model on the TurboPolar cache.

The reference's adapter decodes one token at a time (``benchmarks/turbopolar_fast_attention.py:
247-278``) and leaves prompts to MLX's dense attention (``:56-86``).  Here one layer of a prompt
chunk or of a tree of drafted tokens is: projections, :func:`~turbopolar_b200.norm_rope` (rotation,
with the head norms of models that have them), then

* a prompt chunk: append, decompress-on-read of the history, :func:`~turbopolar_b200.prompt_attention`;
* a tree of drafts: ``tree_attention`` over the compressed cache; the accepted path is appended
  afterwards.

:class:`DraftDecoder` runs a model that way: :meth:`~DraftDecoder.prefill`,
:meth:`~DraftDecoder.verify` (logits of every draft), :meth:`~DraftDecoder.accept`,
:meth:`~DraftDecoder.check` (error words of the kernels), and :meth:`~DraftDecoder.generate`, greedy
decoding whose tokens are those of one-token steps.

``python -m turbopolar_b200.llama_drafts`` decodes with a random-init model.
"""

from __future__ import annotations

import argparse
import time
from typing import Callable, List, Optional, Sequence, Tuple

import torch

from .llama import TurboPolarCache, make_turbo_caches
from .prompt import PromptPlan, prompt_attention
from .rotary import norm_rope


def tree_mask(parents: Sequence[int], device=None) -> torch.Tensor:
    """``(T, T)`` bool: draft ``t`` sees its ancestors and itself.  ``parents[t]`` is the index of an
    earlier draft, or -1 where the draft follows the last cached token."""
    n = len(parents)
    mask = torch.zeros(n, n, dtype=torch.bool)
    for t, p in enumerate(parents):
        if not -1 <= p < t:
            raise ValueError(f"parent {p} of draft {t} must be -1 or an earlier draft")
        if p >= 0:
            mask[t] = mask[p]
        mask[t, t] = True
    return mask.to(device)


def _check_model(model) -> None:
    """Refuse models whose attention is not causal attention over the whole history with heads of 128 channels,
    in a type that ``prompt_attention`` takes."""
    cfg = model.config
    head_dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
    if head_dim != 128:
        raise NotImplementedError("TurboPolar only supports head_dim == 128")
    layers = [layer.self_attn for layer in model.model.layers]
    windows = [getattr(cfg, "sliding_window", None) if getattr(cfg, "use_sliding_window", True) else None]
    windows += [getattr(a, "sliding_window", None) for a in layers]
    kinds = set(getattr(cfg, "layer_types", None) or ["full_attention"])
    if any(w is not None for w in windows) or kinds != {"full_attention"}:
        raise NotImplementedError("DraftDecoder attends the whole history; this model has layers of other attention")
    if getattr(cfg, "attn_logit_softcapping", None) is not None or any(getattr(a, "sinks", None) is not None for a in layers):
        raise NotImplementedError("DraftDecoder knows plain softmax attention only")
    dtype = model.model.embed_tokens.weight.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise NotImplementedError(f"DraftDecoder needs a float16 or bfloat16 model, got {dtype}")


def _norm_eps(attn) -> float:
    """The epsilon of an attention's head norms.  Only norms as Llama's own (``x * rsqrt(mean(x^2) +
    variance_epsilon) * weight``) are known; others have an ``eps`` or another use of the weight."""
    norms = [n for n in (getattr(attn, "q_norm", None), getattr(attn, "k_norm", None)) if n is not None]
    eps = {getattr(n, "variance_epsilon", None) for n in norms}
    if None in eps or len(eps) > 1:
        raise NotImplementedError("head norms need one variance_epsilon, as Llama's RMSNorm has")
    return eps.pop() if eps else 0.0


class DraftDecoder:
    """A Hugging Face Llama model (batch 1, head_dim 128, float16 or bfloat16, attention over the whole history)
    over per-layer TurboPolar caches."""

    def __init__(self, model, cache: Optional[TurboPolarCache] = None, max_seq_len: Optional[int] = None,
                 check_finite: bool = False):
        _check_model(model)
        cfg = model.config
        self.model, self.device = model, next(model.parameters()).device
        self.hq, self.hkv = cfg.num_attention_heads, cfg.num_key_value_heads
        self.cache = cache if cache is not None else make_turbo_caches(
            cfg.num_hidden_layers, self.hq, self.hkv, 128, device=self.device, max_seq_len=max_seq_len,
            check_finite=check_finite)
        # Of the last verify(): per layer the drafts' keys and values; their parents; the offset they follow.
        self._drafts: List[Tuple[torch.Tensor, torch.Tensor]] = []
        self._parents: List[int] = []
        self._verified_at = 0
        self._prompt_error = torch.zeros(1, dtype=torch.int32, device=self.device)  # of all prompts so far

    @property
    def offset(self) -> int:
        return self.cache[0].offset

    def check(self) -> None:
        """Raise ``RuntimeError`` where a kernel of a prompt, a verification or an append has reported that its
        results are unusable.  Synchronises; :meth:`accept` calls it before it appends."""
        words = torch.cat([self._prompt_error, *(layer.runtime.d_state[4:5] for layer in self.cache
                                                 if layer.runtime.d_state is not None)]).tolist()
        if any(words):
            raise RuntimeError(f"TurboPolar kernels reported errors (prompt attention {words[0]}, layers {words[1:]})")

    def _qkv(self, attn, x, cos, sin):
        t = x.shape[1]
        q, k, v = (p(x)[0].view(t, -1, 128) for p in (attn.q_proj, attn.k_proj, attn.v_proj))
        norms = [getattr(attn, name, None) for name in ("q_norm", "k_norm")]
        q, k = norm_rope(q, k, cos, sin, q_weight=getattr(norms[0], "weight", None),
                         k_weight=getattr(norms[1], "weight", None), eps=_norm_eps(attn))
        return q, k, v

    def _layers(self, tokens: torch.Tensor, positions: torch.Tensor, attend: Callable) -> torch.Tensor:
        """Final hidden states of ``tokens`` ``(T,)``; ``attend(layer, attn, q, k, v)`` is the attention."""
        base = self.model.model
        x = base.embed_tokens(tokens[None])
        tables = base.rotary_emb(x, positions[None])
        if any(r.shape[-1] != 128 for r in tables):
            raise NotImplementedError("norm_rope rotates whole heads; this model rotates a part of each")
        cos, sin = (r[0, :, :64] for r in tables)
        for i, layer in enumerate(base.layers):
            h = layer.input_layernorm(x)
            o = attend(i, layer.self_attn, *self._qkv(layer.self_attn, h, cos, sin))
            x = x + layer.self_attn.o_proj(o.to(x.dtype).reshape(1, len(tokens), -1))
            x = x + layer.mlp(layer.post_attention_layernorm(x))
        return base.norm(x)[0]

    @torch.no_grad()
    def prefill(self, tokens: torch.Tensor) -> torch.Tensor:
        """Append a prompt or a further chunk of it ``(T,)``; float32 logits of its last token."""
        self._drafts = []  # drafts of an earlier verify() are rotated for another offset
        start, n = self.offset, len(tokens)
        plan = PromptPlan([n], [start + n], num_q_heads=self.hq, num_kv_heads=self.hkv, device=self.device)

        def attend(i, attn, q, k, v):
            heads_first = lambda y: y.transpose(0, 1)[None]
            hist = self.cache[i].update_and_fetch(heads_first(k), heads_first(v))
            return prompt_attention(q, *(y[0].transpose(0, 1) for y in hist), plan, scale=attn.scaling)

        positions = torch.arange(start, start + n, device=self.device)
        logits = self.model.lm_head(self._layers(tokens, positions, attend)[-1]).float()
        self._prompt_error |= plan.device_error
        return logits

    @torch.no_grad()
    def verify(self, tokens: torch.Tensor, parents: Sequence[int]) -> torch.Tensor:
        """float32 logits ``(T, vocab)`` after each draft of a tree; the cache stays as it is."""
        if len(tokens) != len(parents):
            raise ValueError(f"{len(tokens)} drafts and {len(parents)} parents")
        mask = tree_mask(parents, self.device)
        depth = mask.sum(1) - 1
        self._drafts, drafts = [], []

        def attend(i, attn, q, k, v):
            heads_first = lambda y: y.transpose(0, 1)[None]
            k, v = heads_first(k), heads_first(v)
            drafts.append((k, v))
            return self.cache[i].tree_attention(heads_first(q), k, v, mask, attn.scaling).transpose(1, 2)

        logits = self.model.lm_head(self._layers(tokens, self.offset + depth, attend)).float()
        self._drafts, self._parents, self._verified_at = drafts, list(parents), self.offset
        return logits

    @torch.no_grad()
    def accept(self, path: Sequence[int]) -> None:
        """Append the drafts ``path`` of the last :meth:`verify`: a root, one of its children, and so on.  An
        empty path accepts none."""
        if not self._drafts:
            raise RuntimeError("accept() follows verify()")
        path = [int(i) for i in path]
        for parent, i in zip([-1, *path], path):
            if not 0 <= i < len(self._parents) or self._parents[i] != parent:
                raise ValueError(f"path {path} is not a root of the verified drafts with its descendants")
        if any(layer.offset != self._verified_at for layer in self.cache):
            raise RuntimeError("the caches have changed since verify()")
        if not path:
            self._drafts = []
            return
        self.check()
        index = torch.tensor(path, device=self.device)
        for layer, (k, v) in zip(self.cache, self._drafts):
            layer.runtime.append(k[:, :, index].to(torch.float16), v[:, :, index].to(torch.float16))
        self._drafts = []

    def generate(self, prompt: torch.Tensor, new_tokens: int,
                 drafter: Callable[[List[int]], Tuple[List[int], List[int]]]) -> Tuple[List[int], int]:
        """Greedy tokens after ``prompt``, and the number of verification steps they took.

        ``drafter(tokens)`` proposes ``(drafts, parents)`` for what follows ``tokens``; parents are
        indices of earlier drafts, -1 for the roots.  Each step verifies the last accepted token
        with the drafts under it and keeps the drafts that greedy decoding would have chosen."""
        history = prompt.tolist()
        last, steps, out = int(self.prefill(prompt).argmax()), 0, []
        while len(out) < new_tokens:
            out.append(last)
            history.append(last)
            drafts, parents = drafter(history)
            tokens = torch.tensor([last, *drafts], device=self.device)
            best = self.verify(tokens, [-1, *(p + 1 for p in parents)]).argmax(-1).tolist()
            steps += 1
            path, at = [0], 0
            while True:
                at = next((i + 1 for i, (d, p) in enumerate(zip(drafts, parents)) if p + 1 == at and d == best[at]), None)
                if at is None:
                    break
                path.append(at)
            self.accept(path)
            out += [int(tokens[i]) for i in path[1:]]
            history += [int(tokens[i]) for i in path[1:]]
            last = best[path[-1]]
        return out[:new_tokens], steps


def ngram_drafter(width: int = 2, depth: int = 4) -> Callable[[List[int]], Tuple[List[int], List[int]]]:
    """Drafts from the text itself: what followed the last ``width`` other occurrences of the last
    token, ``depth`` tokens of each, as a tree of chains."""

    def draft(tokens: List[int]):
        drafts, parents, found = [], [], 0
        for i in range(len(tokens) - 2, -1, -1):
            if tokens[i] != tokens[-1]:
                continue
            parent = -1
            for t in tokens[i + 1:i + 1 + depth]:
                drafts.append(t)
                parents.append(parent)
                parent = len(drafts) - 1
            found += 1
            if found == width:
                break
        return drafts, parents

    return draft


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--vocab", type=int, default=4096)
    ap.add_argument("--prompt", type=int, default=1024)
    ap.add_argument("--new", type=int, default=64)
    a = ap.parse_args(argv)
    from .bench_llama import build_model
    dev = torch.device("cuda:0")
    model = build_model(a.layers, a.vocab, dev)
    prompt = torch.randint(0, a.vocab, (a.prompt,), generator=torch.Generator().manual_seed(3)).to(dev)
    decoder = DraftDecoder(model, max_seq_len=a.prompt + a.new + 64)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    tokens, steps = decoder.generate(prompt, a.new, ngram_drafter())
    torch.cuda.synchronize()
    print(f"{len(tokens)} tokens in {steps} verification steps after a prompt of {a.prompt}, "
          f"{time.perf_counter() - t0:.2f} s: {tokens[:16]} ...")


if __name__ == "__main__":
    main()
