"""Prompt chunks and drafted tokens of a small random-init Llama on the TurboPolar cache, against the
adapter's own path (stock attention for the prompt, one fused step per token).

Both paths run float16 layers with differently ordered sums, so logits (of size up to about 1 here) may differ
by float16 rounding that is carried through the layers: 2 layers of about 10 roundings of 2^-11 of the
hidden state, 2e-2 of the logits' size at most."""

import pytest
import torch


def test_tree_mask():
    from turbopolar_b200.llama_drafts import tree_mask
    m = tree_mask([-1, 0, 0, 2, -1])
    assert m.int().tolist() == [[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 0, 1, 1, 0], [0, 0, 0, 0, 1]]
    for bad in ([0], [-1, 1], [-2]):
        with pytest.raises(ValueError, match="parent"):
            tree_mask(bad)


def test_ngram_drafter():
    from turbopolar_b200.llama_drafts import ngram_drafter
    draft = ngram_drafter(width=2, depth=2)
    assert draft([5, 6, 7, 5, 8, 9, 5]) == ([8, 9, 6, 7], [-1, 0, -1, 2])
    assert draft([1, 2, 3]) == ([], [])


def _model(dtype=torch.float16, hq=4, hkv=2):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=512, hidden_size=hq * 128, intermediate_size=512, num_hidden_layers=2,
                      num_attention_heads=hq, num_key_value_heads=hkv, head_dim=128, max_position_embeddings=4096,
                      attn_implementation="sdpa")
    return LlamaForCausalLM(cfg).to("cuda", dtype).eval()


def _steps(model, prompt, tokens):
    """Logits after the prompt and after each token, with the adapter's fused one-token steps."""
    from turbopolar_b200 import llama
    cache = llama.make_turbo_caches(2, model.config.num_attention_heads, model.config.num_key_value_heads, 128,
                                    device="cuda", max_seq_len=1024)
    llama.patch_llama_attention(model)
    try:
        with torch.no_grad():
            rows = [model(input_ids=prompt[None], past_key_values=cache, use_cache=True).logits[0, -1].float()]
            for t in tokens:
                rows.append(model(input_ids=torch.tensor([[t]], device="cuda"), past_key_values=cache,
                                  use_cache=True).logits[0, -1].float())
    finally:
        llama.unpatch_llama_attention(model)
    return torch.stack(rows)


def _near(a, b):
    assert (a - b).abs().max() <= 2e-2 * b.abs().max(), float((a - b).abs().max() / b.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 64, 333])
def test_prefill_and_verify_agree_with_one_token_steps(n):
    from turbopolar_b200.llama_drafts import DraftDecoder
    model = _model()
    prompt = torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(n)).cuda()
    #        0 - 1 - 3
    #          \ 2 - 4      5 is another root
    tokens, parents = [7, 100, 200, 300, 400, 9], [-1, 0, 0, 1, 2, -1]
    dec = DraftDecoder(model, max_seq_len=1024)
    first = dec.prefill(prompt)
    logits = dec.verify(torch.tensor(tokens, device="cuda"), parents)
    assert dec.offset == n
    for path in ([0, 1, 3], [0, 2, 4], [5]):
        want = _steps(model, prompt, [tokens[i] for i in path])
        _near(first, want[0])
        for i, row in zip(path, want[1:]):
            _near(logits[i], row)
    # The accepted path becomes part of the cache.
    dec.accept([0, 2])
    assert dec.offset == n + 2
    _near(dec.verify(torch.tensor([400], device="cuda"), [-1])[0], logits[4])
    with pytest.raises(RuntimeError, match="verify"):
        DraftDecoder(model).accept([0])


@pytest.mark.gpu
def test_prompt_in_chunks():
    from turbopolar_b200.llama_drafts import DraftDecoder
    model = _model()
    prompt = torch.randint(0, 512, (200,), generator=torch.Generator().manual_seed(1)).cuda()
    whole = DraftDecoder(model).prefill(prompt)
    dec = DraftDecoder(model)
    for a, b in ((0, 64), (64, 150), (150, 151), (151, 200)):
        last = dec.prefill(prompt[a:b])
    # Chunks that end inside a page read its rows encoded with zeros in place of later tokens (one
    # radius scale per page), so the histories differ by the format's own error.
    assert torch.nn.functional.cosine_similarity(last, whole, dim=0) > 0.99


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_generate_chooses_what_one_token_steps_choose(dtype):
    from turbopolar_b200.llama_drafts import DraftDecoder, ngram_drafter
    model = _model(dtype)
    prompt = torch.randint(0, 24, (150,), generator=torch.Generator().manual_seed(2)).cuda()
    tokens, steps = DraftDecoder(model, max_seq_len=1024).generate(prompt, 40, ngram_drafter())
    assert len(tokens) == 40 and steps <= 40
    rows = _steps(model, prompt, tokens[:-1])
    for row, t in zip(rows, tokens):   # the best token up to the paths' rounding difference
        assert row[t] >= row.max() - (4e-2 if dtype == torch.float16 else 0.2) * row.abs().max()


@pytest.mark.gpu
def test_head_norms_of_a_model_are_used():
    from turbopolar_b200.llama_drafts import DraftDecoder
    model = _model()

    class Norm(torch.nn.Module):
        variance_epsilon = 1e-5

        def __init__(self, w):
            super().__init__()
            self.weight = torch.nn.Parameter(w)

    prompt = torch.arange(40, device="cuda")
    plain = DraftDecoder(model).prefill(prompt)
    for layer in model.model.layers:
        layer.self_attn.q_norm = Norm(torch.full((128,), 3.0, device="cuda", dtype=torch.float16))
        layer.self_attn.k_norm = Norm(torch.full((128,), 3.0, device="cuda", dtype=torch.float16))
    assert not torch.allclose(DraftDecoder(model).prefill(prompt), plain, atol=1e-3)
