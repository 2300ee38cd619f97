"""Error words that the kernels of prompts and drafts set reach the caller.  The words are set from the host: no
wait is made to run out."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _decoder():
    from transformers import LlamaConfig, LlamaForCausalLM
    from turbopolar_b200.llama_drafts import DraftDecoder
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=64, hidden_size=512, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128)
    return DraftDecoder(LlamaForCausalLM(cfg).to("cuda", torch.float16).eval(), max_seq_len=512)


def test_a_failed_verification_is_not_accepted():
    dec = _decoder()
    dec.check()   # before any call
    dec.prefill(torch.arange(40, device="cuda"))
    dec.verify(torch.tensor([1, 2, 3], device="cuda"), [-1, 0, 1])
    dec.check()
    rt = dec.cache[1].runtime
    rt.d_state[4] = 3   # what the kernel writes when a wait runs out
    assert rt.read_device_error() == 3
    with pytest.raises(RuntimeError, match=r"layers \[0, 3\]"):
        dec.accept([0, 1])
    assert dec.offset == 40 and all(layer.runtime.actual_seq_len == 40 for layer in dec.cache)


def test_the_word_outlives_a_larger_scratch():
    dec = _decoder()
    dec.prefill(torch.arange(40, device="cuda"))
    rt = dec.cache[0].runtime
    dec.verify(torch.tensor([1, 2], device="cuda"), [-1, 0])
    rt.d_state[4] = 3
    dec.verify(torch.zeros(200, dtype=torch.long, device="cuda"), [-1] * 200)
    assert rt.read_device_error() == 3


def test_a_failed_prompt_stops_the_generation(monkeypatch):
    from turbopolar_b200 import llama_drafts, prompt
    dec = _decoder()
    made = []

    class Plan(prompt.PromptPlan):
        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            self.device_error.fill_(len(made) == 0)   # the first plan's
            made.append(1)

    monkeypatch.setattr(llama_drafts, "PromptPlan", Plan)
    dec.prefill(torch.arange(10, device="cuda"))
    dec.prefill(torch.arange(10, device="cuda"))      # a later chunk does not hide it
    with pytest.raises(RuntimeError, match="prompt attention 1"):
        dec.check()
    dec = _decoder()
    made.clear()
    with pytest.raises(RuntimeError, match="prompt attention 1"):
        dec.generate(torch.arange(10, device="cuda"), 4, llama_drafts.ngram_drafter())
