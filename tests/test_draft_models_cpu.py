"""Models that DraftDecoder does not compute are refused before anything is appended."""

import pytest
import torch

SIZES = dict(vocab_size=32, hidden_size=256, intermediate_size=64, num_hidden_layers=2, num_attention_heads=2,
             num_key_value_heads=1, head_dim=128)


def _decoder(model):
    from turbopolar_b200.llama_drafts import DraftDecoder
    return DraftDecoder(model)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_llama(dtype):
    from transformers import LlamaConfig, LlamaForCausalLM
    assert len(list(_decoder(LlamaForCausalLM(LlamaConfig(**SIZES)).to(dtype)).cache)) == 2


def test_float32_models_are_refused():
    from transformers import LlamaConfig, LlamaForCausalLM
    with pytest.raises(NotImplementedError, match="float16 or bfloat16"):
        _decoder(LlamaForCausalLM(LlamaConfig(**SIZES)).float())


def test_sliding_windows_are_refused():
    from transformers import MistralConfig, MistralForCausalLM, Qwen3Config, Qwen3ForCausalLM
    with pytest.raises(NotImplementedError, match="whole history"):
        _decoder(MistralForCausalLM(MistralConfig(**SIZES, sliding_window=64)).half())
    _decoder(MistralForCausalLM(MistralConfig(**SIZES, sliding_window=None)).half())
    some = Qwen3Config(**SIZES, use_sliding_window=True, sliding_window=64, max_window_layers=1)
    with pytest.raises(NotImplementedError, match="whole history"):
        _decoder(Qwen3ForCausalLM(some).half())
    _decoder(Qwen3ForCausalLM(Qwen3Config(**SIZES, use_sliding_window=False)).half())


def test_rotation_of_a_part_of_each_head_is_refused():
    from transformers import LlamaConfig, LlamaForCausalLM
    model = LlamaForCausalLM(LlamaConfig(**SIZES)).half()
    dec = _decoder(model)

    class Half(torch.nn.Module):
        def forward(self, x, positions):
            return (torch.ones(1, positions.shape[1], 64).half(),) * 2

    model.model.rotary_emb = Half()
    with pytest.raises(NotImplementedError, match="whole heads"):
        dec._layers(torch.arange(3), torch.arange(3), None)
