"""DraftDecoder.accept: what it appends, and when it refuses before any layer is appended to."""

import pytest
import torch


class _Runtime:
    d_state = None

    def __init__(self):
        self.tokens = []

    def append(self, k, v):
        assert k.dtype == v.dtype == torch.float16
        self.tokens += k[0, 0, :, 0].tolist()


class _Layer:
    def __init__(self):
        self.runtime = _Runtime()

    @property
    def offset(self):
        return 10 + len(self.runtime.tokens)


@pytest.fixture
def decoder(monkeypatch):
    """A decoder of two layers after verify() of the tree 0 - (1 - 3, 2), 4, with stand-in caches."""
    from turbopolar_b200.llama_drafts import DraftDecoder
    dec = DraftDecoder.__new__(DraftDecoder)
    dec.device, dec.cache = torch.device("cpu"), [_Layer(), _Layer()]
    dec._prompt_error = torch.zeros(1, dtype=torch.int32)
    dec._drafts = []

    class Model:
        lm_head = staticmethod(lambda x: x)

    class Attn:
        scaling = 1.0

    dec.model = Model()

    def layers(tokens, positions, attend):
        rows = tokens.float()[None, None, :, None].expand(1, 2, -1, 128)
        for i, layer in enumerate(dec.cache):
            layer.tree_attention = lambda q, k, v, mask, scale: q
            attend(i, Attn, rows[0].transpose(0, 1), rows[0].transpose(0, 1), rows[0].transpose(0, 1))
            if dec.fails_after == i:
                raise MemoryError("no room")
        return rows[0, 0]

    dec.fails_after = None
    monkeypatch.setattr(dec, "_layers", layers, raising=False)
    dec.verify(torch.tensor([50, 51, 52, 53, 54]), [-1, 0, 0, 1, -1])
    return dec


def _appended(dec):
    return [layer.runtime.tokens for layer in dec.cache]


def test_a_path_is_appended_to_every_layer_once(decoder):
    decoder.accept([0, 1, 3])
    assert _appended(decoder) == [[50, 51, 53]] * 2
    with pytest.raises(RuntimeError, match="follows verify"):
        decoder.accept([0])


@pytest.mark.parametrize("path", [[1], [0, 3], [0, 4], [4, 0], [0, 0], [5], [-1], [0, 1, 2]])
def test_paths_that_are_none(decoder, path):
    with pytest.raises(ValueError, match="path"):
        decoder.accept(path)
    assert _appended(decoder) == [[], []]
    decoder.accept([4])   # the verification still stands
    assert _appended(decoder) == [[54], [54]]


def test_an_empty_path_accepts_nothing(decoder):
    decoder.accept([])
    assert _appended(decoder) == [[], []]
    with pytest.raises(RuntimeError, match="follows verify"):
        decoder.accept([0])


def test_a_verification_that_failed_halfway_is_not_accepted(decoder):
    decoder.fails_after = 0
    with pytest.raises(MemoryError):
        decoder.verify(torch.tensor([60, 61]), [-1, 0])
    with pytest.raises(RuntimeError, match="follows verify"):
        decoder.accept([0])
    assert _appended(decoder) == [[], []]


def test_caches_that_moved_on_are_not_appended_to(decoder):
    decoder.cache[1].runtime.tokens.append(99)
    with pytest.raises(RuntimeError, match="changed since verify"):
        decoder.accept([0])
    assert _appended(decoder) == [[], [99]]


@pytest.mark.gpu
def test_a_prompt_chunk_ends_the_verification():
    from transformers import LlamaConfig, LlamaForCausalLM
    from turbopolar_b200.llama_drafts import DraftDecoder
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=64, hidden_size=512, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128)
    dec = DraftDecoder(LlamaForCausalLM(cfg).to("cuda", torch.float16).eval())
    dec.prefill(torch.arange(20, device="cuda"))
    dec.verify(torch.tensor([1, 2], device="cuda"), [-1, 0])
    dec.prefill(torch.arange(3, device="cuda"))
    with pytest.raises(RuntimeError, match="follows verify"):
        dec.accept([0])
    assert dec.offset == 23
