"""Head norms that DraftDecoder takes from a model: their own epsilon, and only of the kind that it computes."""

import pytest
import torch


class _Attn:
    def __init__(self, q_norm=None, k_norm=None):
        self.q_proj = self.k_proj = self.v_proj = lambda x: x
        if q_norm is not None:
            self.q_norm = q_norm
        if k_norm is not None:
            self.k_norm = k_norm


class _Norm:
    def __init__(self, **fields):
        self.weight = torch.ones(128)
        self.__dict__.update(fields)


@pytest.fixture
def eps_of(monkeypatch):
    from turbopolar_b200 import llama_drafts
    seen = []
    monkeypatch.setattr(llama_drafts, "norm_rope", lambda q, k, cos, sin, q_weight, k_weight, eps: seen.append(eps) or (q, k))
    dec = llama_drafts.DraftDecoder.__new__(llama_drafts.DraftDecoder)

    def call(attn):
        dec._qkv(attn, torch.zeros(1, 3, 256), None, None)
        return seen[-1]

    return call


def test_the_norms_own_epsilon_is_used(eps_of):
    assert eps_of(_Attn(_Norm(variance_epsilon=1e-5), _Norm(variance_epsilon=1e-5))) == 1e-5
    assert eps_of(_Attn(k_norm=_Norm(variance_epsilon=1e-3))) == 1e-3   # also where only keys have one
    eps_of(_Attn())


@pytest.mark.parametrize("norms", [(_Norm(eps=1e-5), _Norm(eps=1e-5)), (_Norm(variance_epsilon=1e-5), _Norm(eps=1e-5)),
                                   (_Norm(variance_epsilon=1e-5), _Norm(variance_epsilon=1e-6)), (None, _Norm())])
def test_other_norms_are_refused(eps_of, norms):
    with pytest.raises(NotImplementedError, match="variance_epsilon"):
        eps_of(_Attn(*norms))
