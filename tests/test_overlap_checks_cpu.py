"""disjoint(): an output that shares an element with an input is refused, slices of one fused buffer are not."""

import itertools

import pytest
import torch


def _places(x):
    """The element offsets of x in its storage."""
    index = torch.zeros((), dtype=torch.long) + x.storage_offset()
    for n, s in zip(x.shape, x.stride()):
        index = index[..., None] + torch.arange(n) * s
    return set(index.flatten().tolist())


def test_token_major_batches_shifted_by_one_sequence():
    from turbopolar_b200._checks import disjoint
    x = torch.zeros(5, 3, 4, 128)      # (T, B + 1, H, 128)
    a, b = x[:, :2].transpose(0, 1), x[:, 1:].transpose(0, 1)
    assert not disjoint(a, b) and not disjoint(b, a)


def test_slices_of_a_fused_projection_are_accepted():
    from turbopolar_b200._checks import disjoint
    x = torch.zeros(2, 5, 9, 128)      # (B, T, H_q + 2 H_kv + a pad, 128)
    q, k, v = x[:, :, :4], x[:, :, 4:6], x[:, :, 6:8]
    for a, b in itertools.permutations((q, k, v), 2):
        assert disjoint(a, b)
    t = x.transpose(0, 1)              # token rows first
    assert disjoint(t[:, :, :4], t[:, :, 4:8]) and not disjoint(t[:, :, :4], t[:, :, 3:7])
    assert disjoint(x[0, :, :4], x[0, :, 4:6]) and disjoint(x[0, :1, :4], x[0, :1, 4:8])
    assert not disjoint(x[:1, :, :4], x[:1, :, 3:7])


@pytest.mark.parametrize("seed", range(40))
def test_never_true_for_shared_elements(seed):
    from turbopolar_b200._checks import disjoint
    g = torch.Generator().manual_seed(seed)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    storage = torch.zeros(1 << 14)
    for _ in range(60):
        shape = (pick(1, 3), pick(1, 4), pick(1, 3), 128)
        strides = (pick(0, 12) * 128, pick(0, 12) * 128, pick(1, 4) * 128, 1)
        views = [storage.as_strided(shape, strides, pick(0, 24) * pick(64, 128)) for _ in range(2)]
        if _places(views[0]) & _places(views[1]):
            assert not disjoint(*views), (shape, strides, [v.storage_offset() for v in views])
