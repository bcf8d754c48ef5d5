"""What PagedDecoder refuses before anything is reserved or launched (no GPU: a stand-in for the model's rows)."""
from types import SimpleNamespace

import pytest
import torch

from tread_b200.paged import PagedCache, PagedDecoder


def _decoder(L=2, Hkv=2, D=64, vocab=50):
    dec = PagedDecoder.__new__(PagedDecoder)
    dec.net = SimpleNamespace(L=L, Hkv=Hkv, D=D, device=torch.device("cpu"), embed=torch.zeros(vocab, 8))
    dec.cache = PagedCache(L, Hkv, D, 10, page_size=4, max_seqs=3, max_len=24, dtype=torch.float32, device="cpu")
    dec.graphs = None
    return dec


def _cache(shapes):
    layers = [SimpleNamespace(keys=torch.zeros(k), values=torch.zeros(v)) for k, v in shapes]
    return SimpleNamespace(layers=layers)


def _unchanged(dec):
    return dec.cache.lens == {} and dec.cache.free_pages == 10


@pytest.mark.parametrize("shapes", [
    [((2, 2, 5, 64), (2, 2, 5, 64))] * 2,                                    # two sequences: only one would be taken
    [((1, 2, 5, 64), (1, 2, 5, 64)), ((1, 2, 6, 64), (1, 2, 6, 64))],        # layers of two lengths
    [((1, 2, 5, 64), (1, 2, 4, 64))] * 2,                                    # values of another length
    [((1, 4, 5, 64), (1, 4, 5, 64))] * 2, [((1, 2, 5, 32), (1, 2, 5, 32))] * 2, [((2, 5, 64), (2, 5, 64))] * 2,
])
def test_admit_refuses_other_layers(shapes):
    dec = _decoder()
    with pytest.raises(ValueError, match="admit: layers"):
        dec.admit(_cache(shapes))
    assert _unchanged(dec)


def test_admit_refuses_a_batch_of_one_layer():
    """One layer's [2, Hkv, T, D] is one tensor too: its first sequence must not pass for the whole."""
    dec = _decoder(L=1)
    with pytest.raises(ValueError, match="admit: layers"):
        dec.admit(_cache([((2, 2, 5, 64), (2, 2, 5, 64))]))
    assert _unchanged(dec)


@pytest.mark.parametrize("tokens", [[-1], [50], torch.tensor([50]), torch.tensor([-1], dtype=torch.int32), [1.5],
                                    torch.tensor([1.0]), torch.tensor([[1]]), [[1]], torch.tensor([True]), [1, 2], []])
def test_step_refuses_tokens(tokens):
    """Outside the vocabulary, not whole numbers, not one a sequence."""
    dec = _decoder()
    seq = dec.cache.new(0)
    with pytest.raises(ValueError, match="step: "):
        dec.step([seq], tokens)
    assert dec.cache.lens == {seq: 0} and dec.cache.free_pages == 10


def test_token_ids_of_any_whole_type():
    dec = _decoder()
    for tokens in ([0, 49], torch.tensor([0, 49]), torch.tensor([0, 49], dtype=torch.int16), (0, 49)):
        ids = dec._ids(tokens)
        assert ids.dtype == torch.int64 and ids.tolist() == [0, 49]
