"""Bookkeeping of the paged cache (no GPU): pages and sequences handed out, grown, refused and given back."""
import random

import pytest
import torch

from tread_b200.paged import OutOfPages, PagedCache, _flat_layers


def _cache(**over):
    kw = dict(num_pages=10, page_size=4, max_seqs=3, max_len=24, dtype=torch.float32, device="cpu")
    kw.update(over)
    return PagedCache(2, 2, 8, **kw)


def _consistent(pc, num_pages):
    held = [p for pages in pc._pages.values() for p in pages]
    assert sorted(held + pc._free) == list(range(num_pages))
    for s in range(pc.max_seqs):
        pages = pc._pages.get(s, [])
        assert pc.table[s].tolist() == pages + [-1] * (pc.table.shape[1] - len(pages))


def test_grow_release_and_reuse():
    pc = _cache()
    a, b = pc.new(5), pc.new()
    assert len(pc._pages[a]) == 2 and pc._pages[b] == [] and pc.free_pages == 8
    pc.reserve(b, 1)
    pc.reserve(b, 4)
    assert len(pc._pages[b]) == 1
    pc.reserve(b, 13)
    _consistent(pc, 10)
    pc.release(a)
    _consistent(pc, 10)
    assert pc.new(24) == a and pc.free_pages == 0
    _consistent(pc, 10)
    assert pc.layer(1)[0].shape == (10, 2, 4, 8)


def test_refusals_change_nothing():
    pc = _cache()
    a = pc.new(20)
    b = pc.new(20)
    for bad, error in ((lambda: pc.new(1), OutOfPages), (lambda: pc.reserve(a, 21), OutOfPages),
                       (lambda: pc.reserve(a, 25), ValueError), (lambda: pc.release(2), ValueError)):
        with pytest.raises(error):
            bad()
        _consistent(pc, 10)
        assert sorted(pc.lens) == sorted([a, b]) and len(pc._free_seqs) == 1
    pc.new(0)
    with pytest.raises(OutOfPages, match="sequences"):
        pc.new(0)
    for bad in (dict(num_pages=0), dict(page_size=0), dict(max_seqs=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            _cache(**bad)


def test_random_walk_stays_consistent():
    rng = random.Random(0)
    pc = _cache(num_pages=20, max_seqs=6, page_size=3, max_len=30)
    for _ in range(500):
        try:
            live = sorted(pc.lens)
            move = rng.random()
            if move < 0.4 or not live:
                pc.new(rng.randrange(0, 32))
            elif move < 0.8:
                pc.reserve(rng.choice(live), rng.randrange(0, 32))
            else:
                pc.release(rng.choice(live))
        except (OutOfPages, ValueError):
            pass
        _consistent(pc, 20)


def test_layers_of_one_tensor_are_seen_as_one():
    K = torch.arange(2 * 3 * 5 * 4.0).view(2, 1, 3, 5, 4)
    flat = _flat_layers(list(K.unbind(0)))
    assert torch.equal(flat, K.view(6, 5, 4).transpose(0, 1)) and flat.data_ptr() == K.data_ptr()
    assert _flat_layers([K[0], K[1].clone()]) is None
    assert _flat_layers([K[1], K[0]]) is None
    assert _flat_layers([K[0, ..., :4, :], K[1, ..., :4, :]]) is None
    assert torch.equal(_flat_layers([K[0]]), K[0, 0].transpose(0, 1))
