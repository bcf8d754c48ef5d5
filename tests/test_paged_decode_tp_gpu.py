"""PagedDecoder over KV-head tensor-parallel rows: every rank pages its own heads, and the steps' all-reduces join
them. Two ranks on one GPU: a host thread each on one stream, the all-reduce restated as a sum between host
barriers (no kernel waits for another)."""
import threading
from types import SimpleNamespace

import pytest
import torch

from tread_b200 import BlockStore, Engine, tp
from tread_b200.configs import random_model, random_tokens
from tread_b200.paged import PagedDecoder

pytestmark = pytest.mark.gpu

STEPS = [[5, 9], [700, 3], [12, 4000]]


@pytest.fixture(scope="module")
def setup():
    model = random_model("tiny").to("cuda:0")
    eng = Engine(model, BlockStore(1 << 30))
    g = torch.Generator().manual_seed(1)
    ids = lambda n: random_tokens(n, model.config.vocab_size, g)  # noqa: E731
    caches = [eng.prefill(ids(20), [ids(31)], ids(n), ratio=0.0)[1] for n in (9, 40)]
    dec = PagedDecoder(model, num_pages=60, page_size=16, max_seqs=4, max_len=200)
    seqs = [dec.admit(c) for c in caches]
    want = torch.stack([dec.step(seqs, t).clone() for t in STEPS])
    return model, caches, want


def _heads(cache, h0, h1):
    return SimpleNamespace(layers=[SimpleNamespace(keys=l.keys[:, h0:h1], values=l.values[:, h0:h1])
                                   for l in cache.layers])


def test_one_rank_is_the_model(setup):
    model, caches, want = setup
    dec = PagedDecoder(tp.TPQwen2Rows.from_model(model), num_pages=60, page_size=16, max_seqs=4, max_len=200)
    seqs = [dec.admit(c) for c in caches]
    got = torch.stack([dec.step(seqs, t).clone() for t in STEPS])
    assert float((got - want).abs().max()) < 1e-4
    dec.net.check_errors()


def test_two_ranks_are_the_model(setup, monkeypatch):
    """fp32, both paths' sums as in the tests of the steps against the HF model: 1e-4."""
    model, caches, want = setup
    world, me = 2, threading.local()
    meet, parts = threading.Barrier(world, timeout=60), [None] * world

    def all_reduce(t, group=None, op=None):
        parts[me.rank] = t.clone()
        meet.wait()
        t.copy_(parts[0] + parts[1])  # one stream: both clones are in front of it
        meet.wait()

    monkeypatch.setattr(tp.dist, "is_initialized", lambda: True)
    monkeypatch.setattr(tp.dist, "get_world_size", lambda group=None: world)
    monkeypatch.setattr(tp.dist, "get_rank", lambda group=None: me.rank)
    monkeypatch.setattr(tp.dist, "all_reduce", all_reduce)
    got, errors = [None] * world, []

    def rank(r):
        me.rank = r
        try:
            net = tp.TPQwen2Rows.from_model(model)
            assert net.Hkv == model.config.num_key_value_heads // world
            with pytest.raises(ValueError, match="tensor-parallel"):
                PagedDecoder(net, num_pages=60, graphs=True)
            dec = PagedDecoder(net, num_pages=60, page_size=16, max_seqs=4, max_len=200)
            seqs = [dec.admit(_heads(c, *net.kv_heads)) for c in caches]
            got[r] = torch.stack([dec.step(seqs, t).clone() for t in STEPS])
        except BaseException as e:
            errors.append(e)
            meet.abort()

    threads = [threading.Thread(target=rank, args=(r,)) for r in range(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert torch.equal(got[0], got[1])
    assert float((got[0] - want).abs().max()) < 1e-4
