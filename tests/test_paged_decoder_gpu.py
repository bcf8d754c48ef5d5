"""PagedDecoder on the GPU where the CPU's stand-in does not reach: ids that are on the device."""
import pytest
import torch

from tread_b200 import BlockStore, Engine
from tread_b200.configs import random_model, random_tokens
from tread_b200.paged import PagedDecoder

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def setup():
    model = random_model("tiny").to("cuda:0")
    eng = Engine(model, BlockStore(1 << 30))
    g = torch.Generator().manual_seed(1)
    prefix, query = random_tokens(30, model.config.vocab_size, g), random_tokens(9, model.config.vocab_size, g)
    return model, eng.prefill(prefix, [], query, ratio=0.0)[1]


@pytest.mark.parametrize("graphs", [False, True])
def test_device_ids_outside_the_vocabulary_are_flagged(setup, graphs):
    model, cache = setup
    V = model.config.vocab_size
    dec = PagedDecoder(model, num_pages=30, page_size=16, max_seqs=4, max_len=100, graphs=graphs)
    for bad, near in ((V, V - 1), (2 ** 40, V - 1), (-1, 0)):
        a, b = dec.admit(cache), dec.admit(cache)
        got = dec.step([a], torch.tensor([bad], device="cuda")).clone()
        with pytest.raises(RuntimeError, match="token"):
            dec.net.check_errors()
        assert torch.equal(got, dec.step([b], [near]))
        dec.net.check_errors()
        dec.release(a), dec.release(b)
    a = dec.admit(cache)
    dec.step([a], torch.tensor([V - 1], device="cuda", dtype=torch.int32))
    dec.net.check_errors()


def _steps(model, cache, graphs):
    dec = PagedDecoder(model, num_pages=30, page_size=16, max_seqs=4, max_len=100, graphs=graphs)
    seq = dec.admit(cache)
    return torch.stack([dec.step([seq], [t])[0].clone() for t in (5, 6, 7)])


def test_a_step_is_captured_on_a_stream_of_the_decoders_device(setup, monkeypatch):
    """torch.cuda.graph without a stream takes one of whichever device captured first."""
    model, cache = setup
    seen, real = [], torch.cuda.graph

    def spy(graph, *args, **kw):
        seen.append((kw.get("stream"), torch.cuda.current_device()))
        return real(graph, *args, **kw)

    monkeypatch.setattr(torch.cuda, "graph", spy)
    got = _steps(model, cache, True)
    assert len(seen) == 1 and seen[0][0] is not None
    assert seen[0][0].device == model.device and seen[0][1] == model.device.index
    assert float((got - _steps(model, cache, False)).abs().max()) < 1e-5


def test_graphs_on_a_device_that_is_not_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    g = torch.Generator().manual_seed(1)
    with torch.cuda.device(1):
        model = random_model("tiny").to("cuda:1")
        cache = Engine(model, BlockStore(1 << 30)).prefill(random_tokens(30, 4096, g), [], random_tokens(9, 4096, g))[1]
        want = _steps(model, cache, False)
    torch.cuda.set_device(0)
    assert float((_steps(model, cache, True) - want).abs().max()) < 1e-5
