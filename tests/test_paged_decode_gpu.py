"""Decode steps over the paged cache, the three operators together as a decode step uses them: against the HF
model's own decoding, in batches of sequences of different lengths, captured, behind the server, and with
adjusted logits against an elementary restatement."""
import json

import numpy as np
import pytest
import torch
from fastapi.testclient import TestClient

from conftest import golden
from golden.stub_tokenizer import SERVER_REQUESTS, StubTokenizer
from paged_oracle import adjust64
from tread_b200 import BlockStore, Engine, kernels
from tread_b200.configs import random_model, random_tokens
from tread_b200.paged import OutOfPages, PagedDecoder
from tread_b200.server import build_app

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def setup():
    model = random_model("tiny").to("cuda:0")
    return model, Engine(model, BlockStore(1 << 30))


def _request(eng, seed, lens=(9, 40, 33, 7)):
    g = torch.Generator().manual_seed(seed)
    V = eng.model.config.vocab_size
    prefix, *docs, query = [random_tokens(n, V, g) for n in lens]
    return eng.prefill(prefix, docs, query, ratio=0.2)[:2]


def _hf_steps(model, cache, tokens):
    """Logits after each of `tokens`, by the HF model over the request's DynamicCache."""
    out = []
    with torch.inference_mode():
        for t in tokens:
            o = model(torch.tensor([[t]], device="cuda:0"), past_key_values=cache, use_cache=True, logits_to_keep=1)
            cache = o.past_key_values
            out.append(o.logits[0, -1])
    return torch.stack(out)


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("page_size", [1, 16, 64, 200])
def test_steps_match_the_hf_model(setup, graphs, page_size):
    """fp32: the same next tokens and logits within the two paths' fp32 differences (both sum about 1e3
    products of size 1 per element through 4 layers: 1e-4 is some hundred roundings of 2^-24 of logits
    of size below 8)."""
    model, eng = setup
    dec = PagedDecoder(model, num_pages=2000 // page_size, page_size=page_size, max_seqs=4, max_len=500, graphs=graphs)
    logits, cache = _request(eng, 1)
    seq = dec.admit(cache)
    g = torch.Generator().manual_seed(2)
    tokens = random_tokens(20, model.config.vocab_size, g).tolist()
    want = _hf_steps(model, cache, tokens)
    got = torch.stack([dec.step([seq], [t])[0].clone() for t in tokens])
    assert float((got - want).abs().max()) < 1e-4
    assert torch.equal(got.argmax(-1), want.argmax(-1))
    dec.net.check_errors()
    dec.release(seq)
    assert dec.cache.free_pages == 2000 // page_size


@pytest.mark.parametrize("graphs", [False, True])
def test_a_batch_of_lengths_equals_each_alone(setup, graphs):
    """Sequences of different lengths that join and leave: each one's logits are what it has alone (up to
    the projections' row counts: fp32, as above)."""
    model, eng = setup
    dec = PagedDecoder(model, num_pages=300, page_size=16, max_seqs=8, max_len=600, graphs=graphs)
    alone = PagedDecoder(model, num_pages=300, page_size=64, max_seqs=8, max_len=600)
    lengths = [(9, 40, 33, 7), (5, 3), (60, 200, 100, 30), (16, 16, 16)]
    requests = [_request(eng, 10 + i, lens)[1] for i, lens in enumerate(lengths)]
    seqs, solo = [dec.admit(c) for c in requests], [alone.admit(c) for c in requests]
    g = torch.Generator().manual_seed(3)
    for members in ([0, 1, 2, 3], [0, 1, 2, 3], [2, 0], [1], [3, 1, 0], [0, 1, 2, 3]):
        tokens = random_tokens(len(members), model.config.vocab_size, g).tolist()
        got = dec.step([seqs[i] for i in members], torch.tensor(tokens, device="cuda:0"))
        for row, i in enumerate(members):
            want = alone.step([solo[i]], [tokens[row]])[0]
            assert float((got[row] - want).abs().max()) < 1e-4
    dec.net.check_errors()


def test_bf16_decoding_stays_near_fp32():
    """bf16 model of the 7B heads (2 layers): paged steps against a full prefill of the same tokens."""
    from tread_b200.engine import prefill_full

    model = random_model("qwen2.5-7b", dtype=torch.bfloat16, device="cuda:0", layers=2, init_on_device=True, vocab=4096)
    eng = Engine(model, BlockStore(4 << 30))
    g = torch.Generator().manual_seed(4)
    prefix, query = random_tokens(300, 4096, g), random_tokens(50, 4096, g)
    more = random_tokens(5, 4096, g)
    dec = PagedDecoder(model, num_pages=50, page_size=64, max_seqs=2, max_len=1000, graphs=True)
    seq = dec.admit(eng.prefill(prefix, [], query)[1], room=5)
    for i, t in enumerate(more.tolist()):
        got = torch.log_softmax(dec.step([seq], [t])[0].float(), -1)
        full = prefill_full(model, prefix, [], torch.cat([query, more[:i + 1]]))[0]
        kl = float((got.exp() * (got - torch.log_softmax(full.float(), -1))).sum())
        assert abs(kl) < 1e-3
    dec.net.check_errors()


def test_caches_that_are_not_one_tensor(setup):
    """A DynamicCache whose layers the HF model has appended to."""
    model, eng = setup
    _, cache = _request(eng, 5)
    want = _hf_steps(model, cache, [11, 12, 13])  # appends to `cache`: its layers are tensors of their own now
    dec = PagedDecoder(model, num_pages=20, max_seqs=2, max_len=600)
    seq = dec.admit(cache)
    assert dec.cache.lens[seq] == 9 + 40 + 33 + 7 + 3
    again = PagedDecoder(model, num_pages=20, max_seqs=2, max_len=600)
    first = again.admit(_request(eng, 5)[1])
    got = [again.step([first], [t])[0] for t in (11, 12, 13)]
    assert float((got[-1] - want[-1]).abs().max()) < 1e-4
    a, b = dec.step([seq], [14]), again.step([first], [14])
    assert float((a - b).abs().max()) < 1e-4


def test_step_refusals_change_nothing(setup):
    model, eng = setup
    dec = PagedDecoder(model, num_pages=7, page_size=16, max_seqs=3, max_len=96)
    a = dec.admit(_request(eng, 6, (20, 43))[1])  # 63 tokens, 4 pages
    b = dec.admit(_request(eng, 7, (20, 28))[1])  # 48 tokens, 3 pages
    with pytest.raises(OutOfPages):
        dec.admit(_request(eng, 8, (3, 3))[1])
    dec.step([a], [5])  # the 64th token: its page is there
    for bad in (([a], [1]), ([b], [1]), ([a, b], [1, 2])):
        with pytest.raises(OutOfPages):
            dec.step(*bad)
    for bad in (([a, a], [1, 2]), ([a], [1, 2]), ([], []), ([2], [1])):
        with pytest.raises(ValueError):
            dec.step(*bad)
    assert dec.cache.lens == {a: 64, b: 48} and dec.cache.free_pages == 0
    dec.release(b)
    assert dec.step([a], [5]).shape == (1, model.config.vocab_size)
    dec.net.check_errors()


def test_append_attend_and_adjust_captured_together(setup):
    """A greedy loop in one graph: step, adjust, argmax, history: against the same loop run eagerly and the
    logits' definition."""
    model, eng = setup
    _, cache = _request(eng, 9)
    V = model.config.vocab_size

    def loop(dec, seq, logits, steps, history, n):
        out = []
        for _ in range(steps):
            adj = kernels.adjust_logits(logits[None], tokens=history[:, :n], repetition=1.4, frequency=0.3, presence=0.2)
            want, size = adjust64(logits[None], tokens=history[:, :n], repetition=1.4, frequency=0.3, presence=0.2)
            assert bool(((adj.double() - want).abs() <= 4 * 2.0 ** -24 * size + 1e-40).all())
            nxt = int(adj.argmax())
            out.append(nxt)
            history[0, n] = nxt
            n += 1
            logits = dec.step([seq], [nxt])[0]
        return out

    answers = []
    for graphs in (False, True):
        dec = PagedDecoder(model, num_pages=40, page_size=16, max_seqs=2, max_len=300, graphs=graphs)
        seq = dec.admit(cache)
        history = torch.zeros(1, 64, dtype=torch.int64, device="cuda:0")
        history[0, :4] = torch.tensor([5, 6, 7, 5])
        first = torch.randn(V, device="cuda:0", generator=torch.Generator("cuda:0").manual_seed(1))
        answers.append(loop(dec, seq, first, 12, history, 4))
    assert answers[0] == answers[1] and len(set(answers[0])) > 1


# ---- behind the server --------------------------------------------------------------------------


def _client(g, decoder=True, **kw):
    model = random_model("tiny").to("cuda:0")
    V = model.config.vocab_size
    eng = Engine(model, BlockStore(int(g["gpu_budget"]), cpu_budget_bytes=int(g["cpu_budget"])))
    dec = PagedDecoder(model, num_pages=40, page_size=16, max_len=512, max_seqs=2) if decoder else None
    return TestClient(build_app(model, StubTokenizer(V), eng, eos_ids={V - 1}, max_context=512, decoder=dec, **kw)), dec


def test_server_with_a_paged_decoder_answers_as_the_reference():
    g = golden("server.npz")
    want = json.loads(str(g["responses"]))
    client, dec = _client(g)
    for (prefix, docs, suffix, tenant, max_tokens, ratio, policy), ref in zip(SERVER_REQUESTS, want):
        r = client.post("/v1/completions", json=dict(prefix=prefix, documents=docs, suffix=suffix, tenant=tenant,
                                                     max_tokens=max_tokens, recompute_ratio=ratio, policy=policy))
        assert r.status_code == 200, r.text
        body = r.json()
        for k in ("ttft_ms", "total_ms"):
            body["tread"].pop(k)
        assert body == ref
        assert dec.cache.lens == {} and dec.cache.free_pages == 40


@pytest.mark.parametrize("decoder", [False, True])
def test_server_adjusts_logits(decoder):
    g = golden("server.npz")
    client, dec = _client(g, decoder)
    base = dict(prefix="You are a careful assistant. ", documents=["alpha doc about rivers and lakes"],
                suffix="Q: which?", max_tokens=8, recompute_ratio=0.0)
    ask = lambda **kw: client.post("/v1/completions", json={**base, **kw})  # noqa: E731
    plain = ask().json()["text"].split()
    assert ask(repetition_penalty=1.0, logit_bias={}, allowed_token_ids=None).json()["text"].split() == plain
    # only these tokens, then one of them banned by its bias
    only = ask(allowed_token_ids=[3, 17, 4000]).json()["text"].split()
    assert set(only) <= {"3", "17", "4000"} and len(only) == 8
    fewer = ask(allowed_token_ids=[3, 17, 4000], logit_bias={only[0]: -10000.0}).json()["text"].split()
    assert only[0] not in fewer and len(fewer) == 8
    # a presence penalty above every difference: no token twice
    once = ask(presence_penalty=100.0, max_tokens=16).json()["text"].split()
    assert len(set(once)) == len(once) == 16
    assert ask(repetition_penalty=1.3, frequency_penalty=0.4).status_code == 200
    for bad in (dict(repetition_penalty=0.0), dict(repetition_penalty=1e-50), dict(logit_bias={"4096": 1.0}), dict(allowed_token_ids=[-1]),
                dict(allowed_token_ids=[]), dict(logit_bias={"x": 1.0}), dict(logit_bias={"1": 1e9})):
        assert ask(**bad).status_code == 422, bad
    if dec is not None:
        assert dec.cache.lens == {}


def test_server_without_a_free_page_answers_503():
    """The decoder's pages are held by another user of it: the request fails, nothing leaks, and the next one
    works."""
    client, dec = _client(golden("server.npz"))
    body = dict(prefix="You are a careful assistant. ", documents=["alpha doc"], suffix="Q: which?", max_tokens=4)
    held = dec.cache.new(500)
    more = dec.cache.new(100)
    assert client.post("/v1/completions", json=body).status_code == 503
    assert sorted(dec.cache.lens) == sorted([held, more])
    dec.release(held)
    dec.release(more)
    assert client.post("/v1/completions", json=body).status_code == 200
    assert dec.cache.lens == {}


def test_server_refuses_a_decoder_that_is_too_small():
    model = random_model("tiny").to("cuda:0")
    dec = PagedDecoder(model, num_pages=4, page_size=16, max_len=512)
    with pytest.raises(ValueError, match="64 tokens"):
        build_app(model, StubTokenizer(4096), Engine(model, BlockStore(1 << 20)), eos_ids={1}, max_context=512, decoder=dec)
