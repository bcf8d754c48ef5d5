"""A greedy decode loop in one graph: the decode step, the adjustment of its logits, the choice of the token, the
history's and the positions' update, replayed token by token against the same loop step by step."""
import pytest
import torch

from tread_b200 import BlockStore, Engine, kernels
from tread_b200.configs import random_model, random_tokens
from tread_b200.paged import PagedDecoder

pytestmark = pytest.mark.gpu

PENALTIES = dict(repetition=1.4, frequency=0.3, presence=0.2)


@torch.inference_mode()
def test_replays_of_one_graph_are_the_loop():
    model = random_model("tiny").to("cuda:0")
    V = model.config.vocab_size
    eng = Engine(model, BlockStore(1 << 30))
    g = torch.Generator().manual_seed(3)
    prompts = [random_tokens(n, V, g) for n in (13, 30)]
    caches = [eng.prefill(p[:5], [], p[5:], ratio=0.0)[1] for p in prompts]
    steps, room = 20, 64
    history = torch.full((2, room), -1, dtype=torch.int64, device="cuda")
    for i, p in enumerate(prompts):
        history[i, :len(p)] = p.cuda()
    start = torch.tensor([7, 11], device="cuda")

    def adjusted(logits, history, lens, prompt):
        return kernels.adjust_logits(logits, tokens=history, lens=lens, prompt_lens=prompt, **PENALTIES)

    dec = PagedDecoder(model, num_pages=40, page_size=16, max_seqs=2, max_len=200)
    seqs = [dec.admit(c, room=steps) for c in caches]
    prompt = torch.tensor([len(p) for p in prompts], device="cuda")
    want, hist, lens, tokens = [], history.clone(), prompt.clone(), start.clone()
    for _ in range(steps):
        hist[torch.arange(2), lens] = tokens
        lens += 1
        tokens = adjusted(dec.step(seqs, tokens), hist, lens, prompt).argmax(-1)
        want.append(tokens.tolist())

    dec = PagedDecoder(model, num_pages=40, page_size=16, max_seqs=2, max_len=200)
    seqs = [dec.admit(c, room=steps) for c in caches]
    table = dec.cache.table[torch.tensor(seqs, device="cuda")]
    hist, lens, tokens, pos = history.clone(), prompt.clone(), start.clone(), torch.full((2,), -1, device="cuda")

    def turn():
        hist.scatter_(1, lens[:, None], tokens[:, None])
        lens.add_(1)
        logits = dec._forward(tokens, pos, table)
        tokens.copy_(adjusted(logits, hist, lens, prompt).argmax(-1))
        pos.add_(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        turn()  # position -1: nothing is appended
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        turn()
    hist.copy_(history), lens.copy_(prompt), tokens.copy_(start)
    pos.copy_(torch.tensor([dec.cache.lens[s] for s in seqs]))
    got = []
    for _ in range(steps):
        graph.replay()
        got.append(tokens.tolist())
    dec.net.check_errors()
    assert got == want and len({t for pair in got for t in pair}) > 2
