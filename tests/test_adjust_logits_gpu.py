"""Adjusting logits (tread_adjust_logits) against the definition in 64 bits."""
import pytest
import torch

from paged_oracle import adjust64
from tread_b200 import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _check(got, logits, **kw):
    """fp32: at most 4 roundings, each half a step (2^-24) of a term or partial sum, whose sizes `size`
    adds up; then half a step of the output's type."""
    want, size = adjust64(logits, **kw)
    f = torch.finfo(got.dtype)
    over = want.float().to(got.dtype).isinf()  # past the type's range (3.4e38 x 1.5 in fp32): infinite
    want = torch.where(over, want.sign() * torch.inf, want)
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    off = (got.double() - want).abs()[fine]
    bound = (4 * 2.0 ** -24 * size + 1.01 * f.eps / 2 * want.abs())[fine] + f.smallest_normal * f.eps / 2
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.3g} of the bound"


def _case(B, V, H, dtype, seed, biases=9):
    g = _gen(seed)
    logits = (4 * torch.randn(B, V, device=DEV, generator=g)).to(dtype)
    few = max(1, min(V, 40))
    tokens = torch.randint(0, few, (B, H), device=DEV, generator=g) * max(1, V // few)
    tokens = tokens.clamp(max=V - 1)
    lens = torch.randint(0, H + 1, (B,), device=DEV, generator=g)
    rows = lambda lo, hi: lo + (hi - lo) * torch.rand(B, device=DEV, generator=g)  # noqa: E731
    return logits, dict(
        tokens=tokens, lens=lens, prompt_lens=(lens.double() * rows(0, 1)).long(), repetition=rows(0.7, 2.0),
        presence=rows(-0.5, 1.0), frequency=rows(-0.2, 0.5),
        bias_ids=torch.randint(0, V, (B, biases), device=DEV, generator=g),
        bias=3 * torch.randn(B, biases, device=DEV, generator=g),
        allowed=torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), device=DEV, generator=g).to(torch.int32))


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("out", [FP, BF, HF])
@pytest.mark.parametrize("B,V,H", [(1, 1, 1), (2, 31, 5), (3, 32, 50), (2, 33, 9), (5, 1001, 300), (2, 20000, 40)])
def test_everything_together(dtype, out, B, V, H):
    logits, kw = _case(B, V, H, dtype, B + V + H)
    _check(kernels.adjust_logits(logits, out=torch.empty(B, V, dtype=out, device=DEV), **kw), logits, **kw)


@pytest.mark.parametrize("keep", [(), ("tokens", "lens", "prompt_lens", "repetition"), ("tokens", "presence"),
                                  ("tokens", "lens", "frequency"), ("bias_ids", "bias"), ("allowed",),
                                  ("tokens", "prompt_lens", "presence", "frequency", "allowed")])
def test_each_part_alone(keep):
    logits, kw = _case(3, 5000, 200, BF, 5)
    kw = {k: v for k, v in kw.items() if k in keep}
    got = kernels.adjust_logits(logits, **kw)
    _check(got, logits, **kw)
    if not keep:
        assert torch.equal(got, logits.float())


@pytest.mark.parametrize("V", [151935, 152064, 151936])
def test_whole_vocabularies(V):
    logits, kw = _case(3, V, 2000, BF, V)
    _check(kernels.adjust_logits(logits, **kw), logits, **kw)


def test_neutral_penalties_change_nothing():
    logits, kw = _case(2, 3000, 100, FP, 6)
    got = kernels.adjust_logits(logits, tokens=kw["tokens"], lens=kw["lens"])
    assert torch.equal(got, logits)


def test_numbers_and_shared_rows():
    """One penalty, one bias list and one mask for every row equal the same ones given per row."""
    B, V = 4, 777
    logits, kw = _case(B, V, 60, BF, 7)
    one = dict(repetition=1.3, presence=0.4, frequency=0.2, bias_ids=kw["bias_ids"][0], bias=kw["bias"][0],
               allowed=kw["allowed"][0])
    per_row = {k: torch.full((B,), v, device=DEV) if isinstance(v, float) else v.expand(B, -1).contiguous()
               for k, v in one.items()}
    base = dict(tokens=kw["tokens"], lens=kw["lens"], prompt_lens=kw["prompt_lens"])
    a, b = kernels.adjust_logits(logits, **base, **one), kernels.adjust_logits(logits, **base, **per_row)
    assert torch.equal(a, b)
    _check(b, logits, **base, **per_row)


def test_one_history_and_one_row_of_logits_for_all():
    logits, kw = _case(4, 777, 60, BF, 16)
    kw["tokens"], kw["lens"] = kw["tokens"][:1].expand(4, -1), kw["lens"][:1].repeat(4)
    logits = logits[:1].expand(4, -1)
    _check(kernels.adjust_logits(logits, **kw), logits, **kw)


@pytest.mark.parametrize("rep", [1e-39, 1e-30, 1e30, 3e38])
def test_repetition_far_from_one(rep):
    """Reciprocals that overflow, lose digits or vanish."""
    x = torch.tensor([[1e-3, -1e-3, 2e-39, -2e-39, 3.0, -3.0, 1e30, -1e30]], device=DEV)
    kw = dict(tokens=torch.arange(8, device=DEV)[None], repetition=rep)
    _check(kernels.adjust_logits(x, **kw), x, **kw)


def test_padding_ids_and_lengths_out_of_range():
    logits, kw = _case(3, 500, 40, BF, 8)
    kw["tokens"][:, ::3] = -1
    kw["tokens"][:, 1::5] = 500
    kw["tokens"][0, 2], kw["tokens"][0, 4] = 2 ** 40, -2 ** 40
    kw["bias_ids"][:, ::2] = -1
    kw["bias_ids"][1, 1], kw["bias_ids"][1, 3] = 500, 2 ** 40 + 3
    kw["lens"] = torch.tensor([40, 2 ** 40, -5], device=DEV)
    kw["prompt_lens"] = torch.tensor([-3, 20, 2 ** 40], device=DEV)
    _check(kernels.adjust_logits(logits, **kw), logits, **kw)


def test_the_same_biased_token_twice():
    """Biases of one token add up in their order, every time alike."""
    logits, _ = _case(2, 300, 4, FP, 9)
    g = _gen(10)
    ids = torch.randint(0, 5, (2, 64), device=DEV, generator=g) * 59
    bias = torch.randn(2, 64, device=DEV, generator=g)
    got = kernels.adjust_logits(logits, bias_ids=ids, bias=bias)
    _check(got, logits, bias_ids=ids, bias=bias)
    for _ in range(5):
        assert torch.equal(kernels.adjust_logits(logits, bias_ids=ids, bias=bias), got)


def test_a_grammar_that_allows_nothing_and_special_logits():
    V = 100
    logits = torch.randn(3, V, device=DEV, generator=_gen(11))
    logits[0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0])
    logits[1, :4] = torch.tensor([torch.finfo(FP).min, torch.finfo(FP).max, -0.0, 1e-40])
    tokens = torch.arange(4, device=DEV).repeat(3, 1)
    kw = dict(tokens=tokens, repetition=1.5, presence=0.5)
    _check(kernels.adjust_logits(logits, **kw), logits, **kw)
    allowed = torch.full((3, 4), -1, dtype=torch.int32, device=DEV)
    allowed[1] = 0
    got = kernels.adjust_logits(logits, allowed=allowed)
    assert bool((got[1] == float("-inf")).all()) and torch.equal(got[2], logits[2])
    assert bool(got[0, 2].isnan())  # allowed: a NaN stays one


def test_in_place_strided_and_unaligned():
    for dtype in (BF, FP):
        logits, kw = _case(3, 1000, 50, dtype, 12)
        want = kernels.adjust_logits(logits, out=torch.empty_like(logits), **kw)
        wide = torch.full((3, 1103), 7, dtype=dtype, device=DEV)
        view = wide[:, 1:1001]
        view.copy_(logits)
        got = kernels.adjust_logits(view, out=view, **kw)
        assert torch.equal(got, want)
        assert bool((wide[:, 0] == 7).all()) and bool((wide[:, 1001:] == 7).all())
        part = {**kw, "tokens": torch.cat([kw["tokens"][:, :1], kw["tokens"]], 1)[:, 1:]}
        assert torch.equal(kernels.adjust_logits(logits, out=torch.empty_like(logits), **part), want)


def test_long_histories():
    B, V, H = 2, 4000, 40000
    logits, kw = _case(B, V, H, BF, 13)
    kw["lens"][:] = H
    kw["tokens"][1] = 17  # one token, forty thousand times
    kw["prompt_lens"] = torch.tensor([H - 1, 5], device=DEV)
    _check(kernels.adjust_logits(logits, **kw), logits, **kw)


def test_many_biases_and_every_row_offset():
    """More biases than threads, rows that start at every offset from a 16-byte boundary, vectors of the
    mask that straddle its words, vocabularies of one vector and less."""
    for V in (1003, 2051, 40, 9, 3):
        logits, kw = _case(9, V, 64, BF, V, biases=700)
        _check(kernels.adjust_logits(logits, **kw), logits, **kw)
        f, kf = _case(5, V, 64, FP, V + 1, biases=300)
        _check(kernels.adjust_logits(f, out=torch.empty(5, V, dtype=HF, device=DEV), **kf), f, **kf)


@pytest.mark.parametrize("H", [4000, 5500, 6200, 6600, 7400, 16383, 16384])
def test_shared_memory_of_every_size(H):
    """Histories whose lists bring a CTA's shared memory to either side of 48 KB, and both widths of counters."""
    logits, kw = _case(64, 152064, H, BF, H)
    few = slice(0, 2)
    got = kernels.adjust_logits(logits, **kw)
    _check(got[few], logits[few], **{k: v[few] for k, v in kw.items()})


@pytest.mark.parametrize("H", [9000, 20000])
@pytest.mark.parametrize("where", ["new", "in place"])
def test_more_changed_tokens_than_a_slice_has_room_for(H, where):
    """Histories of thousands of different tokens side by side, with biases among them."""
    B, V = 64, 152064
    logits, kw = _case(B, V, H, BF, H, biases=300)
    g = _gen(H + 1)
    kw["tokens"] = torch.randint(0, 16000, (B, H), device=DEV, generator=g)
    kw["bias_ids"] = torch.randint(0, 17000, (B, 300), device=DEV, generator=g)
    kw["lens"][:3] = H
    kw["prompt_lens"][0] = H
    kw["allowed"][1] = -1
    few = slice(0, 3)
    before = logits[few].clone()
    got = kernels.adjust_logits(logits, out=logits if where == "in place" else None, **kw)
    _check(got[few], before, **{k: v[few] for k, v in kw.items()})


def test_graph_replay_and_streams():
    logits, kw = _case(4, 20000, 100, BF, 14)
    want = kernels.adjust_logits(logits, **kw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kernels.adjust_logits(logits, **kw)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        g.replay()
        other = kernels.adjust_logits(logits, stream=s, **kw)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(other, want)


def test_refuses_bad_tensors():
    logits, kw = _case(2, 100, 10, BF, 15)
    for bad in (dict(tokens=kw["tokens"].int()), dict(tokens=kw["tokens"][:1]), dict(lens=kw["lens"].cpu()),
                dict(lens=kw["lens"][:1]), dict(repetition=kw["repetition"].double()), dict(repetition=0.0),
                dict(repetition=-1.0), dict(repetition=float("nan")), dict(bias=None), dict(bias=kw["bias"][:, :3]),
                dict(allowed=kw["allowed"].long()), dict(allowed=kw["allowed"][:, :3]), dict(tokens=None),
                dict(presence=kw["presence"].cpu()), dict(out=torch.empty(2, 99, device=DEV)),
                dict(out=torch.empty(2, 100))):
        with pytest.raises(ValueError):
            kernels.adjust_logits(logits, **{**kw, **bad})
    with pytest.raises(ValueError):
        kernels.adjust_logits(logits.cpu())
    with pytest.raises(TypeError):
        kernels.adjust_logits(logits, out=torch.empty(2, 100, dtype=torch.float64, device=DEV))
