"""Attention of one new token over a paged cache (tread_paged_attn) against the definition in 64 bits."""
import pytest
import torch

from paged_oracle import attend64, attend_bound, make_table
from tread_b200 import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
NAN = float("nan")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _case(lens, Hq, Hkv, D, page, dtype, seed, width=None, stretch=1.0):
    """Pools whose slots behind every sequence's length, and whose free pages, hold NaN."""
    g = _gen(seed)
    table, pool = make_table(lens, page, g, width=width)
    q = (stretch * torch.randn(len(lens), Hq, D, device=DEV, generator=g)).to(dtype)
    kp, vp = (torch.full((pool, Hkv, page, D), NAN, dtype=dtype, device=DEV) for _ in range(2))
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            m = min(page, n - i * page)
            for p in (kp, vp):
                p[table[b, i].long(), :, :m] = torch.randn(Hkv, m, D, device=DEV, generator=g).to(dtype)
    return q, kp, vp, table, torch.tensor(lens, device=DEV)


def _check(got, q, kp, vp, table, lens, scale=None):
    out, size, reach = attend64(q, kp, vp, table, lens, scale)
    off = (got.double() - out).abs()
    bound = attend_bound(out, size, reach, lens, q.shape[2], q.dtype)
    assert bool((off <= bound).all()), f"off by {float((off / bound).nan_to_num(9e9).max()):.3g} of the bound"


HEADS = [(28, 4, 128), (40, 8, 128), (14, 2, 64), (4, 4, 64), (16, 1, 128), (9, 3, 256), (32, 2, 256)]
EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 250, 500, 0]


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("page", [16, 64])
def test_lengths_around_every_edge(dtype, Hq, Hkv, D, page):
    c = _case(EDGES, Hq, Hkv, D, page, dtype, Hq + D)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = kernels.paged_attn(*c, err=err)
    _check(got, *c)
    assert int(got[-1].count_nonzero()) == 0 and int(err) == 0


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_any_group(dtype, G, D):
    c = _case([1, 0, 47, 300, 2111], 2 * G, 2, D, 16, dtype, G + D)
    _check(kernels.paged_attn(*c), *c)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("page", [1, 3, 8, 20, 48, 128, 300])
def test_any_page_size(dtype, page):
    c = _case([1, 7, 59, 100, 333], 14, 2, 64, page, dtype, page)
    _check(kernels.paged_attn(*c), *c)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens", [[1], [17], [1000], [8257], [16640, 3], [5000] * 3, [1] * 300, [0, 0, 0], [0, 9000, 0, 1]])
def test_few_and_many_sequences(dtype, lens):
    c = _case(lens, 28, 4, 128, 64, dtype, len(lens) + lens[0])
    _check(kernels.paged_attn(*c), *c)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_sharp_softmax(dtype):
    """Scores of a few hundred, whose largest comes late, early and in the middle."""
    c = _case([3000, 700, 64], 14, 2, 64, 16, dtype, 3, stretch=30.0)
    _check(kernels.paged_attn(*c), *c)


def test_scores_that_rise_all_along():
    """Every key raises the running maximum."""
    q, kp, vp, table, lens = _case([2000, 900], 7, 1, 128, 16, BF, 4)
    q = torch.ones_like(q)
    for b, n in enumerate(lens.tolist()):
        for t in range(n):
            kp[table[b, t // 16].long(), :, t % 16] = t / 100
    _check(kernels.paged_attn(q, kp, vp, table, lens), q, kp, vp, table, lens)


def test_infinite_and_lowest_scores():
    """A key with a score of -inf has no weight; keys that all lie at the type's lowest share it evenly."""
    q, kp, vp, table, lens = _case([40, 40], 4, 2, 64, 16, BF, 5)
    q = torch.zeros_like(q)
    q[:, :, 0] = 1
    for b in range(2):
        for t in range(40):
            kp[table[b, t // 16].long(), :, t % 16, 0] = float("-inf") if b == 0 and t % 2 else torch.finfo(BF).min
    got = kernels.paged_attn(q, kp, vp, table, lens, sm_scale=0.125)
    v = vp[table.long()].double().transpose(2, 3).flatten(1, 2)[:, :40]  # [B, T, Hkv, D]
    want = torch.stack([v[0, ::2].mean(0), v[1].mean(0)]).repeat_interleave(2, 1)
    assert bool(((got.double() - want).abs() <= 2.0 ** -7 * v.abs().amax(1).repeat_interleave(2, 1)).all())
    # with every score at -inf no key is left: zeros, as for a sequence without keys
    kp[..., 0] = float("-inf")
    assert int(kernels.paged_attn(q, kp, vp, table, lens).count_nonzero()) == 0


def test_nan_and_infinity_of_valid_keys_come_through():
    q, kp, vp, table, lens = _case([100, 100], 4, 2, 64, 16, BF, 6)
    kp[table[0, 1].long(), 0, 3, 5] = NAN   # sequence 0, KV head 0
    vp[table[1, 2].long(), 1, 4, 7] = NAN   # sequence 1, KV head 1, element 7
    got = kernels.paged_attn(q, kp, vp, table, lens)
    assert bool(got[0, :2].isnan().all()) and not bool(got[0, 2:].isnan().any())
    assert bool(got[1, 2:, 7].isnan().all()) and int(got[1].isnan().sum()) == 2


def test_bad_lengths_and_pages_are_flagged_and_not_read():
    c = q, kp, vp, table, lens = _case([100, 50, 40, 64], 4, 2, 128, 16, BF, 7)
    good = kernels.paged_attn(*c)
    for bad in (-1, table.shape[1] * 16 + 1, 2 ** 40, -2 ** 40):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        l2 = lens.clone()
        l2[1] = bad
        got = kernels.paged_attn(q, kp, vp, table, l2, err=err)
        assert int(err) == 2 and int(got[1].count_nonzero()) == 0
        assert torch.equal(got[[0, 2, 3]], good[[0, 2, 3]])
    for bad in (-1, kp.shape[0], 2 ** 31 - 1):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        t2 = table.clone()
        t2[2, 1] = bad  # keys 16..31 of 40 count as masked
        got = kernels.paged_attn(q, kp, vp, t2, lens, err=err)
        assert int(err) == 2 and torch.equal(got[[0, 1, 3]], good[[0, 1, 3]])
        t3 = table.clone()
        t3[2, 1] = table[2, 2]
        kp3, vp3 = kp.clone(), vp.clone()
        short = kernels.paged_attn(q, kp3, vp3, torch.cat([t3[:, :1], t3[:, 2:], t3[:, :1]], 1),
                                   torch.where(torch.arange(4, device=DEV) == 2, 24, lens))
        off = (got[2].float() - short[2].float()).abs()
        assert bool((off <= 2.0 ** -7 * short[2].float().abs() + 2.0 ** -7 * vp[table[2, :1].long()].float().abs().amax()).all())


def test_strided_queries_layer_views_and_scale():
    """Queries that are columns of a projection, one layer's view of a pool of all layers, a given scale."""
    c = q, kp, vp, table, lens = _case([77, 300, 5], 14, 2, 64, 16, BF, 8)
    wide = torch.zeros(3, 20 * 64, dtype=BF, device=DEV)
    wide[:, :14 * 64] = q.flatten(1)
    pool = [torch.full((p.shape[0], 3, *p.shape[1:]), NAN, dtype=BF, device=DEV) for p in (kp, vp)]
    for a, p in zip(pool, (kp, vp)):
        a[:, 1] = p
    out = torch.empty_like(q)
    got = kernels.paged_attn(wide[:, :14 * 64].unflatten(1, (14, 64)), pool[0][:, 1], pool[1][:, 1], table, lens,
                             out=out, sm_scale=0.3)
    assert got is out
    _check(got, *c, scale=0.3)
    # every second row of queries, and a table that is a part of a wider one
    q2 = torch.zeros(6, 14, 64, dtype=BF, device=DEV)
    q2[::2] = q
    t2 = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    t2[:, 2:2 + table.shape[1]] = table
    assert torch.equal(kernels.paged_attn(q2[::2], kp, vp, t2[:, 2:2 + table.shape[1]], lens), kernels.paged_attn(*c))


def test_shared_pages_and_repeated_calls_give_the_same_bits():
    """Sequences that share a prefix's pages, and the same call again and again."""
    q, kp, vp, table, lens = _case([640, 640, 640], 28, 4, 128, 64, BF, 9)
    table[1] = table[0]
    table[2, :9] = table[0, :9]
    q[1] = q[0]
    got = kernels.paged_attn(q, kp, vp, table, lens)
    _check(got, q, kp, vp, table, lens)
    for _ in range(5):
        assert torch.equal(kernels.paged_attn(q, kp, vp, table, lens), got)


def test_one_table_row_for_all_sequences():
    """Several queries over the pages of one sequence (a table expanded by stride 0), at lengths of their own."""
    q, kp, vp, table, _ = _case([1000], 28, 4, 128, 64, BF, 22)
    g = _gen(23)
    q = torch.randn(6, 28, 128, device=DEV, generator=g).to(BF)
    lens = torch.tensor([1000, 1, 64, 999, 0, 500], device=DEV)
    table = table.expand(6, -1)
    _check(kernels.paged_attn(q, kp, vp, table, lens), q, kp, vp, table, lens)


def test_output_over_the_queries():
    """out = q: every query is read before its row is written, in shares of one item and of several."""
    for lens in ([8000, 3], [60] * 100, [0, 5, 700]):
        q, *rest = _case(lens, 28, 4, 128, 64, BF, 21)
        want = kernels.paged_attn(q, *rest)
        got = kernels.paged_attn(q, *rest, out=q)
        assert got is q and torch.equal(q, want)


def test_other_streams_and_graphs():
    """Two graphs with calls of different sizes, and an eager call, each on a stream of its own, replayed
    together again and again."""
    cases = [_case([8000, 100], 28, 4, 128, 64, BF, 11), _case([300] * 20, 28, 4, 128, 64, BF, 12),
             _case([2500], 28, 4, 128, 64, BF, 13)]
    want = [kernels.paged_attn(*c) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kernels.paged_attn(*c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        last = kernels.paged_attn(*cases[2], stream=streams[2])
    torch.cuda.synchronize()
    for got, ref in zip(outs + [last], want):
        assert torch.equal(got, ref)


def test_lengths_on_the_device_decide_a_replay():
    """One captured call serves growing lengths."""
    q, kp, vp, table, lens = _case([500, 64], 14, 2, 64, 16, BF, 14)
    now = torch.tensor([1, 0], device=DEV)
    kernels.paged_attn(q, kp, vp, table, now)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kernels.paged_attn(q, kp, vp, table, now)
    for n in ((1, 0), (16, 1), (499, 63), (500, 64)):
        now.copy_(torch.tensor(n))
        g.replay()
        _check(out, q, kp, vp, table, now)


def test_long_pool_offsets_past_32_bits():
    page, Hkv, D = 256, 8, 128
    N = 2 ** 32 // (page * Hkv * D) + 4
    kp = torch.zeros(N, Hkv, page, D, dtype=BF, device=DEV)
    vp = torch.zeros(N, Hkv, page, D, dtype=BF, device=DEV)
    table = torch.tensor([[N - 1, 0, N - 2]], dtype=torch.int32, device=DEV)
    g = _gen(15)
    for i in table[0].long():
        kp[i], vp[i] = (torch.randn(Hkv, page, D, device=DEV, generator=g).to(BF) for _ in range(2))
    c = torch.randn(1, 40, D, device=DEV, generator=g).to(BF), kp, vp, table, torch.tensor([700], device=DEV)
    _check(kernels.paged_attn(*c), *c)


def test_attn_refuses_bad_tensors():
    q, kp, vp, table, lens = _case([20, 30], 4, 2, 64, 16, BF, 16)
    for bad in (dict(q=q.cpu()), dict(q=q.float()), dict(q=q[:, :, :32]), dict(table=table[:1]), dict(table=table.long()),
                dict(lens=lens.int()), dict(lens=lens[:1]), dict(lens=lens.cpu()), dict(v_pages=vp[:-1]),
                dict(out=torch.empty(2, 4, 64, device=DEV)), dict(k_pages=kp.transpose(1, 2)), dict(q=q.transpose(0, 1))):
        with pytest.raises(ValueError):
            kernels.paged_attn(**{**dict(q=q, k_pages=kp, v_pages=vp, table=table, lens=lens), **bad})
    with pytest.raises(RuntimeError, match="heads"):
        kernels.paged_attn(q[:, :3], kp, vp, table, lens)
    off = torch.empty(kp.numel() + 1, dtype=BF, device=DEV)[1:].view(kp.shape)  # 2 bytes off a 16-byte boundary
    with pytest.raises(RuntimeError, match="16-byte"):
        kernels.paged_attn(q, off, vp, table, lens)
    with pytest.raises(RuntimeError, match="16-byte"):
        odd = torch.empty(2, 4 * 64 + 1, dtype=BF, device=DEV)[:, :256].unflatten(1, (4, 64))
        kernels.paged_attn(odd, kp, vp, table, lens)
    with pytest.raises(RuntimeError, match="head_dim"):
        kernels.paged_attn(q[..., :32].contiguous(), kp[..., :32].contiguous(), vp[..., :32].contiguous(), table, lens)
