"""How exactly the weights of paged attention meet the values: 16-bit types take each weight as the sum of two
numbers of the type, fp16 raised by 2^13 first. Bounds count what that loses, and are shown here (on the CPU, on
the arithmetic restated) to be passed by a kernel that drops the second part or does not raise fp16's weights."""
import pytest
import torch

from paged_oracle import attend64, make_table
from tread_b200 import kernels

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _bound(out, size, reach, n, top, plain, D, dtype):
    """How far the output may be off the 64-bit one, with u = half a step of the type, p the softmax:
    u |out| for the last rounding, and half of the type's smallest number below its normal range;
    2 d size (size = sum p |v|) for weights off by a relative d: fp32 scores summed over D products,
    (D + 2) 2^-24 reach; the exponential, 2^-20 (1 + reach / 8); fp32 sums, n 2^-24;
    u^2 size for a weight of 16 bits in two parts: the first leaves at most u of it, whose rounding is u of that;
    fp16's second part ends at 2^-24 (its rounding at 2^-25), the weights being raised by 2^13 against a maximum
    that is at most the largest score: 2^-38 of the largest weight, top, for each |v| (plain = sum |v|)."""
    f = torch.finfo(dtype)
    u = f.eps / 2
    d = (D + 2) * 2.0 ** -24 * reach + 2.0 ** -20 * (1 + reach / 8) + n * 2.0 ** -24
    off = u * out.abs() + 2 * d * size
    if dtype != FP:
        off = off + u * u * size
    if dtype == HF:
        off = off + 2.0 ** -38 * top * plain
    return 1.01 * off + f.smallest_normal * u


def _scores(n, far, at, gen, H):
    """[H, n] scores between -2 and 0 in steps of 2^-6 (exact in every type), key `at` the others' `far` nats up."""
    s = -torch.randint(0, 129, (H, n), generator=gen).double() / 64
    if far:
        s[:, at % n] = float(far)
    return s


def _restated(s, v, dtype, parts, raised):
    """The 16-bit kernel's arithmetic on scores [H, n] and values [n, D]: weights against the maximum, in `parts`
    parts of the type, raised by 2^raised; sums and products in 64 bits; one rounding to the type."""
    w = torch.exp(s - s.amax(-1, keepdim=True)).float() * 2.0 ** raised
    hi = w.to(dtype)
    used = hi.double()
    if parts == 2:
        used = used + (w - hi.float()).to(dtype).double()
    return ((used @ v.double()) / w.double().sum(-1, keepdim=True)).to(dtype).double()


def _exact(s, v):
    p = torch.softmax(s, -1)
    return p @ v.double(), p @ v.double().abs(), p.amax(-1, keepdim=True), v.double().abs().sum(0)


def _passes(dtype, parts, raised, n, far, scale):
    g = torch.Generator().manual_seed(n + far)
    s = _scores(n, far, n // 2, g, 16)
    v = (scale * torch.randn(n, 64, generator=g)).to(dtype)
    if far:
        v[n // 2] = 0
    out, size, top, plain = _exact(s, v)
    off = (_restated(s, v, dtype, parts, raised) - out).abs()
    return bool((off <= _bound(out, size, s.abs().amax(-1, keepdim=True), n, top, plain, 64, dtype)).all())


def _aligned(n, dtype, gen):
    """(scores [n], values [n]) whose weights' first roundings to the type all push the sum the same way: values of
    random size with the sign of what the rounding leaves out. Every unit of 16 keys has a score of 0, the largest,
    so that each running maximum is 0; their weights have no rounding, and their values cancel the others' sum, so
    that the output's own rounding is small. (With random signs the roundings average out as the root of n.)"""
    s = _scores(n, 0, 0, gen, 1)[0]
    s[::16] = 0
    w = torch.exp(s).float()
    v = ((w - w.to(dtype).float()) >= 0).float() * 2 - 1
    v = v * (0.5 + torch.rand(n, generator=gen))
    v[s == 0] = 0
    v[s == 0] = -(w * v).sum() / (s == 0).sum()
    return s, v


# from about 1200 keys on, the bound's fp32 sums (2 n 2^-24) pass what one rounding of fp16's weights can add (0.3 u)
@pytest.mark.parametrize("dtype,n", [(BF, 20), (BF, 64), (BF, 300), (BF, 2000), (HF, 20), (HF, 64), (HF, 300)])
def test_the_bound_tells_one_part_from_two(dtype, n):
    g = torch.Generator().manual_seed(n)
    s, v = _aligned(n, dtype, g)
    v = v.to(dtype)[:, None]
    out, size, top, plain = _exact(s[None], v)
    raised = 13 if dtype == HF else 0
    bound = _bound(out, size, s.abs().amax().view(1, 1), n, top, plain, 64, dtype)
    off = lambda parts: (_restated(s[None], v, dtype, parts, raised) - out).abs()  # noqa: E731
    assert bool((off(2) <= bound).all()) and bool((off(1) > bound).all())


@pytest.mark.parametrize("n", [20, 300, 2000])
@pytest.mark.parametrize("far", [12, 14, 16, 18])
def test_the_bound_tells_raised_weights_of_fp16(n, far):
    assert _passes(HF, 2, 13, n, far, 1000.0) and not _passes(HF, 2, 0, n, far, 1000.0)
    assert _passes(BF, 2, 0, n, far, 1000.0)


# ---- the kernel ---------------------------------------------------------------------------------


def _attend(dtype, n, far, at, scale, D=64, G=7, Hkv=2, page=16, seed=0):
    """Queries that read the scores out of the keys' first G elements: score of head h = key's element h."""
    g = torch.Generator().manual_seed(seed + n)
    table, pool = make_table([n], page, torch.Generator("cuda").manual_seed(seed))
    q = torch.zeros(1, Hkv * G, D)
    q[0, torch.arange(Hkv * G), torch.arange(Hkv * G) % G] = 1
    kp, vp = torch.zeros(pool, Hkv, page, D), torch.zeros(pool, Hkv, page, D)
    ids = table[0, torch.arange(n) // page].long().cpu()
    for h in range(Hkv):
        k = torch.zeros(n, D)
        k[:, :G] = _scores(n, far, at, g, G).T.float()
        v = scale * torch.randn(n, D, generator=g)
        if far:
            v[at % n] = 0
        kp[ids, h, torch.arange(n) % page] = k
        vp[ids, h, torch.arange(n) % page] = v
    q, kp, vp = (t.to("cuda", dtype) for t in (q, kp, vp))
    lens = torch.tensor([n], device="cuda")
    got = kernels.paged_attn(q, kp, vp, table, lens, sm_scale=1.0).double()
    out, size, reach = attend64(q, kp, vp, table, lens, 1.0)
    k, v = (p[table[0].long()].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :n] for p in (kp, vp))
    p = torch.softmax(q[0].double().view(Hkv, G, D) @ k.transpose(1, 2), -1)
    top = p.amax(-1).view(1, Hkv * G, 1)
    plain = v.abs().sum(1).repeat_interleave(G, 0)[None]
    off = (got - out).abs()
    bound = _bound(out, size, reach, n, top, plain, D, dtype)
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("n", [1, 20, 64, 300, 2000, 9000])
@pytest.mark.parametrize("D,G", [(64, 7), (128, 5), (256, 8), (128, 16)])
def test_weights_keep_sixteen_bits(dtype, n, D, G):
    _attend(dtype, n, 0, 0, 1.0, D=D, G=G)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n", [20, 64, 300, 2000])
def test_roundings_that_add_up(dtype, n):
    D, page = 64, 16
    s, v = _aligned(n, dtype, torch.Generator().manual_seed(n))
    table, pool = make_table([n], page, torch.Generator("cuda").manual_seed(n))
    ids, slots = table[0, torch.arange(n) // page].long().cpu(), torch.arange(n) % page
    q, kp, vp = torch.zeros(1, 4, D), torch.zeros(pool, 1, page, D), torch.zeros(pool, 1, page, D)
    q[..., 0] = 1
    kp[ids, 0, slots, 0] = s.float()
    vp[ids, 0, slots] = v[:, None]
    q, kp, vp = (t.to("cuda", dtype) for t in (q, kp, vp))
    got = kernels.paged_attn(q, kp, vp, table, torch.tensor([n], device="cuda"), sm_scale=1.0).double().cpu()
    out, size, top, plain = _exact(s[None], v.to(dtype)[:, None])
    bound = _bound(out, size, s.abs().amax().view(1, 1), n, top, plain, D, dtype)
    assert bool(((got - out).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("n", [20, 300, 2000, 8000])
@pytest.mark.parametrize("far", [8, 12, 14, 16, 18])
def test_a_far_key_whose_value_is_zero(dtype, n, far):
    """An attention sink: the keys far below it make the whole output. The first key, the last, one between."""
    for at in (0, n // 2, n - 1):
        _attend(dtype, n, far, at, 1000.0, seed=at)


@pytest.mark.gpu
def test_fp16_scores_whose_steps_are_wide():
    """Scores past 2^27, 16 apart in fp32, that rise by a step or two every few units: what the running maximum may
    lag is a difference, not a sum that rounds up to a whole step, which would take the weights out of fp16's range."""
    n, page, D, B = 512, 16, 64, 300  # so many sequences (over the same pages) that a share is a whole one
    table, pool = make_table([n], page, torch.Generator("cuda").manual_seed(1))
    step = (torch.arange(n, device="cuda") // 64).to(HF)  # every warp sees each of them
    q, kp = torch.zeros(B, 8, D, dtype=HF, device="cuda"), torch.zeros(pool, 1, page, D, dtype=HF, device="cuda")
    q[..., 0], q[..., 1] = 128, 2.0 ** -9
    kp[..., 0] = 128
    at = torch.arange(n, device="cuda")
    kp[table[0, at // page].long(), 0, at % page, 1] = step
    vp = torch.randn(pool, 1, page, D, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(HF)
    got = kernels.paged_attn(q, kp, vp, table.expand(B, -1), torch.full((B,), n, device="cuda"), sm_scale=2.0 ** 13)
    assert bool(got.isfinite().all()) and float(got.abs().max()) <= float(vp.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_infinite_values_stay_in_their_element(dtype):
    """Not finite in the element and the heads that read it, whatever the weight's two parts are; the others as
    without it."""
    g = torch.Generator("cuda").manual_seed(3)
    table, pool = make_table([100], 16, g)
    q = torch.randn(1, 8, 64, device="cuda", generator=g).to(dtype)
    kp, vp = (torch.randn(pool, 2, 16, 64, device="cuda", generator=g).to(dtype) for _ in range(2))
    lens = torch.tensor([100], device="cuda")
    want = kernels.paged_attn(q, kp, vp, table, lens)
    for sign in (1, -1):
        v2 = vp.clone()
        v2[table[0, 3].long(), 1, 5, 9] = sign * torch.inf
        got = kernels.paged_attn(q, kp, v2, table, lens)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[0, 4:, 9] = True
        assert torch.equal(got.isfinite(), ~hit) and torch.equal(got[~hit], want[~hit])
        if dtype == FP:
            assert bool((got[hit] == sign * torch.inf).all())
