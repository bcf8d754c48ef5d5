"""Appending to a paged cache (tread_paged_append) against the definition in 64 bits: places, rotation,
copies, every slot that no row names left as it was, padding rows, and rows that are out of range."""
import pytest
import torch

from paged_oracle import inv_freq, make_table, rotate64, rotate_bound
from tread_b200 import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _case(counts, past, Hq, Hkv, D, page, dtype, seed):
    """New tokens `counts[i]` of sequence i behind `past[i]` earlier ones, rows of all sequences packed."""
    g = _gen(seed)
    lens = [a + n for a, n in zip(past, counts)]
    table, pool = make_table(lens, page, g)
    R = sum(counts)
    seq = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(counts)]).to(DEV)
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(past, counts)]).to(DEV)
    qkv = torch.randn(R, (Hq + 2 * Hkv) * D, device=DEV, generator=g).to(dtype)
    q = qkv[:, :Hq * D].unflatten(1, (Hq, D))
    k = qkv[:, Hq * D:(Hq + Hkv) * D].unflatten(1, (Hkv, D))
    v = qkv[:, (Hq + Hkv) * D:].unflatten(1, (Hkv, D))
    kp = torch.randn(pool, Hkv, page, D, device=DEV, generator=g).to(dtype)
    vp = torch.randn(pool, Hkv, page, D, device=DEV, generator=g).to(dtype)
    return q, k, v, kp, vp, table, pos, seq


def _check(got, want, x, dtype, exact=False):
    if exact:
        assert torch.equal(got, want.to(dtype))
        return
    off = (got.double() - want).abs()
    assert bool((off <= rotate_bound(x, want, dtype)).all()), f"off by {float(off.max()):.3g}"


def _check_pages(kp, vp, kp0, vp0, k, v, table, pos, seq, angle, inv):
    page = kp.shape[2]
    at, slot = table[seq.long(), pos // page].long(), pos % page
    want_k = k.double() if inv is None else rotate64(k, angle, inv)
    _check(kp[at, :, slot], want_k, k, kp.dtype, exact=inv is None)
    assert torch.equal(vp[at, :, slot], v)
    for new, old in ((kp, kp0), (vp, vp0)):  # every other slot as it was
        keep = torch.ones(new.shape[0], page, dtype=torch.bool, device=DEV)
        keep[at, slot] = False
        assert torch.equal(new.transpose(1, 2)[keep], old.transpose(1, 2)[keep])


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("Hq,Hkv,D,page,counts,past", [
    (28, 4, 128, 64, [1], [8256]),
    (28, 4, 128, 16, [1] * 9, [0, 1, 15, 16, 17, 31, 32, 63, 200]),
    (14, 2, 64, 16, [5, 1, 40], [0, 100, 7]),
    (4, 2, 64, 7, [3, 20], [6, 0]),
    (8, 1, 256, 1, [2, 3], [0, 5]),
    (3, 3, 6, 4, [9], [2]),          # a head of 6: single elements
    (40, 8, 128, 32, [1500], [33]),  # tiles of several rows
])
def test_append_rows(dtype, Hq, Hkv, D, page, counts, past):
    q, k, v, kp, vp, table, pos, seq = _case(counts, past, Hq, Hkv, D, page, dtype, 1)
    kp0, vp0, inv = kp.clone(), vp.clone(), inv_freq(D)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = kernels.paged_append(k, v, kp, vp, table, pos, seq=seq, inv_freq=inv, q=q, err=err)
    _check(got, rotate64(q, pos, inv), q, dtype)
    _check_pages(kp, vp, kp0, vp0, k, v, table, pos, seq, pos, inv)
    assert int(err) == 0


@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_scaling(dtype):
    """cos and sin times a factor: the rotation's bound times it, and two roundings more (2^-24 of the factor
    each, inside the 2^-21)."""
    q, k, v, kp, vp, table, pos, seq = _case([20], [700], 4, 2, 64, 16, dtype, 11)
    inv, factor = inv_freq(64), 1.7
    got = kernels.paged_append(k, v, kp, vp, table, pos, seq=seq, inv_freq=inv, attn_scaling=factor, q=q)
    at, slot = table[0, pos // 16].long(), pos % 16
    for a, x in ((got, q), (kp[at, :, slot], k)):
        want = rotate64(x, pos, inv) * factor
        assert bool(((a.double() - want).abs() <= factor * rotate_bound(x, want, dtype)).all())


def test_append_without_seq_is_one_row_a_sequence():
    q, k, v, kp, vp, table, pos, seq = _case([1] * 6, [3, 0, 100, 64, 63, 5], 4, 2, 128, 64, BF, 2)
    kp2, vp2, inv = kp.clone(), vp.clone(), inv_freq(128)
    a = kernels.paged_append(k, v, kp, vp, table, pos, inv_freq=inv, q=q)
    b = kernels.paged_append(k, v, kp2, vp2, table, pos, seq=seq, inv_freq=inv, q=q)
    assert torch.equal(a, b) and torch.equal(kp, kp2) and torch.equal(vp, vp2)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("where", [1, 4096, 16384, 131071, 2 ** 24 + 1, 2 ** 31 - 1, -1, -16384])
def test_rotation_keeps_far_positions(dtype, where):
    """The angle of far and negative positions is formed in 64 bits (the token's place is another thing)."""
    q, k, v, kp, vp, table, pos, seq = _case([7], [2], 4, 2, 128, 16, dtype, 3)
    kp0, vp0, inv = kp.clone(), vp.clone(), inv_freq(128)
    angle = torch.full_like(pos, where)
    got = kernels.paged_append(k, v, kp, vp, table, pos, seq=seq, inv_freq=inv, rope_pos=angle, q=q)
    _check(got, rotate64(q, angle, inv), q, dtype)
    _check_pages(kp, vp, kp0, vp0, k, v, table, pos, seq, angle, inv)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_copy_from_a_dense_cache_of_all_layers(dtype):
    """[L, 1, Hkv, T, D] moved into pages [N, L, Hkv, page, D] in one call, then one layer of it again
    through the layer's view of the pool."""
    g = _gen(4)
    L, H, T, D, page = 3, 2, 77, 64, 16
    table, pool = make_table([T], page, g)
    K, V = (torch.randn(L, 1, H, T, D, device=DEV, generator=g).to(dtype) for _ in range(2))
    kp, vp = (torch.zeros(pool, L, H, page, D, dtype=dtype, device=DEV) for _ in range(2))
    pos, seq = torch.arange(T, device=DEV), torch.zeros(T, dtype=torch.int32, device=DEV)
    flat = lambda t: t.view(L * H, T, D).transpose(0, 1)  # noqa: E731
    kernels.paged_append(flat(K), flat(V), kp.flatten(1, 2), vp.flatten(1, 2), table, pos, seq=seq)
    at = table[0].long()
    for src, pages in ((K, kp), (V, vp)):
        assert torch.equal(pages[at].permute(1, 2, 0, 3, 4).reshape(L, H, -1, D)[:, :, :T], src[:, 0])
    kp2, vp2 = torch.zeros_like(kp), torch.zeros_like(vp)
    for l in range(L):
        kernels.paged_append(K[l, 0].transpose(0, 1), V[l, 0].transpose(0, 1), kp2[:, l], vp2[:, l], table, pos, seq=seq)
    assert torch.equal(kp, kp2) and torch.equal(vp, vp2)


def test_special_values_pass_through():
    q, k, v, kp, vp, table, pos, seq = _case([4], [0], 2, 2, 64, 16, BF, 5)
    v = v.clone()
    v[0, 0, 0], v[1, 0, 3], v[2, 1, 5] = float("inf"), float("nan"), -0.0
    kernels.paged_append(k, v, kp, vp, table, pos, seq=seq)
    got = vp[table[0, 0].long()].transpose(0, 1)[:4]
    assert torch.equal(got.view(torch.int16), v.view(torch.int16))


@pytest.mark.parametrize("R", [1, 5, 700])
def test_padding_rows_leave_everything(R):
    q, k, v, kp, vp, table, pos, seq = _case([R + 3], [10], 4, 2, 128, 16, BF, 6)
    pad = torch.zeros(R + 3, dtype=torch.bool, device=DEV)
    pad[::2] = True
    pos2 = torch.where(pad, -1, pos)
    kp0, vp0, inv = kp.clone(), vp.clone(), inv_freq(128)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = kernels.paged_append(k, v, kp, vp, table, pos2, seq=seq, inv_freq=inv, q=q, err=err)
    assert int(err) == 0 and int(got[pad].count_nonzero()) == 0
    _check(got[~pad], rotate64(q, pos, inv)[~pad], q[~pad], BF)
    _check_pages(kp, vp, kp0, vp0, k[~pad], v[~pad], table, pos[~pad], seq[~pad], pos[~pad], inv)


def test_rows_out_of_range_are_skipped_and_flagged():
    """A sequence, position or page id that does not exist: nothing is written for that row."""
    for what in ("sequence", "negative sequence", "position", "page", "negative page"):
        q, k, v, kp, vp, table, pos, seq = _case([1] * 5, [3, 20, 40, 17, 0], 4, 2, 128, 16, BF, 7)
        if what == "sequence":
            seq[2] = 5
        elif what == "negative sequence":
            seq[2] = -1
        elif what == "position":
            pos[2] = table.shape[1] * 16
        elif what == "page":
            table[2, 2] = kp.shape[0]
        else:
            table[2, 2] = -1
        kp0, vp0, inv = kp.clone(), vp.clone(), inv_freq(128)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = kernels.paged_append(k, v, kp, vp, table, pos, seq=seq, inv_freq=inv, q=q, err=err)
        assert int(err) == 1 and int(got[2].count_nonzero()) == 0
        ok = torch.arange(5, device=DEV) != 2
        _check_pages(kp, vp, kp0, vp0, k[ok], v[ok], table, pos[ok], seq[ok], pos[ok], inv)


def test_queries_rotate_in_place_and_odd_alignment():
    q, k, v, kp, vp, table, pos, seq = _case([33], [5], 4, 2, 128, 16, BF, 8)
    inv = inv_freq(128)
    q1 = q.contiguous()
    want = kernels.paged_append(k, v, kp.clone(), vp.clone(), table, pos, seq=seq, inv_freq=inv, q=q1.clone())
    got = kernels.paged_append(k, v, kp, vp, table, pos, seq=seq, inv_freq=inv, q=q1, q_out=q1)
    assert got is q1 and torch.equal(got, want)
    # keys that start 2 bytes off a vector, and a row stride that no vector divides
    wide = torch.zeros(33, 2 * 128 + 3, dtype=BF, device=DEV)
    off = wide[:, 1:257].unflatten(1, (2, 128))
    off.copy_(k)
    kp2, vp2 = kp.clone(), vp.clone()
    kernels.paged_append(off, v, kp2, vp2, table, pos, seq=seq, inv_freq=inv)
    assert torch.equal(kp, kp2) and torch.equal(vp, vp2)


def test_pool_offsets_past_32_bits():
    """Slots whose element offset in the pool passes 2^32."""
    page, H, D = 256, 8, 128
    N = 2 ** 32 // (page * H * D) + 4
    kp = torch.zeros(N, H, page, D, dtype=BF, device=DEV)
    table = torch.tensor([[N - 1, 0, N - 2]], dtype=torch.int32, device=DEV)
    pos = torch.tensor([255, 256, 767], device=DEV)
    k = torch.randn(3, H, D, device=DEV, generator=_gen(9)).to(BF)
    seq = torch.zeros(3, dtype=torch.int32, device=DEV)
    kernels.paged_append(k, k, kp, kp, table, pos, seq=seq)
    assert torch.equal(kp[N - 1, :, 255], k[0]) and torch.equal(kp[0, :, 0], k[1]) and torch.equal(kp[N - 2, :, 255], k[2])
    assert int(kp.count_nonzero()) == int(k.count_nonzero())


def test_append_refuses_bad_tensors():
    q, k, v, kp, vp, table, pos, seq = _case([4], [0], 4, 2, 64, 16, BF, 10)
    inv = inv_freq(64)
    call = lambda **o: kernels.paged_append(**{**dict(k=k, v=v, k_pages=kp, v_pages=vp, table=table, pos=pos,  # noqa: E731
                                                      seq=seq, inv_freq=inv, q=q), **o})
    for bad in (dict(k=k.cpu()), dict(table=table.cpu()), dict(pos=pos.int()), dict(pos=pos[:3]), dict(seq=seq.long()),
                dict(table=table.long()), dict(v=v[:, :1]), dict(inv_freq=inv[:5]), dict(inv_freq=inv.double()),
                dict(inv_freq=None), dict(q=q[:3]), dict(q_out=torch.empty(4, 4, 64, device=DEV)), dict(seq=None),
                dict(v_pages=vp[:-1]), dict(rope_pos=pos.float()), dict(err=torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(TypeError):
        call(k=k.float(), v=v.float(), q=None)
