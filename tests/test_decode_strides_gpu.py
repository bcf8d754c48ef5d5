"""Views that PyTorch makes of dimensions of one element: their strides are any number and mean nothing."""
import pytest
import torch

from paged_oracle import inv_freq
from tread_b200 import kernels

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _odd(x, dims):
    """x with the strides of dimensions `dims` (of size one) odd."""
    assert all(x.shape[d] == 1 for d in dims)
    return x.as_strided(x.shape, [7 * s + 3 if d in dims else s for d, s in enumerate(x.stride())])


def _rand(*shape, seed):
    return torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(BF)


@pytest.mark.parametrize("Hkv,dims_q,dims_p", [(2, (0,), (0,)), (1, (0,), (0, 1)), (1, (), (1,))])
def test_attention_of_one_sequence_one_page_one_head(Hkv, dims_q, dims_p):
    q, kp, vp = _rand(1, 4, 64, seed=1), _rand(1, Hkv, 16, 64, seed=2), _rand(1, Hkv, 16, 64, seed=3)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([11], device="cuda")
    want = kernels.paged_attn(q, kp, vp, table, lens)
    got = kernels.paged_attn(_odd(q, dims_q), _odd(kp, dims_p), _odd(vp, dims_p), table, lens)
    assert torch.equal(got, want)


def test_appending_one_row_of_one_head_to_one_page():
    x = [_rand(1, 1, 64, seed=s) for s in (4, 5, 6)]
    pools = [torch.zeros(1, 1, 16, 64, dtype=BF, device="cuda") for _ in range(4)]
    table, pos = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([5], device="cuda")
    want = kernels.paged_append(x[0], x[1], pools[0], pools[1], table, pos, inv_freq=inv_freq(64), q=x[2])
    k, v, q = (_odd(t, (0, 1)) for t in x)
    got = kernels.paged_append(k, v, _odd(pools[2], (0, 1)), _odd(pools[3], (0, 1)), table, pos, inv_freq=inv_freq(64), q=q)
    assert torch.equal(got, want) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
