"""Outputs over their inputs: the same elements are fine, others are refused, columns beside each other are not."""
import pytest
import torch

from paged_oracle import inv_freq
from tread_b200 import kernels

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _buffer(*shape, dtype=BF):
    return torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dtype)


def _pages():
    return [_buffer(4, 2, 16, 64) for _ in range(2)]


def test_attention_output():
    kp, vp = _pages()
    table, lens = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), torch.tensor([20, 31], device="cuda")
    wide = _buffer(4, 4, 64)
    q = wide[::2]  # rows 0 and 2
    want = kernels.paged_attn(q, kp, vp, table, lens)
    for bad in (wide[:2], wide[1:3], wide[2:]):
        with pytest.raises(ValueError, match="overlaps q"):
            kernels.paged_attn(q, kp, vp, table, lens, out=bad)
    flat = wide.flatten()
    with pytest.raises(ValueError, match="overlaps q"):
        kernels.paged_attn(q, kp, vp, table, lens, out=flat[64:64 + 512].view(2, 4, 64))
    assert torch.equal(kernels.paged_attn(q, kp, vp, table, lens, out=_buffer(2, 4, 64)), want)
    one = wide[2:3]
    got = kernels.paged_attn(wide[:1], kp, vp, table[:1], lens[:1], out=one)  # between the other's rows
    assert torch.equal(got, want[:1])


def test_rotated_queries():
    kp, vp = _pages()
    table, pos = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 2], device="cuda")
    qkv = _buffer(3, 8 * 64)
    q, k, v = (qkv[:, a:b].unflatten(1, (-1, 64)) for a, b in ((0, 256), (256, 384), (384, 512)))
    flat = qkv.flatten()
    call = lambda **kw: kernels.paged_append(k, v, kp, vp, table, pos, inv_freq=inv_freq(64), q=q, **kw)  # noqa: E731
    for at, name in ((0, "q"), (64, "q"), (512, "q")):
        with pytest.raises(ValueError, match=f"overlaps {name}"):
            call(q_out=flat[at:at + 768].view(3, 4, 64))
    with pytest.raises(ValueError, match="overlaps k"):
        kernels.paged_append(k[:1], v[:1], kp, vp, table[:1], pos[:1], inv_freq=inv_freq(64), q=q[:1],
                             q_out=flat[256:512].view(1, 4, 64))
    with pytest.raises(ValueError, match="overlaps v"):
        kernels.paged_append(k[:1], v[:1], kp, vp, table[:1], pos[:1], inv_freq=inv_freq(64), q=q[:1],
                             q_out=flat[384:640].view(1, 4, 64))
    assert call().shape == (3, 4, 64)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_adjusted_logits(dtype):
    wide = _buffer(3, 300, dtype=dtype)
    x = wide[:, :100]
    want = kernels.adjust_logits(x, out=torch.empty(3, 100, dtype=dtype, device="cuda"))
    for bad in (wide[:, 1:101], wide[:, 99:199], wide.flatten()[:300].view(3, 100), wide.flatten()[300:600].view(3, 100)):
        with pytest.raises(ValueError, match="overlaps logits"):
            kernels.adjust_logits(x, out=bad)
    assert torch.equal(kernels.adjust_logits(x, out=wide[:, 100:200]), want)  # columns beside the logits
    assert torch.equal(kernels.adjust_logits(x, out=wide[:, 200:]), want)
    assert torch.equal(kernels.adjust_logits(x, out=x), want)
