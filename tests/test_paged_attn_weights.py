"""The weights of paged attention: inside the type's range wherever the scores lie."""
import pytest
import torch

from paged_oracle import make_table
from tread_b200 import kernels

HF = torch.float16


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
