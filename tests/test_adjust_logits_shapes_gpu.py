"""Adjusting logits where the launch changes its shape: slices on either side of the shared memory that needs no
attribute (24 KB), the largest slice, as many rows as there are CTAs and more, counters of 16 and 32 bits."""
import pytest
import torch

from test_adjust_logits_gpu import _case, _check
from tread_b200 import kernels

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("H", [50, 16383, 16384])
@pytest.mark.parametrize("B,V", [
    (64, 110000), (64, 111000),            # 9 slices with 148 SMs: 16-bit counters below and above 24 KB
    (148, 24000), (148, 24800),            # 4 slices: the same for 32-bit counters
    (592, 18432), (700, 18432), (700, 18433),  # one slice of the largest size; one token more makes two
    (700, 100), (2000, 3),                 # more rows than CTAs, rows of one vector and less
])
def test_slices_of_every_size(dtype, H, B, V):
    logits, kw = _case(B, V, H, dtype, B + V + H, biases=3)
    rows = torch.tensor([0, 1, B // 2, B - 1], device="cuda")
    kw["lens"][rows[:2]] = torch.tensor([H, H - 1], device="cuda")
    got = kernels.adjust_logits(logits, **kw)
    _check(got[rows], logits[rows], **{k: v[rows] for k, v in kw.items()})
