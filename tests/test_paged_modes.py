"""A paged cache that is made in inference mode and used outside of it, and the other way (no GPU)."""
import pytest
import torch

from tread_b200.paged import PagedCache


@pytest.mark.parametrize("made", [False, True])
@pytest.mark.parametrize("used", [False, True])
def test_pages_are_handed_out_and_given_back(made, used):
    with torch.inference_mode(made):
        pc = PagedCache(1, 1, 8, 6, page_size=2, max_seqs=2, max_len=12, dtype=torch.float32, device="cpu")
    with torch.inference_mode(used):
        a, b = pc.new(3), pc.new()
        pc.reserve(b, 1)
        pc.reserve(b, 4)
        assert pc.table[b].tolist() == pc._pages[b] + [-1] * 4
        pc.release(a)
        assert pc.table[a].tolist() == [-1] * 6 and pc.free_pages == 4
        assert pc.new(6) == a
