"""The decode step's entry points called by several host threads at once, through the C ABI (the Python binding
holds the interpreter's lock for a whole call)."""
import threading

import pytest
import torch

from test_decode_capi import ADJUST_LOGITS
from tread_b200 import _capi as C

pytestmark = pytest.mark.gpu


def test_adjust_logits_of_two_sizes_from_two_threads():
    """Two sizes whose slices need 53 and 71 KB of shared memory, with counters of 32 bits: one call's limit must not
    replace the other's before its launch."""
    tokens = torch.zeros(20000, dtype=torch.int64, device="cuda")
    failed, outs = [], []

    def work(V, count):
        B = 64
        x = torch.randn(B, V, device="cuda", generator=torch.Generator("cuda").manual_seed(V)).bfloat16()
        lens, out = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.empty(B, V, device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        args = ADJUST_LOGITS.pack(x.data_ptr(), out.data_ptr(), tokens.data_ptr(), lens.data_ptr(), 0, 0, 0, 0, 0, 0, 0,
                                  V, V, 0, 0, 0, 0, B, V, 20000, 0, C.TREAD_BF16, C.TREAD_F32, 1.5, 0.0, 0.0)
        ready.wait()
        for _ in range(count):
            if C.lib().tread_adjust_logits(args, s.cuda_stream):
                failed.append(C.lib().tread_last_error().decode())
                break
        s.synchronize()
        outs.append((x, out))

    C.lib()
    ready = threading.Barrier(2)
    threads = [threading.Thread(target=work, args=(V, 4000)) for V in (118784, 160000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]
    assert all(torch.equal(out, x.float()) for x, out in outs)
