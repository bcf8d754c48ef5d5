"""Reading and clearing the error words (no GPU: the selector's flag stands in as a CPU tensor)."""
from types import SimpleNamespace

import pytest
import torch

from tread_b200 import kernels
from tread_b200.qwen2 import Qwen2Rows
from tread_b200.tp import TPQwen2Rows


@pytest.mark.parametrize("cls", [Qwen2Rows, TPQwen2Rows])
@pytest.mark.parametrize("made_in_inference_mode", [False, True])
def test_an_error_is_told_and_cleared(cls, made_in_inference_mode, monkeypatch):
    """Words made inside Engine.prefill are inference tensors; the check may be called outside of it."""
    with torch.inference_mode(made_in_inference_mode):
        err, sel = torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(kernels, "selector_flags", lambda device: sel)
    net = SimpleNamespace(err=err, device=torch.device("cpu"), world=1)
    cls.check_errors(net)
    with torch.inference_mode():
        err[0] = 1
        sel[0] = 2
    with pytest.raises(RuntimeError, match="reported an error"):
        cls.check_errors(net)
    assert int(err.max()) == 0 and int(sel.max()) == 0
    cls.check_errors(net)
