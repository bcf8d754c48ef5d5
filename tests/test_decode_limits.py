"""Limits of the decode-step entry points at the value itself (no GPU: nothing is launched)."""
from test_decode_capi import _logits_call
from tread_b200 import _capi as C


def test_a_history_whose_counts_pass_a_counter_is_refused():
    """2^30 times one token would set the mark above the count; 2^30 - 1 is the last that fits (not launched here:
    no rows)."""
    assert _logits_call(H=2 ** 30, tok_ld=2 ** 30) == 1
    assert "history" in C.lib().tread_last_error().decode()
    assert _logits_call(H=2 ** 30 - 1, tok_ld=2 ** 30, B=0) == 0
