"""Host-side argument checks of the decode-step entry points (no GPU: nothing is launched)."""
import struct

import pytest

from tread_b200 import _capi as C

# the argument structs' fields in order, natively aligned
PAGED_APPEND = struct.Struct("@12P10q8if0q")
PAGED_ATTN = struct.Struct("@8P6q7if")
ADJUST_LOGITS = struct.Struct("@11P6q6i3f0q")


def _append_call(**over):
    a = dict(k=256, k_ld=1024, k_sh=128, v=256, v_ld=1024, v_sh=128, q=256, q_ld=1024, q_sh=128, q_out=256, kp=256,
             vp=256, ps=2 * 16 * 128, hs=16 * 128, N=8, page=16, table=256, t_ld=4, S=4, P=4, seq=None, pos=256,
             rpos=None, R=3, Hq=4, Hkv=2, D=128, inv=256, scale=1.0, err=None, dtype=C.TREAD_BF16)
    a.update(over)
    return C.lib().tread_paged_append(PAGED_APPEND.pack(*(a[n] or 0 for n in (
        "k v q q_out kp vp table seq pos rpos inv err k_ld k_sh v_ld v_sh q_ld q_sh ps hs N t_ld page S P R Hq Hkv D dtype "
        "scale").split())), None)


@pytest.mark.parametrize("over,needle", [
    (dict(R=-1), "R < 0"), (dict(k=None), "null"), (dict(pos=None), "null"), (dict(Hkv=0), "heads"),
    (dict(Hq=-1), "heads"), (dict(D=127), "head_dim"), (dict(D=258), "head_dim"), (dict(q=None), "query heads"),
    (dict(inv=None), "query heads"), (dict(q_out=None), "query heads"), (dict(dtype=7), "dtype"),
    (dict(page=0), "page geometry"), (dict(N=-1), "page geometry"), (dict(ps=100), "page geometry"),
    (dict(hs=100), "page geometry"), (dict(table=None), "page table"), (dict(t_ld=3), "page table"),
    (dict(R=5), "without seq"),
])
def test_paged_append_rejects_bad_arguments(over, needle):
    assert _append_call(**over) == 1
    assert needle in C.lib().tread_last_error().decode()


def _attn_call(**over):
    a = dict(q=256, q_ld=512, kp=256, vp=256, ps=2 * 16 * 128, hs=16 * 128, N=8, page=16, table=256, t_ld=4, P=4,
             lens=256, B=3, Hq=4, Hkv=2, D=128, scale=0.1, out=256, dtype=C.TREAD_BF16, ws=256, ws_bytes=None, err=None)
    a.update(over)
    n = C.lib().tread_paged_attn_workspace_bytes(4, 2, 128) if a["ws_bytes"] is None else a["ws_bytes"]
    a["ws_bytes"] = n
    return C.lib().tread_paged_attn(PAGED_ATTN.pack(*(a[k] or 0 for k in (
        "q kp vp out table lens err ws q_ld ps hs N t_ld ws_bytes page P B Hq Hkv D dtype scale").split())), None)


@pytest.mark.parametrize("over,needle", [
    (dict(B=-1), "B < 0"), (dict(q=None), "null"), (dict(lens=None), "null"), (dict(Hq=3), "heads"),
    (dict(Hq=34), "heads"), (dict(Hkv=0), "heads"), (dict(D=96), "head_dim"), (dict(dtype=9), "dtype"),
    (dict(page=0), "page geometry"), (dict(hs=16), "page geometry"), (dict(table=None), "page table"),
    (dict(t_ld=2), "page table"), (dict(q=264), "16-byte"), (dict(kp=264), "16-byte"), (dict(out=264), "16-byte"),
    (dict(q_ld=516), "16-byte"), (dict(ps=2 * 16 * 128 + 4), "16-byte"), (dict(P=2 ** 28, t_ld=2 ** 28), "2^31"),
    (dict(P=2 ** 26, t_ld=2 ** 26, B=9), "2^34"),
    (dict(ws=None), "workspace"), (dict(ws=264), "workspace"), (dict(ws_bytes=100), "workspace"),
])
def test_paged_attn_rejects_bad_arguments(over, needle):
    assert _attn_call(**over) == 1
    assert needle in C.lib().tread_last_error().decode()


def _logits_call(**over):
    a = dict(x=256, ld=100, out=256, ld_out=100, B=2, V=100, tok=256, tok_ld=8, H=8, lens=256, plens=256, rep=None,
             rep_all=1.2, pres=None, pres_all=0.0, freq=None, freq_all=0.0, ids=256, ids_ld=2, bias=256, bias_ld=2,
             nb=2, allowed=256, al_ld=4, dtype=C.TREAD_BF16, odt=C.TREAD_F32)
    a.update(over)
    return C.lib().tread_adjust_logits(ADJUST_LOGITS.pack(*(a[k] or 0 for k in (
        "x out tok lens plens rep pres freq ids bias allowed ld ld_out tok_ld ids_ld bias_ld al_ld B V H nb dtype odt "
        "rep_all pres_all freq_all").split())), None)


@pytest.mark.parametrize("over,needle", [
    (dict(B=-1), "B < 0"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(dtype=5), "dtype"),
    (dict(odt=5), "dtype"), (dict(ld=99), "row stride"), (dict(ld_out=99), "row stride"), (dict(H=-1), "history"),
    (dict(tok_ld=7), "history"), (dict(H=2 ** 30 + 1, tok_ld=2 ** 31), "history"), (dict(bias=None), "biases"), (dict(nb=-1), "biases"), (dict(nb=2049), "2048 biases"),
    (dict(B=65536), "65535 rows"), (dict(V=2 ** 31 - 1, ld=2 ** 31, ld_out=2 ** 31), "rows"), (dict(rep_all=0.0), "repetition"),
    (dict(rep_all=float("nan")), "repetition"),
])
def test_adjust_logits_rejects_bad_arguments(over, needle):
    assert _logits_call(**over) == 1
    assert needle in C.lib().tread_last_error().decode()


def test_null_arguments_are_refused():
    for name in ("tread_paged_append", "tread_paged_attn", "tread_adjust_logits"):
        assert getattr(C.lib(), name)(None, None) == 1
        assert "null" in C.lib().tread_last_error().decode()


def test_binding_refuses_host_tensors():
    import torch

    from tread_b200 import kernels

    x, pages = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    table, pos = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="no CPU path"):
        kernels.paged_append(x, x, pages, pages, table, pos)
    with pytest.raises(ValueError, match="no CPU path"):
        kernels.paged_attn(x, pages, pages, table, pos)
    with pytest.raises(ValueError, match="no CPU path"):
        kernels.adjust_logits(torch.zeros(2, 5))
    with pytest.raises(TypeError, match="k_pages must be a tensor"):
        kernels.paged_attn(x, [1], pages, table, pos)


def test_packed_structs_have_the_headers_layout(tmp_path):
    """Sizes and last fields' offsets, as the C compiler lays the structs out."""
    import os
    import subprocess

    from conftest import ROOT

    src = tmp_path / "layout.c"
    src.write_text("""#include <stddef.h>
        #include <stdio.h>
        #include "tread_b200.h"
        int main(void) {
          printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(tread_paged_append_args),
                 offsetof(tread_paged_append_args, attn_scaling), sizeof(tread_paged_attn_args),
                 offsetof(tread_paged_attn_args, sm_scale), sizeof(tread_adjust_logits_args),
                 offsetof(tread_adjust_logits_args, frequency_all));
          return 0;
        }""")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, check=True).stdout.split()]
    append, attn, logits = PAGED_APPEND.size, PAGED_ATTN.size, ADJUST_LOGITS.size
    assert got == [append, append - 8, attn, attn - 4, logits, logits - 8]


def test_empty_calls_are_noops():
    assert _append_call(R=0) == 0
    assert _attn_call(B=0) == 0
    assert _logits_call(B=0) == 0 and _logits_call(V=0) == 0
