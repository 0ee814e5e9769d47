"""CPU checks of the training operators' C structs: the ctypes mirrors have the
C compiler's field offsets and sizes, and the constants the header's values."""

from __future__ import annotations

import ctypes
import json
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_structs_and_constants_match_the_c_header(tmp_path):
    import torch
    from qqt_b200 import _capi
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    want = {}
    for cls in (_capi.QqtSeq, _capi.QqtPolicyLoss):
        for f in cls._fields_:
            want[f"offsetof({cls.__name__}, {f[0]})"] = getattr(cls, f[0]).offset
        want[f"sizeof({cls.__name__})"] = ctypes.sizeof(cls)
    want["QQT_MAX_HEADS"] = _capi.MAX_HEADS
    for name, dtype in (("QQT_F32", torch.float32), ("QQT_F16", torch.float16),
                        ("QQT_BF16", torch.bfloat16)):
        want[name] = _capi.DTYPES[dtype]
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "qqt_b200.h"',
             "int main(void) {"]
    lines += [f'printf("%s\\"{k}\\": %zu", "{"{" if i == 0 else ","}", (size_t)({k}));'
              for i, k in enumerate(want)]
    lines += ['printf("}");', "return 0; }"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    got = json.loads(subprocess.run([str(exe)], check=True, capture_output=True).stdout)
    assert got == want


def test_work_sizes_cover_both_directions_and_every_type():
    """One workspace serves any call of a size, and nothing is asked for where
    there is nothing to do."""
    from qqt_b200 import _capi
    L = _capi.lib()
    assert L.qqt_recurrence_work_bytes(0, 4, 4) == 0
    assert L.qqt_recurrence_work_bytes(8, 4, 4) == 0          # one segment
    assert L.qqt_policy_loss_work_bytes(0) >= 0
    assert L.qqt_recurrence_chunks(0) == 0 and L.qqt_recurrence_chunks(9) == 2
    n = L.qqt_layernorm_work_bytes(1, 7)
    assert n >= 2 * 7 * 4


@pytest.mark.parametrize("off", [4, 8, 12])
def test_workspaces_off_their_alignment_are_refused(off):
    """The kernels move workspaces by accesses of up to 16 bytes: refused before
    anything is launched (made-up addresses)."""
    from qqt_b200 import _capi
    L, P = _capi.lib(), 0x100000
    s = _capi.QqtSeq(P, 1024, 1024)
    r = ctypes.byref(s)
    assert L.qqt_recurrence_work_bytes(4096, 1, 1024) > 0
    assert L.qqt_recurrence_forward(r, r, None, P, 0, 4096, 1, 1024, r, P, P, P + off, None) == 2
    assert L.qqt_recurrence_backward(r, P, r, r, None, P, 0, 4096, 1, 1024, r, r, P, P + off,
                                     None) == 2
    assert L.qqt_layernorm_backward(P, 8, P, 8, 0, 4, 8, P, P, P, P, P, P, P + off, None) == 2
    a = _capi.QqtPolicyLoss(logits=P, row_stride=7, rows=4, actions=P, action_stride=1, old_logp=P,
                            adv=P, stats=P, work=P + off, grad_scale=1.0, dtype=0, n_heads=1)
    a.width[0] = 7
    assert L.qqt_policy_loss(ctypes.byref(a), None) == 2
