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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_workspaces_of_their_stated_size_are_enough(dtype):
    """Every entry with a workspace of exactly the bytes that its _work_bytes
    names, both directions: what lies behind it is unchanged, and the results
    are those of the Python calls."""
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from qqt_b200 import _capi, norm, policy_loss, recurrence
    L, dt = _capi.lib(), getattr(torch, dtype)
    code, st = _capi.DTYPES[dt], torch.cuda.current_stream().cuda_stream
    gen = torch.Generator(device="cuda").manual_seed(5)
    spare = 1 << 16

    def r(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    class Work:
        def __init__(self, nbytes):
            self.buf = torch.full((nbytes + spare,), 0xA5, dtype=torch.uint8, device="cuda")
            self.n, self.p = nbytes, self.buf.data_ptr()

        def check(self):
            assert bool((self.buf[self.n:] == 0xA5).all())

    # widths on either side of where the plans of 4 and of 8 values a vector differ
    for n, d in ((1, 7), (700, 64), (5000, 130), (3000, 512), (2000, 520), (999, 1352), (77, 8200),
                 (40, 16385), (600, 20000)):
        x, dy, w = r(n, d).to(dt), r(n, d).to(dt), r(d)
        _, mean, rstd = norm.layer_norm_forward(x, w)
        want = norm.layer_norm_backward(dy, x, mean, rstd, w)
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        work = Work(L.qqt_layernorm_work_bytes(n, d))
        assert L.qqt_layernorm_backward(
            dy.data_ptr(), d, x.data_ptr(), d, code, n, d, mean.data_ptr(), rstd.data_ptr(),
            w.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), work.p, st) == 0
        work.check()
        assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), want))
    # uncut, cut in two directions alike and not, few and many channels
    for t, n, d in ((40, 3, 64), (4096, 1, 1024), (10007, 3, 517), (5000, 1, 3), (600, 40, 128),
                    (2000, 2, 258)):
        x, g, dh = (r(t, n, d).to(dt) for _ in range(3))
        h, last, saved = recurrence.gated_recurrence_forward(x, g)
        want = recurrence.gated_recurrence_backward(dh, None, x, g, saved)
        seq = [_capi.QqtSeq(v.data_ptr(), n * d, d) for v in (x, g, dh)]
        h2, dx, dg = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
        out = [_capi.QqtSeq(v.data_ptr(), n * d, d) for v in (h2, dx, dg)]
        l2, c2, d0 = torch.empty_like(last), torch.empty_like(saved), torch.empty_like(last)
        ref = ctypes.byref
        work = Work(L.qqt_recurrence_work_bytes(t, n, d))
        assert L.qqt_recurrence_forward(ref(seq[0]), ref(seq[1]), None, None, code, t, n, d,
                                        ref(out[0]), l2.data_ptr(), c2.data_ptr(), work.p, st) == 0
        work.check()
        assert L.qqt_recurrence_backward(ref(seq[2]), None, ref(seq[0]), ref(seq[1]), None,
                                         c2.data_ptr(), code, t, n, d, ref(out[1]), ref(out[2]),
                                         d0.data_ptr(), work.p, st) == 0
        work.check()
        assert all(torch.equal(p, q) for p, q in zip((h2, l2, c2, dx, dg, d0),
                                                     (h, last, saved) + want))
    for n, v in ((1, 7), (5000, 7), (9000, 7), (600, 40), (300, 2000), (20, 40000)):
        z, adv, old = r(n, v).to(dt), r(n), r(n) - 3
        act = torch.zeros((n, 1), dtype=torch.int64, device="cuda")
        mask = r(n) > -1
        want = policy_loss.policy_loss_and_grad(z, act, old, adv, mask=mask)
        stats, logp, dz = torch.empty(5, device="cuda"), torch.empty_like(adv), torch.empty_like(z)
        work = Work(L.qqt_policy_loss_work_bytes(n))
        a = _capi.QqtPolicyLoss(
            logits=z.data_ptr(), row_stride=v, rows=n, actions=act.data_ptr(), action_stride=1,
            old_logp=old.data_ptr(), adv=adv.data_ptr(), mask=mask.data_ptr(), logp=logp.data_ptr(),
            stats=stats.data_ptr(), dlogits=dz.data_ptr(), dlogits_stride=v, work=work.p,
            clip_low=0.2, clip_high=0.2, grad_scale=1.0, dtype=code, n_heads=1)
        a.width[0] = v
        assert L.qqt_policy_loss(ctypes.byref(a), st) == 0
        work.check()
        assert all(torch.equal(p, q) for p, q in zip((stats, logp, dz), want))
