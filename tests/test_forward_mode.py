"""Forward-mode derivatives of the training operators: they have none, and a
dual tensor says so instead of losing its tangent.  On the host, with the
kernels' calls replaced by ones that return their input."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwad

from qqt_b200 import norm, recurrence


def _cases(monkeypatch):
    monkeypatch.setattr(norm, "layer_norm_forward",
                        lambda x, w, b=None, eps=0, stats=True: (x * 1, x[:, 0] * 1, x[:, 0] * 1))
    monkeypatch.setattr(recurrence, "gated_recurrence_forward",
                        lambda x, g, h0=None, reset=None, save=True: (x * 1, x[0] * 1, x * 1))
    x, w = torch.ones(4, 8), torch.ones(8)
    s, h0 = torch.ones(3, 2, 8), torch.ones(2, 8)
    return [(norm.layer_norm, (x, w, w.clone())),
            (recurrence.gated_recurrence, (s, s.clone(), h0))]


@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_raises(grad, monkeypatch):
    for f, args in _cases(monkeypatch):
        for i in range(3):
            with fwad.dual_level(), torch.set_grad_enabled(grad):
                dual = [fwad.make_dual(v, torch.ones_like(v)) if k == i else v
                        for k, v in enumerate(args)]
                with pytest.raises(NotImplementedError, match="forward mode"):
                    f(*dual)


def test_tensors_without_one_go_through(monkeypatch):
    for f, args in _cases(monkeypatch):
        want = f(*args)
        with fwad.dual_level():
            got = f(*args)
        for p, q in zip(want if isinstance(want, tuple) else [want],
                        got if isinstance(got, tuple) else [got]):
            assert torch.equal(p, q) and not q.requires_grad
