"""The training operators on tensors of more than 2^32 elements: what lies
beyond that offset gets the values that the same rows or ticks get on their
own.  The operators' sums do not depend on where a row lies, so norms and
losses are compared bit for bit; the recurrence is cut into other segments
there, and held to the bound of tests/test_recurrence.py."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def test_layer_norm():
    from qqt_b200.norm import layer_norm_backward, layer_norm_forward
    n, d = (1 << 32) // 2048 + 5, 2048
    x = torch.zeros((n, d), dtype=BF, device="cuda")
    x[-4:] = torch.randn((4, d), device="cuda").to(BF)
    w, b = torch.rand(d, device="cuda"), torch.rand(d, device="cuda")
    y, mean, rstd = layer_norm_forward(x, w, b)
    ys, ms, rs = layer_norm_forward(x[-4:].clone(), w, b)
    assert torch.equal(y[-4:], ys) and torch.equal(mean[-4:], ms) and torch.equal(rstd[-4:], rs)
    dy = y
    dx = layer_norm_backward(dy, x, mean, rstd, w, need_dw=False)[0]
    assert torch.equal(dx[-4:], layer_norm_backward(ys, x[-4:].clone(), ms, rs, w)[0])


def test_recurrence():
    from qqt_b200.recurrence import gated_recurrence_backward, gated_recurrence_forward
    t, d, tail = 65700, 65536, 64
    x = torch.zeros((t, 1, d), dtype=BF, device="cuda")
    g = torch.ones((t, 1, d), dtype=BF, device="cuda")
    x[-tail:] = torch.randn((tail, 1, d), device="cuda").to(BF)
    reset = torch.zeros((t, 1), dtype=torch.bool, device="cuda")
    reset[-tail] = True
    h, last, saved = gated_recurrence_forward(x, g, None, reset)
    hs, ls, ss = gated_recurrence_forward(x[-tail:].clone(), g[-tail:].clone())
    bound = 2 * 2.0 ** -8 * hs.float().abs() + 400 * 2.0 ** -24 * 5
    assert bool(((h[-tail:].float() - hs.float()).abs() <= bound).all())
    dx, dg, _ = gated_recurrence_backward(h, None, x, g, saved, reset)
    xs, gs, _ = gated_recurrence_backward(hs, None, x[-tail:].clone(), g[-tail:].clone(), ss)
    for a, b in ((dx, xs), (dg, gs)):
        # (h, the incoming gradient, may differ by a rounding: 2^-8 of its sum over a memory)
        bound = 4 * 2.0 ** -8 * b.float().abs() + 2.0 ** -8 * 5
        assert bool(((a[-tail:].float() - b.float()).abs() <= bound).all())


def test_policy_loss():
    from qqt_b200.policy_loss import policy_loss_and_grad
    n, v = 65540, 65536
    z = torch.zeros((n, v), dtype=BF, device="cuda")
    z[-4:] = 2 * torch.randn((4, v), device="cuda").to(BF)
    a = torch.randint(0, v, (n,), device="cuda")
    old = torch.full((n,), -11.0, device="cuda")
    adv = torch.ones(n, device="cuda")
    mask = torch.zeros(n, dtype=torch.bool, device="cuda")
    mask[-4:] = True
    stats, logp, dz = policy_loss_and_grad(z, a, old, adv, mask=mask, clip=100.0 / 101,
                                           entropy_coef=0.01)
    s2, l2, d2 = policy_loss_and_grad(z[-4:].clone(), a[-4:], old[-4:], adv[-4:], clip=100.0 / 101,
                                      entropy_coef=0.01)
    assert torch.equal(logp[-4:], l2) and torch.equal(dz[-4:], d2)
    assert (stats - s2).abs().max().item() <= 1e-6 * s2.abs().max().item()
    assert not dz[:4].any()
