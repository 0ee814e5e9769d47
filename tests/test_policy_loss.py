"""Clipped policy loss, its gradient and the log-probabilities
(csrc/policy_loss.cu) against their definitions in float64.

Tolerances.  log p = z - m - log S: z - m is exact or one rounding of |z - m|,
and S, a sum of positive terms added in trees and chains of at most 64, is
off by at most 70 2^-24 of itself (exp costs 2 units), which is what log S is
off by absolutely, besides its own rounding.  So logp and entropy are held to
100 2^-24 (1 + |value| + max |z - m|) per head, a ratio to that bound times
itself, and a gradient value to u |v| + the same bound times the row's
coefficient (u: the logits' unit roundoff).  Means over rows add terms of
those errors.
"""

from __future__ import annotations

import math

import pytest
import torch

from qqt_b200 import _capi
from qqt_b200.policy_loss import policy_logp, policy_loss, policy_loss_and_grad

gpu = pytest.mark.gpu
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
C = 100 * 2.0 ** -24
OPT = dict(clip=(0.2, 0.3), kl_coef=0.05, entropy_coef=0.02)


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _ref(d, opt, grad_scale=1.0):
    z = d["logits"].double()
    legal = d.get("legal")
    legal = torch.ones(z.shape, dtype=torch.bool, device=z.device) if legal is None else legal.bool()
    n = z.shape[0]
    heads = d.get("heads") or [z.shape[1]]
    acts = d["actions"].reshape(n, -1)
    logp = torch.zeros(n, dtype=torch.float64, device=z.device)
    ent, size, at, parts = logp.clone(), logp.clone(), 0, []
    for k, w in enumerate(heads):
        lg = legal[:, at:at + w]
        zz = torch.where(lg, z[:, at:at + w], -math.inf)
        m = zz.amax(1, keepdim=True)
        m = torch.where(m == -math.inf, 0.0, m)
        e = torch.where(zz == -math.inf, 0.0, (zz - m).exp())
        s = e.sum(1, keepdim=True)
        p = torch.where(s > 0, e / s, 0.0)
        lp = zz - m - torch.log(s)
        h = -torch.where(p > 0, p * lp, 0.0).sum(1)
        logp = logp + torch.where(s[:, 0] > 0, lp.gather(1, acts[:, k:k + 1])[:, 0], -math.inf)
        ent = ent + h
        size = size + torch.where(zz == -math.inf, 0.0, (zz - m).abs()).amax(1).clamp(max=1e4)
        parts.append((p, lp, h))
        at += w
    out = {"logp": logp, "entropy": ent, "tol": C * (1 + size + logp.abs().clamp(max=1e4))}
    if "old_logp" not in d:
        return out
    lo, hi = opt["clip"]
    mask = torch.ones(n, dtype=torch.bool, device=z.device) if d.get("mask") is None \
        else d["mask"].bool()
    live = mask & (logp > -math.inf)
    lp = torch.where(live, logp, 0.0)
    a = torch.where(live, d["adv"].double(), 0.0)
    r = torch.where(live, (lp - d["old_logp"].double()).exp(), 1.0)
    pg = -torch.minimum(r * a, r.clamp(1 - lo, 1 + hi) * a)
    kl, g = torch.zeros_like(lp), torch.zeros_like(lp)
    if d.get("ref_logp") is not None:
        q = torch.where(live, d["ref_logp"].double() - lp, 0.0)
        kl = torch.expm1(q) - q
        g = -opt["kl_coef"] * torch.expm1(q)
    bound = ((a > 0) & (r > 1 + hi)) | ((a < 0) & (r < 1 - lo))
    g = g + torch.where(bound, 0.0, -a * r)
    cnt = max(1, int(mask.sum()))
    cf = ((r > 1 + hi) | (r < 1 - lo)).double()
    means = [(torch.where(live, v, 0.0)).sum() / cnt for v in (pg, kl, ent, cf)]
    out["stats"] = torch.stack([means[0] + opt["kl_coef"] * means[1]
                                - opt["entropy_coef"] * means[2]] + means)
    sc = torch.where(live, grad_scale / cnt, 0.0)[:, None]
    grads = []
    for k, (p, lpk, h) in enumerate(parts):
        one = torch.zeros_like(p).scatter_(1, acts[:, k:k + 1], 1.0)
        t = torch.where(p > 0, p * (lpk + h[:, None]), 0.0)
        grads.append(torch.where(live[:, None], sc * (g[:, None] * (one - p)
                                                      + opt["entropy_coef"] * t), 0.0))
    out["dlogits"] = torch.cat(grads, 1)
    out["coef"] = sc * (a.abs() * r + g.abs() + opt["entropy_coef"] * (1 + ent))[:, None]
    out["row_terms"] = (a.abs() * r + 1 + kl + ent)
    return out


def _data(n, v, heads, dtype, seed, legal=False, mask=True, ref=True):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(s, generator=g, device="cuda")

    def u(*s):
        return torch.rand(s, generator=g, device="cuda")

    d = {"logits": (2 * r(n, v)).to(dtype)}
    if legal:
        d["legal"] = u(n, v) < 0.5
    widths, at, acts = heads or [v], 0, []
    for w in widths:
        if legal:
            d["legal"][:, at] = True
            p = torch.where(d["legal"][:, at:at + w], u(n, w), -1.0)
        else:
            p = u(n, w)
        acts.append(p.argmax(1))
        at += w
    d["heads"] = heads
    d["actions"] = torch.stack(acts, 1)
    logp = _ref(d, OPT)["logp"].float()
    far = (0.4 + u(n)) * torch.sign(r(n))
    d["old_logp"] = logp - torch.where(u(n) < 0.2, far, 0.03 * r(n))
    d["adv"] = r(n)
    if ref:
        d["ref_logp"] = logp + 0.4 * r(n)
    if mask:
        d["mask"] = u(n) < 0.8
    return d


def _check(d, opt=OPT, grad_scale=1.0):
    dtype = d["logits"].dtype
    want = _ref(d, opt, grad_scale)
    kw = {k: d[k] for k in ("legal", "heads") if d.get(k) is not None}
    logp, ent = policy_logp(d["logits"], d["actions"], **kw)
    fine = torch.isfinite(want["logp"])
    assert torch.equal(fine, torch.isfinite(logp)) and bool((logp[~fine] == -math.inf).all())
    assert bool(((logp.double() - want["logp"])[fine].abs() <= want["tol"][fine]).all())
    assert bool(((ent.double() - want["entropy"]).abs() <= want["tol"] * 2).all())
    kw.update({k: d[k] for k in ("ref_logp", "mask") if d.get(k) is not None})
    stats, lp2, dz = policy_loss_and_grad(d["logits"], d["actions"], d["old_logp"], d["adv"],
                                          grad_scale=grad_scale, **kw, **opt)
    assert torch.equal(lp2, logp)
    tol = want["tol"][fine].max().item() if fine.any() else 0.0
    terms = want["row_terms"][torch.isfinite(want["row_terms"])]
    bound = 4 * tol * (1 + (terms.mean().item() if terms.numel() else 0.0))
    assert bool(((stats.double() - want["stats"]).abs() <= bound).all()), (stats, want["stats"])
    err = (dz.double() - want["dlogits"]).abs()
    lim = UNIT[dtype] * want["dlogits"].abs() + want["coef"] * tol
    if dtype == torch.float16:
        lim = lim + 2.0 ** -25
    assert torch.isfinite(dz).all() and bool((err <= lim).all()), (err - lim).max().item()
    return stats, logp, dz


SIZES = [(1, 1, None, False), (1, 7, [5, 2], True), (64, 7, [5, 2], True), (1000, 7, [5, 2], False),
         (333, 2, None, True), (50, 33, None, True), (129, 127, [100, 20, 7], True),
         (70, 128, None, False), (40, 1000, None, True), (31, 4099, None, False),
         (24, 8192, None, True), (9, 32001, None, False), (5, 70001, None, True),
         (3, 140000, None, False), (70001, 7, [5, 2], True), (200003, 3, None, False),
         (65, 24, [3] * 8, True), (6, 40000, [20001, 19999], True)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,v,heads,legal", SIZES)
def test_loss_gradient_and_logp_match_float64(n, v, heads, legal, dtype):
    _need_cuda()
    _check(_data(n, v, heads, dtype, n + v, legal), grad_scale=64.0 * n)
    assert _capi.device_error() == 0


@gpu
@pytest.mark.parametrize("v,heads", [(7, [5, 2]), (900, None), (20000, None)])
def test_optional_terms(v, heads):
    """No mask, no reference policy, no entropy bonus, one clip width."""
    _need_cuda()
    d = _data(60, v, heads, torch.float32, 3, mask=False, ref=False)
    opt = dict(clip=(0.2, 0.2), kl_coef=0.0, entropy_coef=0.0)
    stats, _, dz = _check(d, opt)
    again = policy_loss_and_grad(d["logits"], d["actions"], d["old_logp"], d["adv"], heads=heads)
    assert torch.equal(again[0], stats) and torch.equal(again[2], dz)


@gpu
@pytest.mark.parametrize("v,heads", [(7, [5, 2]), (200, None), (5000, None), (60000, None)])
def test_masked_places(v, heads):
    """Rows without a legal category, illegal actions, logits of -inf, of the
    type's lowest value, and NaN and infinities in illegal places or masked
    rows: they add nothing and reach nothing else."""
    _need_cuda()
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        d = _data(40, v, heads, dtype, 17, legal=True)
        d["mask"][:] = True
        d["legal"][3] = False                                  # nothing is legal
        d["legal"][4, d["actions"][4, 0]] = False              # the action is not
        d["logits"][5][~d["legal"][5]] = float("nan")
        d["logits"][6][~d["legal"][6]] = float("inf")
        d["logits"][7][~d["legal"][7]] = -math.inf
        low = torch.finfo(dtype).min
        act8 = d["actions"][8, 0]
        d["logits"][8, :] = low                                # a fill below everything
        d["logits"][8, act8] = 0.0
        d["logits"][9, :] = low                                # and nothing else: uniform
        d["logits"][10, 0] = -math.inf if int(d["actions"][10, 0]) != 0 else 0.0
        d["old_logp"][8:11] = _ref(d, OPT)["logp"][8:11].float()
        d["ref_logp"][8:11] = d["old_logp"][8:11]
        _, logp, dz = _check(d, grad_scale=64.0)
        assert logp[3] == -math.inf and logp[4] == -math.inf
        assert not dz[3].any() and not dz[4].any()
        assert not dz[~d["legal"]].any()
        # a masked row may hold anything at all
        d["mask"][[5, 11]] = False
        clean = _check(d, grad_scale=64.0)
        d["logits"][11] = float("nan")
        d["adv"][11] = float("inf")
        d["old_logp"][11] = float("nan")
        stats, _, dz = policy_loss_and_grad(
            d["logits"], d["actions"], d["old_logp"], d["adv"], d["ref_logp"], d["legal"],
            d["mask"], heads, grad_scale=64.0, **OPT)
        assert torch.equal(stats, clean[0]) and torch.equal(dz, clean[2])
        d["mask"][:] = False                                   # no row counts
        stats, _, dz = policy_loss_and_grad(
            d["logits"], d["actions"], d["old_logp"], d["adv"], d["ref_logp"], d["legal"],
            d["mask"], heads, **OPT)
        assert not stats.any() and not dz.any()
    assert _capi.device_error() == 0


@gpu
@pytest.mark.parametrize("v", [7, 300, 20000])
def test_nan_in_a_legal_place_shows(v):
    _need_cuda()
    d = _data(8, v, None, torch.float32, 2, mask=False)
    d["logits"][2, v // 2] = float("nan")
    stats, logp, dz = policy_loss_and_grad(d["logits"], d["actions"], d["old_logp"], d["adv"])
    assert logp[2].isnan() and stats[0].isnan() and dz[2].isnan().all()
    assert torch.isfinite(logp[[0, 1, 3, 4, 5, 6, 7]]).all() and torch.isfinite(dz[3:]).all()


@gpu
@pytest.mark.parametrize("v", [7, 300, 20000])
def test_action_outside_its_head(v):
    _need_cuda()
    d = _data(6, v, None, torch.float32, 4, mask=False, ref=False)
    d["actions"][1], d["actions"][4] = v, -1
    assert _capi.device_error() == 0
    stats, logp, dz = policy_loss_and_grad(d["logits"], d["actions"], d["old_logp"], d["adv"])
    torch.cuda.synchronize()
    assert _capi.device_error() == 1 << 2                      # QQT_DEV_BAD_ACTION
    assert logp[1] == -math.inf and logp[4] == -math.inf
    assert not dz[1].any() and not dz[4].any() and torch.isfinite(stats).all()


@gpu
@pytest.mark.parametrize("v,heads", [(7, [5, 2]), (130, None), (9000, None)])
def test_layouts_give_the_same_values(v, heads):
    _need_cuda()
    d = _data(37, v, heads, torch.bfloat16, 6, legal=True)
    args = [d["old_logp"], d["adv"], d["ref_logp"]]
    want = policy_loss_and_grad(d["logits"], d["actions"], *args, d["legal"], d["mask"], heads, **OPT)
    for off in (0, 1, 3):
        wide = torch.full((37, v + 5), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, off:off + v] = d["logits"]
        lw = torch.ones((37, v + 9), dtype=torch.bool, device="cuda")
        lw[:, off:off + v] = d["legal"]
        aw = torch.zeros((37, 5), dtype=torch.int64, device="cuda")
        aw[:, 1:1 + d["actions"].shape[1]] = d["actions"]
        got = policy_loss_and_grad(wide[:, off:off + v], aw[:, 1:1 + d["actions"].shape[1]], *args,
                                   lw[:, off:off + v], d["mask"].to(torch.uint8), heads, **OPT)
        assert all(torch.equal(p, q) for p, q in zip(want, got))
    got = policy_loss_and_grad(d["logits"].t().contiguous().t(), d["actions"], *args,
                               d["legal"].t().contiguous().t(), d["mask"], heads, **OPT)
    assert all(torch.equal(p, q) for p, q in zip(want, got))


@gpu
@pytest.mark.parametrize("n,v,heads", [(50, 7, [5, 2]), (20, 400, None), (6, 10000, None)])
def test_autograd_and_differences(n, v, heads):
    """policy_loss's gradient is policy_loss_and_grad's times the incoming one
    (one more rounding each), and a central difference along a random direction
    agrees: h^2 / 6 of a third derivative and the loss's rounding over h,
    1e-3 of the scale together for h = 1e-2; 5e-3 is allowed."""
    _need_cuda()
    d = _data(n, v, heads, torch.float32, 31, legal=True)
    args = (d["actions"], d["old_logp"], d["adv"], d["ref_logp"], d["legal"], d["mask"], heads)
    z = d["logits"].clone().requires_grad_(True)
    loss, stats = policy_loss(z, *args, **OPT)
    (3.0 * loss).backward()
    s2, _, dz = policy_loss_and_grad(d["logits"], *args, **OPT)
    assert torch.equal(stats, s2) and loss.item() == s2[0].item() and not stats.requires_grad
    assert bool(((z.grad - 3 * dz).abs() <= 4 * 2.0 ** -24 * (3 * dz).abs() + 1e-12).all())
    gen = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(z.shape, generator=gen, device="cuda")
    f = [_ref({**d, "logits": d["logits"].double() + s * w.double()}, OPT)["stats"][0].item()
         for s in (1e-2, -1e-2)]
    dot = dz.double() * w.double()
    num = (f[0] - f[1]) / 2e-2
    assert abs(num - dot.sum().item()) <= 5e-3 * max(dot.square().sum().sqrt().item(),
                                                      abs(dot.sum().item()))


@gpu
def test_empty_repeatable_streams_and_graphs():
    _need_cuda()
    e = torch.empty(0, device="cuda")
    stats, logp, dz = policy_loss_and_grad(torch.empty((0, 7), device="cuda"),
                                           torch.empty((0, 2), dtype=torch.int64, device="cuda"),
                                           e, e, heads=(5, 2))
    assert not stats.any() and logp.shape == (0,) and dz.shape == (0, 7)
    for n, v, heads in ((5000, 7, [5, 2]), (300, 2000, None), (200, 33000, None)):
        d = _data(n, v, heads, torch.bfloat16, 8)
        args = (d["logits"], d["actions"], d["old_logp"], d["adv"], d["ref_logp"], None, d["mask"],
                heads)
        want = policy_loss_and_grad(*args, **OPT)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(want, policy_loss_and_grad(*args, **OPT)))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = policy_loss_and_grad(*args, **OPT)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = policy_loss_and_grad(*args, **OPT)
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_refusals():
    z, a = torch.zeros(4, 7), torch.zeros((4, 2), dtype=torch.int64)
    r, m = torch.zeros(4), torch.ones(4, dtype=torch.bool)
    ok = dict(logits=z, actions=a, old_logp=r, advantage=r, heads=(5, 2), mask=m)
    for bad in (dict(logits=z.double()), dict(actions=a.int()), dict(legal=z)):
        with pytest.raises(TypeError):
            policy_loss_and_grad(**{**ok, **bad})
    for bad in (dict(logits=z[0]), dict(heads=(5, 3)), dict(heads=(7, 0)), dict(heads=(1,) * 9),
                dict(actions=a[:, 0]), dict(actions=a[:3]),
                dict(legal=torch.ones((4, 6), dtype=torch.bool))):
        with pytest.raises(ValueError):
            policy_loss_and_grad(**{**ok, **bad})
    with pytest.raises(ValueError, match="CUDA"):
        policy_loss_and_grad(**ok)
    with pytest.raises(ValueError, match="CUDA"):
        policy_logp(z, a, heads=(5, 2))


@gpu
def test_refusals_of_the_row_arguments():
    _need_cuda()
    z, a = torch.zeros((4, 7), device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    r = torch.zeros(4, device="cuda")
    ok = dict(logits=z, actions=a, old_logp=r, advantage=r)
    for bad in (dict(old_logp=r.double()), dict(mask=r)):
        with pytest.raises(TypeError):
            policy_loss_and_grad(**{**ok, **bad})
    for bad in (dict(advantage=r[:3]), dict(kl_coef=0.1), dict(clip=-0.1), dict(clip=(1.5, 0.1)),
                dict(mask=torch.ones(5, dtype=torch.bool, device="cuda")),
                dict(ref_logp=r.cpu()), dict(actions=a.cpu())):
        with pytest.raises(ValueError):
            policy_loss_and_grad(**{**ok, **bad})


def test_c_entry_refusals():
    import ctypes
    L = _capi.lib()
    P = 0x100000                 # never dereferenced

    def call(**kw):
        a = _capi.QqtPolicyLoss(logits=P, row_stride=7, rows=4, actions=P, action_stride=1,
                                old_logp=P, adv=P, logp=P, stats=P, work=P, clip_low=0.2,
                                clip_high=0.2, grad_scale=1.0, dtype=0, n_heads=1)
        a.width[0] = 7
        for k, v in kw.items():
            if k == "width":
                a.width[0] = v
            else:
                setattr(a, k, v)
        return L.qqt_policy_loss(ctypes.byref(a), None)

    assert L.qqt_policy_loss(None, None) == 1
    assert call(dtype=5) == 1 and call(rows=-1) == 1 and call(n_heads=0) == 1
    assert call(width=0) == 1 and call(logits=None) == 1 and call(actions=None) == 1
    assert call(old_logp=None) == 1 and call(adv=None) == 1 and call(work=None) == 1
    assert call(n_heads=9) == 3 and call(rows=1 << 33) == 3


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [[5, 2], [3] * 8, [60, 40], [900, 500], [20001, 19999]])
def test_head_without_a_value_beside_a_head_of_nan(heads, dtype):
    """A row is dead by any one head -- an action outside it, an illegal action,
    no legal place -- whatever the others hold: NaN or an infinity there neither
    brings it back nor reaches the sums or the rows around it.  The values of
    the other rows are those of the same batch with the row's places all
    illegal, bit for bit."""
    _need_cuda()
    v = sum(heads)
    d = _data(12, v, heads, dtype, 41, legal=True)
    d["mask"][:] = True
    ends = [sum(heads[:k + 1]) for k in range(len(heads))]
    rows = {0: ("outside", 0), 3: ("outside", 1), 4: ("illegal", 0), 6: ("empty", 1),
            9: ("outside", len(heads) - 1), 11: ("empty", 0)}
    clean = d["legal"].clone()
    clean[list(rows)] = False
    args = (d["old_logp"], d["adv"], d["ref_logp"])
    want = policy_loss_and_grad(d["logits"], d["actions"], *args, clean, d["mask"], heads, **OPT)
    for bad in (float("nan"), float("inf")):
        z, legal, acts = d["logits"].clone(), d["legal"].clone(), d["actions"].clone()
        for r, (how, k) in rows.items():
            other = (k + 1) % len(heads)
            z[r, ends[other] - heads[other] + int(acts[r, other])] = bad     # a legal place
            at = ends[k] - heads[k]
            if how == "outside":
                acts[r, k] = -1 if r % 2 else heads[k]
            elif how == "illegal":
                legal[r, at + int(acts[r, k])] = False
            else:
                legal[r, at:ends[k]] = False
        stats, logp, dz = policy_loss_and_grad(z, acts, *args, legal, d["mask"], heads, **OPT)
        lp, _ = policy_logp(z, acts, legal, heads)
        p = z.clone().requires_grad_(True)
        loss, s2 = policy_loss(p, acts, *args, legal, d["mask"], heads, **OPT)
        loss.backward()
        torch.cuda.synchronize()
        assert _capi.device_error() == 1 << 2                  # QQT_DEV_BAD_ACTION
        assert bool((logp[list(rows)] == -math.inf).all()) and torch.equal(lp, logp)
        assert not dz[list(rows)].any() and not p.grad[list(rows)].any()
        assert torch.equal(stats, want[0]) and torch.equal(s2, want[0])
        assert torch.equal(logp, want[1]) and torch.equal(dz, want[2])
        keep = [r for r in range(12) if r not in rows]
        assert torch.isfinite(p.grad[keep]).all() and torch.isfinite(stats).all()


@gpu
@pytest.mark.parametrize("v,heads", [(7, [5, 2]), (24, [3] * 8), (100, [60, 40]), (1000, None),
                                     (20000, None)])
def test_padding_actions_of_masked_rows_raise_nothing(v, heads):
    """Rows that the mask leaves out hold any action (-1, -100, the head's width,
    far out): the device error word stays clear and the counted rows' values are
    what they are without the padding.  In a counted row the same action raises."""
    _need_cuda()
    d = _data(30, v, heads, torch.float32, 23, legal=True)
    d["mask"][:] = True
    d["mask"][[0, 4, 11, 29]] = False
    args = (d["old_logp"], d["adv"], d["ref_logp"], d["legal"], d["mask"], heads)
    want = policy_loss_and_grad(d["logits"], d["actions"], *args, **OPT)
    acts = d["actions"].clone()
    acts[0], acts[4], acts[11], acts[29] = -1, -100, (heads or [v])[-1], 1 << 40
    stats, logp, dz = policy_loss_and_grad(d["logits"], acts, *args, **OPT)
    z = d["logits"].clone().requires_grad_(True)
    loss, s2 = policy_loss(z, acts, *args, **OPT)
    loss.backward()
    torch.cuda.synchronize()
    assert _capi.device_error() == 0
    assert torch.equal(stats, want[0]) and torch.equal(dz, want[2]) and torch.equal(s2, stats)
    assert torch.equal(logp[d["mask"]], want[1][d["mask"]])
    assert not z.grad[~d["mask"]].any()
    acts[7] = -1
    policy_loss_and_grad(d["logits"], acts, *args, **OPT)
    assert _capi.device_error() == 1 << 2                      # QQT_DEV_BAD_ACTION


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v,heads", [(7, [5, 2]), (40, None), (100, [60, 40]), (2000, None),
                                     (30000, None)])
def test_actions_far_below_the_maximum_keep_their_logp(v, heads, dtype):
    """An action more than 1e4 below its row's maximum, wherever that lies, down
    to the type's lowest value: log p = z - m - log S has one rounding of |z - m|
    and the bound of the other values besides.  Its ratio is 0, its gradient
    finite, also with an entropy bonus above 1."""
    _need_cuda()
    d = _data(12, v, heads, dtype, 37, ref=False, mask=False)
    low = torch.finfo(dtype).min
    half = dtype == torch.float16
    tops = [0.0, 0.0, -3.2e4, -3.2e4, 5e4, 3.0e4] if half else [0.0, 0.0, -3e6, 3e6, -5e29, 2e7]
    below = [low, -6.0e4, -6.5e4, low, -2e4, -2.5e4] if half \
        else [low, -2e30, -4e6, -3e6, -2e30, low]
    at = 0
    for k, w in enumerate(heads or [v]):
        for r, (top, act) in enumerate(zip(tops, below)):
            z = torch.full((w,), top, device="cuda") - torch.rand(w, device="cuda")
            z[d["actions"][r, k]] = act
            d["logits"][r, at:at + w] = z.to(dtype)
        at += w
    want = _ref(d, OPT)["logp"]
    assert bool((want[:6] < -1e4).all())
    logp, ent = policy_logp(d["logits"], d["actions"], heads=heads)
    # two heads at the lowest value: beyond float32, which holds -inf there
    past = torch.isinf(want.float())
    assert bool((logp[past] == -math.inf).all()) and (len(heads or [v]) > 1 or not past.any())
    assert bool(((logp.double() - want).abs() <= C * (1 + want.abs()))[~past].all()), (logp, want)
    assert torch.isfinite(ent).all()
    stats, lp2, dz = policy_loss_and_grad(d["logits"], d["actions"], want.float(), d["adv"],
                                          heads=heads, clip=0.2, entropy_coef=2.0)
    assert torch.equal(lp2, logp) and torch.isfinite(dz).all()
    assert _capi.device_error() == 0


@gpu
@pytest.mark.parametrize("v,heads", [(7, [5, 2]), (300, None), (20000, None)])
def test_advantage_of_zero_beside_a_ratio_beyond_float32(v, heads):
    """exp(logp - old) of 200 is a number in 64 bits, and 0 of it is 0: the row
    adds its entropy and nothing else, in the loss and in the gradient alike.  A
    NaN ratio is not hidden by the advantage."""
    _need_cuda()
    d = _data(9, v, heads, torch.float32, 19, ref=False, mask=False)
    d["adv"][2], d["adv"][5] = 0.0, -0.0
    d["old_logp"][[2, 5]] -= 200.0
    opt = dict(clip=(0.2, 0.3), kl_coef=0.0, entropy_coef=0.02)
    _check(d, opt)
    p = d["logits"].clone().requires_grad_(True)
    loss, stats = policy_loss(p, d["actions"], d["old_logp"], d["adv"], heads=heads, **opt)
    loss.backward()
    assert torch.isfinite(stats).all() and torch.isfinite(p.grad).all()
    d["old_logp"][2] = float("nan")
    stats, _, dz = policy_loss_and_grad(d["logits"], d["actions"], d["old_logp"], d["adv"],
                                        heads=heads, **opt)
    assert stats[1].isnan() and dz[2].isnan().all() and torch.isfinite(dz[5]).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,v,heads", [(50, 7, [5, 2]), (300, 120, [100, 20]), (20, 3000, None),
                                       (6, 40001, None)])
def test_autograd_in_16_bits(n, v, heads, dtype):
    """The autograd loss and its scaled gradient against float64 (the scale's
    product is one more rounding), the scaled loss as mixed precision trains."""
    _need_cuda()
    d = _data(n, v, heads, dtype, n + v, legal=True)
    scale = 64.0 * n
    want = _ref(d, OPT, scale)
    z = d["logits"].clone().requires_grad_(True)
    loss, stats = policy_loss(z, d["actions"], d["old_logp"], d["adv"], d["ref_logp"], d["legal"],
                              d["mask"], heads, **OPT)
    (scale * loss).backward()
    assert z.grad.dtype == dtype and loss.dtype == torch.float32
    tol = want["tol"].max().item()
    terms = want["row_terms"].mean().item()
    assert bool(((stats.double() - want["stats"]).abs() <= 4 * tol * (1 + terms)).all())
    err = (z.grad.double() - want["dlogits"]).abs()
    lim = UNIT[dtype] * want["dlogits"].abs() + want["coef"] * tol + 2.0 ** -25
    assert bool((err <= lim).all()), (err - lim).max().item()


@gpu
@pytest.mark.parametrize("n,v", [(1000003, 40), (300007, 64)])
def test_many_rows_of_moderate_width(n, v):
    """Means over a million rows: a thread adds n / 1024 of the rows' terms one
    after the other and trees the rest, so a sum is off by at most (n / 1024 + 20)
    2^-24 of its terms' magnitudes, besides the rows' own errors."""
    _need_cuda()
    d = _data(n, v, None, torch.float32, 71)
    want = _ref(d, OPT)
    stats, logp, dz = policy_loss_and_grad(d["logits"], d["actions"], d["old_logp"], d["adv"],
                                           d["ref_logp"], None, d["mask"], **OPT)
    assert bool(((logp.double() - want["logp"]).abs() <= want["tol"]).all())
    bound = (want["row_terms"] * (4 * want["tol"] + (n / 1024 + 20) * 2.0 ** -24)).mean().item()
    assert bool(((stats.double() - want["stats"]).abs() <= bound / 0.7).all()), \
        (stats, want["stats"], bound)
    err = (dz.double() - want["dlogits"]).abs()
    lim = UNIT[torch.float32] * want["dlogits"].abs() + want["coef"] * want["tol"][:, None]
    assert bool((err <= lim).all())
