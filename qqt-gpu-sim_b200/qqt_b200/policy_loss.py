"""Clipped policy loss with a KL term and an entropy bonus, on the kernels of
csrc/policy_loss.cu, straight from the logits: no log-softmax is stored.

    logp = sum over heads of log softmax(logits over the legal)[action]
    r = exp(logp - old_logp),  q = ref_logp - logp
    loss = mean over the rows of `mask` of
           -min(r A, clip(r, 1 - lo, 1 + hi) A)
           + kl_coef (exp(q) - 1 - q) - entropy_coef H

(train/ppo.py:397-424, train/model.py:216-256).  logits (N, V) are float32,
float16 or bfloat16; `heads` splits V into independent categorical heads
((5, 2): the moves and the bomb), one head by default.  A row without a
legal category in some head, or whose action is not legal, has logp -inf and
adds nothing to the sums or the gradient.

`policy_loss` is differentiable in the logits.  `policy_loss_and_grad` gives
loss and gradient in one pass over the logits, for `logits.backward(dlogits)`.
`policy_logp` gives the log-probabilities and entropies alone.
"""

from __future__ import annotations

import torch

from . import _capi as capi


def _bytes(t: torch.Tensor) -> torch.Tensor:
    return t.view(torch.uint8) if t.dtype == torch.bool else t


def _args(logits, actions, legal, heads):
    """Checked arguments shared by every entry: a filled QqtPolicyLoss and the
    tensors it points into."""
    capi.need(logits.dtype in capi.DTYPES,
              f"logits must be float32, float16 or bfloat16, got {logits.dtype}", TypeError)
    capi.need(logits.dim() == 2 and logits.shape[1] > 0,
              f"logits must be (N, V), got {tuple(logits.shape)}")
    n, v = logits.shape
    heads = (v,) if heads is None else tuple(int(w) for w in heads)
    capi.need(0 < len(heads) <= capi.MAX_HEADS, f"1 to {capi.MAX_HEADS} heads, got {len(heads)}")
    capi.need(min(heads) > 0 and sum(heads) == v, f"heads {heads} do not add up to {v} logits")
    capi.need(actions.dtype == torch.int64, "actions must be int64", TypeError)
    if actions.dim() == 1:
        actions = actions[:, None]
    capi.need(actions.shape == (n, len(heads)),
              f"actions must be (N, heads) = {(n, len(heads))}, got {tuple(actions.shape)}")
    if legal is not None:
        capi.need(legal.dtype in (torch.bool, torch.uint8), "legal must be bool or uint8", TypeError)
        capi.need(legal.shape == (n, v), f"legal must be (N, V), got {tuple(legal.shape)}")
        legal = _bytes(legal)
        if v > 1 and legal.stride(1) != 1:
            legal = legal.contiguous()
    capi.need_cuda(logits, actions, legal)
    if v > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    if len(heads) > 1 and actions.stride(1) != 1:
        actions = actions.contiguous()
    a = capi.QqtPolicyLoss(logits.data_ptr(), logits.stride(0), n, capi.ptr(legal),
                           0 if legal is None else legal.stride(0), actions.data_ptr(),
                           actions.stride(0))
    a.dtype, a.n_heads = capi.DTYPES[logits.dtype], len(heads)
    a.width[:len(heads)] = heads
    a.grad_scale = 1.0
    return a, (logits, actions, legal)


def _loss_args(a, n, dev, old_logp, advantage, ref_logp, mask, clip, kl_coef, entropy_coef):
    keep = []
    for name, field, t in (("old_logp", "old_logp", old_logp), ("advantage", "adv", advantage),
                           ("ref_logp", "ref_logp", ref_logp)):
        if t is None and name == "ref_logp":
            capi.need(kl_coef == 0, "a KL term needs ref_logp")
            continue
        capi.need(t.dtype == torch.float32, f"{name} must be float32", TypeError)
        capi.need(t.shape == (n,), f"{name} must be (N,) = {(n,)}, got {tuple(t.shape)}")
        t = t.contiguous()
        setattr(a, field, t.data_ptr())
        keep.append(t)
    if mask is not None:
        capi.need(mask.dtype in (torch.bool, torch.uint8), "mask must be bool or uint8", TypeError)
        capi.need(mask.shape == (n,), f"mask must be (N,) = {(n,)}, got {tuple(mask.shape)}")
        mask = _bytes(mask).contiguous()
        a.mask = mask.data_ptr()
        keep.append(mask)
    lo, hi = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    capi.need(0 <= lo <= 1 and hi >= 0, f"clip must be in [0, 1] below and not negative above: {clip}")
    a.clip_low, a.clip_high, a.kl_coef, a.entropy_coef = lo, hi, kl_coef, entropy_coef
    for t in keep:
        capi.need(t.device == dev, f"tensors on different devices: {dev} and {t.device}")
    work = torch.empty(int(capi.lib().qqt_policy_loss_work_bytes(n)), dtype=torch.uint8, device=dev)
    a.work = work.data_ptr()
    return keep + [work]


def _launch(a, dev):
    capi.check(capi.lib().qqt_policy_loss(a, capi.stream_ptr(dev)), "qqt_policy_loss")


def policy_logp(logits: torch.Tensor, actions: torch.Tensor, legal: torch.Tensor | None = None,
                heads=None):
    """(logp, entropy), float32 (N,), of `actions` (N,) or (N, heads) int64
    under the masked heads; not differentiable."""
    a, keep = _args(logits, actions, legal, heads)
    logp, ent = torch.empty((2, logits.shape[0]), dtype=torch.float32, device=logits.device)
    a.logp, a.entropy = logp.data_ptr(), ent.data_ptr()
    _launch(a, logits.device)
    return logp, ent


def policy_loss_and_grad(logits: torch.Tensor, actions: torch.Tensor, old_logp: torch.Tensor,
                         advantage: torch.Tensor, ref_logp: torch.Tensor | None = None,
                         legal: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                         heads=None, clip=0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0,
                         grad_scale: float = 1.0):
    """(stats, logp, dlogits): stats (5,) float32 = loss and the means of the
    policy term, KL, entropy and clipped share over the rows of `mask`; logp
    (N,); dlogits (N, V) of the logits' type = grad_scale * dloss/dlogits
    (grad_scale: the loss scaling of float16 training).  clip: one width or
    (below, above)."""
    a, keep = _args(logits, actions, legal, heads)
    n, v = logits.shape
    dev = logits.device
    keep = keep, _loss_args(a, n, dev, old_logp, advantage, ref_logp, mask, clip, kl_coef,
                            entropy_coef)
    logp = torch.empty(n, dtype=torch.float32, device=dev)
    stats = torch.empty(5, dtype=torch.float32, device=dev)
    dz = torch.empty((n, v), dtype=logits.dtype, device=dev)
    a.logp, a.stats, a.dlogits, a.dlogits_stride = (logp.data_ptr(), stats.data_ptr(),
                                                    dz.data_ptr(), v)
    a.grad_scale = grad_scale
    _launch(a, dev)
    return stats, logp, dz


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, old_logp, advantage, ref_logp, legal, mask, opts):
        heads, clip, kl_coef, entropy_coef = opts
        a, keep = _args(logits, actions, legal, heads)
        dev = logits.device
        keep = keep, _loss_args(a, logits.shape[0], dev, old_logp, advantage, ref_logp, mask, clip,
                                kl_coef, entropy_coef)
        stats = torch.empty(5, dtype=torch.float32, device=dev)
        a.stats = stats.data_ptr()
        _launch(a, dev)
        ctx.save_for_backward(logits, actions, old_logp, advantage, ref_logp, legal, mask)
        ctx.opts = opts
        # two outputs, no shared storage: the loss carries the gradient, the
        # statistics do not
        loss = stats[0].clone()
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    def backward(ctx, dloss, _):
        logits, actions, old_logp, advantage, ref_logp, legal, mask = ctx.saved_tensors
        heads, clip, kl_coef, entropy_coef = ctx.opts
        a, keep = _args(logits, actions, legal, heads)
        dev = logits.device
        keep = keep, _loss_args(a, logits.shape[0], dev, old_logp, advantage, ref_logp, mask, clip,
                                kl_coef, entropy_coef)
        up = dloss.to(torch.float32).contiguous()
        dz = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        a.upstream, a.dlogits, a.dlogits_stride = up.data_ptr(), dz.data_ptr(), logits.shape[1]
        _launch(a, dev)
        return dz, None, None, None, None, None, None, None


def policy_loss(logits: torch.Tensor, actions: torch.Tensor, old_logp: torch.Tensor,
                advantage: torch.Tensor, ref_logp: torch.Tensor | None = None,
                legal: torch.Tensor | None = None, mask: torch.Tensor | None = None, heads=None,
                clip=0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0):
    """(loss, stats): the loss, differentiable in the logits, and the (5,)
    statistics of `policy_loss_and_grad`.  The backward pass reads the logits
    again instead of keeping a gradient of their size."""
    return _PolicyLoss.apply(logits, actions, old_logp, advantage, ref_logp, legal, mask,
                             (heads, clip, kl_coef, entropy_coef))
