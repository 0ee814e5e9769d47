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
legal category in some head, or whose action is illegal or outside its head,
has logp -inf and adds nothing to the sums or the gradient, whatever its
other heads hold; an action outside its head also sets the device error word,
unless the mask leaves its row out.

`policy_loss` is differentiable in the logits.  `policy_loss_and_grad` gives
loss and gradient in one pass over the logits, for `logits.backward(dlogits)`.
`policy_logp` gives the log-probabilities and entropies alone.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _capi as capi


_F32 = torch.float32
_FLAGS = (torch.bool, torch.uint8)


def _args(logits, actions, legal, heads):
    """(QqtPolicyLoss, N, V, stream, tensors it points into) of the arguments
    that every entry shares; raises on those that do not go together."""
    code = capi.DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be (N, V), got {tuple(logits.shape)}")
    n, v = logits.shape
    heads = (v,) if heads is None else tuple(heads)
    nh = len(heads)
    if not 0 < nh <= capi.MAX_HEADS:
        raise ValueError(f"1 to {capi.MAX_HEADS} heads, got {nh}")
    if min(heads) <= 0 or sum(heads) != v:
        raise ValueError(f"heads {heads} do not add up to {v} logits")
    if actions.dtype is not torch.int64:
        raise TypeError("actions must be int64")
    if actions.dim() == 1:
        actions = actions[:, None]
    if actions.shape != (n, nh):
        raise ValueError(f"actions must be (N, heads) = {(n, nh)}, got {tuple(actions.shape)}")
    if legal is not None:
        if legal.dtype not in _FLAGS:
            raise TypeError("legal must be bool or uint8")
        if legal.shape != (n, v):
            raise ValueError(f"legal must be (N, V) = {(n, v)}, got {tuple(legal.shape)}")
        if v > 1 and legal.stride(1) != 1:
            legal = legal.contiguous()
    stream = capi.launch_stream(logits, actions, legal)
    if v > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    if nh > 1 and actions.stride(1) != 1:
        actions = actions.contiguous()
    a = capi.QqtPolicyLoss(logits.data_ptr(), logits.stride(0), n,
                           None if legal is None else legal.data_ptr(),
                           0 if legal is None else legal.stride(0), actions.data_ptr(),
                           actions.stride(0))
    a.dtype, a.n_heads, a.grad_scale = code, nh, 1.0
    a.width[:nh] = heads
    return a, n, v, stream, (logits, actions, legal)


def _row_values(t, n, dev, what):
    if t.dtype is not _F32:
        raise TypeError(f"{what} must be float32")
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{what} must be (N,) = {(n,)}, got {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError(f"tensors on different devices: {dev} and {t.device}")
    return t if t.stride(0) == 1 else t.contiguous()


def _loss_args(a, n, dev, old_logp, advantage, ref_logp, mask, clip, kl_coef, entropy_coef):
    """Fills in the loss's arguments; returns the tensors they point into."""
    old_logp = _row_values(old_logp, n, dev, "old_logp")
    advantage = _row_values(advantage, n, dev, "advantage")
    a.old_logp, a.adv = old_logp.data_ptr(), advantage.data_ptr()
    if ref_logp is not None:
        ref_logp = _row_values(ref_logp, n, dev, "ref_logp")
        a.ref_logp = ref_logp.data_ptr()
    elif kl_coef != 0:
        raise ValueError("a KL term needs ref_logp")
    if mask is not None:
        if mask.dtype not in _FLAGS:
            raise TypeError("mask must be bool or uint8")
        if mask.dim() != 1 or mask.shape[0] != n:
            raise ValueError(f"mask must be (N,) = {(n,)}, got {tuple(mask.shape)}")
        if mask.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {mask.device}")
        mask = mask if mask.stride(0) == 1 else mask.contiguous()
        a.mask = mask.data_ptr()
    lo, hi = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    if not (0 <= lo <= 1 and hi >= 0):
        raise ValueError(f"clip must be in [0, 1] below and not negative above: {clip}")
    a.clip_low, a.clip_high, a.kl_coef, a.entropy_coef = lo, hi, kl_coef, entropy_coef
    work = advantage.new_empty(capi.lib().qqt_policy_loss_work_bytes(n) // 4)
    a.work = work.data_ptr()
    return old_logp, advantage, ref_logp, mask, work


def _launch(a, stream):
    rc = capi.lib().qqt_policy_loss(a, stream)
    if rc:
        capi.check(rc, "qqt_policy_loss")


def policy_logp(logits: torch.Tensor, actions: torch.Tensor, legal: torch.Tensor | None = None,
                heads=None):
    """(logp, entropy), float32 (N,), of `actions` (N,) or (N, heads) int64
    under the masked heads; not differentiable."""
    a, n, _, stream, keep = _args(logits, actions, legal, heads)
    logp = logits.new_empty(n, dtype=_F32)
    ent = torch.empty_like(logp)
    a.logp, a.entropy = logp.data_ptr(), ent.data_ptr()
    _launch(a, stream)
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
    a, n, v, stream, keep = _args(logits, actions, legal, heads)
    dev = logits.device
    keep = keep, _loss_args(a, n, dev, old_logp, advantage, ref_logp, mask, clip, kl_coef,
                            entropy_coef)
    logp = logits.new_empty(n, dtype=_F32)
    stats = logp.new_empty(5)
    dz = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty((n, v))
    a.logp, a.stats, a.dlogits, a.dlogits_stride = (logp.data_ptr(), stats.data_ptr(),
                                                    dz.data_ptr(), v)
    a.grad_scale = grad_scale
    _launch(a, stream)
    return stats, logp, dz


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, old_logp, advantage, ref_logp, legal, mask, opts):
        heads, clip, kl_coef, entropy_coef = opts
        a, n, v, stream, keep = _args(logits, actions, legal, heads)
        dev = logits.device
        keep = keep, _loss_args(a, n, dev, old_logp, advantage, ref_logp, mask, clip,
                                kl_coef, entropy_coef)
        stats = logits.new_empty(5, dtype=_F32)
        a.stats = stats.data_ptr()
        _launch(a, stream)
        ctx.save_for_backward(logits, actions, old_logp, advantage, ref_logp, legal, mask)
        ctx.opts = opts
        # two outputs, no shared storage: the loss carries the gradient, the
        # statistics do not
        loss = stats[0].clone()
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        logits, actions, old_logp, advantage, ref_logp, legal, mask = ctx.saved_tensors
        heads, clip, kl_coef, entropy_coef = ctx.opts
        a, n, v, stream, keep = _args(logits, actions, legal, heads)
        dev = logits.device
        keep = keep, _loss_args(a, n, dev, old_logp, advantage, ref_logp, mask, clip,
                                kl_coef, entropy_coef)
        up = dloss.to(torch.float32).contiguous()
        dz = logits.new_empty((n, v))
        a.upstream, a.dlogits, a.dlogits_stride = up.data_ptr(), dz.data_ptr(), v
        _launch(a, stream)
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
