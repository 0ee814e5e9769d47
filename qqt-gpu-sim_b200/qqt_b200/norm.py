"""Layer norm on the kernels of csrc/layer_norm.cu, forward and backward.

`layer_norm` is differentiable; `layer_norm_forward` and
`layer_norm_backward` are its two halves for training loops that keep their
own graph.  The normalised dimensions are the weight's: (128,) for the MLP's
norms, (C, H, W) for the CNN's.  x and dy are float32, float16 or bfloat16,
with any row stride; weight and bias are float32 (the framework's parameters
are), as are all statistics and sums.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import _capi as capi


def _rows(t: torch.Tensor, d: int):
    """t as (rows, d) with a unit inner stride: a view where the layout allows
    one, else a copy."""
    r = t.reshape(-1, d) if t.numel() else t.new_empty((t.numel() // d, d))
    if d > 1 and r.stride(1) != 1:
        r = r.contiguous()
    return r


def _check(x, weight, bias, what="x"):
    capi.need(x.dtype in capi.DTYPES, f"{what} must be float32, float16 or bfloat16, got {x.dtype}",
              TypeError)
    capi.need(weight.dtype == torch.float32 and (bias is None or bias.dtype == torch.float32),
              "weight and bias must be float32", TypeError)
    nd = weight.dim()
    capi.need(nd >= 1 and weight.numel() > 0, "weight must have at least one value")
    capi.need(x.dim() >= nd and x.shape[x.dim() - nd:] == weight.shape,
              f"{what} of shape {tuple(x.shape)} does not end in {tuple(weight.shape)}")
    capi.need(bias is None or bias.shape == weight.shape, "bias and weight differ in shape")


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                       eps: float = 1e-5, stats: bool = True):
    """(y, mean, rstd): y of x's shape and type, contiguous; mean and rstd
    float32, one per row (None with stats=False)."""
    _check(x, weight, bias)
    capi.need(eps >= 0, "eps must not be negative")
    capi.need_cuda(x, weight, bias)
    d = weight.numel()
    xr = _rows(x, d)
    w = weight.contiguous()
    b = None if bias is None else bias.contiguous()
    n = xr.shape[0]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty((2, n), dtype=torch.float32, device=x.device)
    capi.check(capi.lib().qqt_layernorm_forward(
        xr.data_ptr(), capi.DTYPES[x.dtype], n, d, xr.stride(0), w.data_ptr(), capi.ptr(b), eps,
        y.data_ptr(), capi.ptr(mean), capi.ptr(rstd), capi.stream_ptr(x.device)),
        "qqt_layernorm_forward")
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor, need_dx: bool = True, need_dw: bool = True):
    """(dx, dweight, dbias) for dL/dy = dy; dx has x's type, dweight and dbias
    are float32 of the weight's shape (None where not needed)."""
    _check(x, weight, None)
    capi.need(dy.shape == x.shape and dy.dtype == x.dtype, "dy must have x's shape and type")
    d = weight.numel()
    n = x.numel() // d
    capi.need(mean.shape == (n,) and rstd.shape == (n,) and mean.dtype == torch.float32
              and rstd.dtype == torch.float32 and mean.is_contiguous() and rstd.is_contiguous(),
              "mean and rstd must be the forward pass's")
    capi.need_cuda(x, dy, mean, rstd, weight)
    xr, dyr, w = _rows(x, d), _rows(dy, d), weight.contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_dx else None
    dw = db = work = None
    L = capi.lib()
    if need_dw:
        dw, db = torch.empty((2,) + tuple(weight.shape), dtype=torch.float32, device=x.device)
        work = torch.empty(int(L.qqt_layernorm_work_bytes(n, d)), dtype=torch.uint8,
                           device=x.device)
    capi.check(L.qqt_layernorm_backward(
        dyr.data_ptr(), dyr.stride(0), xr.data_ptr(), xr.stride(0), capi.DTYPES[x.dtype], n, d,
        mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), capi.ptr(dx), capi.ptr(dw), capi.ptr(db),
        capi.ptr(work), capi.stream_ptr(x.device)), "qqt_layernorm_backward")
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, mean, rstd, weight)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, mean, rstd, weight = ctx.saved_tensors
        nx, nw, nb = ctx.needs_input_grad[:3]
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, nx, nw or nb)
        return dx, dw if nw else None, db if nb else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the weight's trailing
    dimensions of x; differentiable in x, weight and bias."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_forward(x, weight, bias, eps, stats=False)[0]


class LayerNorm(nn.Module):
    """nn.LayerNorm's parameters and state_dict keys on `layer_norm`."""

    def __init__(self, normalized_shape, eps: float = 1e-5):
        super().__init__()
        shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
        self.weight = nn.Parameter(torch.ones(shape))
        self.bias = nn.Parameter(torch.zeros(shape))
        self.eps = eps

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)
