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
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _capi as capi

_F32 = torch.float32


def _rows(t: torch.Tensor, d: int) -> torch.Tensor:
    """t as (rows, d) with a unit inner stride: a view where the layout allows
    one, else a copy."""
    if t.dim() != 2 or t.shape[1] != d:
        t = t.reshape(-1, d) if t.numel() else t.new_empty((t.numel() // d, d))
    return t if d == 1 or t.stride(1) == 1 else t.contiguous()


def _check(x, weight, bias) -> int:
    """The element type's code; raises on arguments that do not go together."""
    code = capi.DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    if weight.dtype is not _F32 or (bias is not None and bias.dtype is not _F32):
        raise TypeError("weight and bias must be float32")
    ws, nd = weight.shape, weight.dim()
    if nd < 1 or weight.numel() == 0:
        raise ValueError("weight must have at least one value")
    if x.shape[-nd:] != ws:
        raise ValueError(f"x of shape {tuple(x.shape)} does not end in {tuple(ws)}")
    if bias is not None and bias.shape != ws:
        raise ValueError("bias and weight differ in shape")
    return code


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                       eps: float = 1e-5, stats: bool = True):
    """(y, mean, rstd): y of x's shape and type, contiguous; mean and rstd
    float32, one per row (None with stats=False)."""
    code = _check(x, weight, bias)
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    stream = capi.launch_stream(x, weight, bias)
    d = weight.numel()
    xr = _rows(x, d)
    w = weight.contiguous()
    b = None if bias is None else bias.contiguous()
    n = xr.shape[0]
    y = torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
    mean = rstd = None
    if stats:
        mean = w.new_empty(n)
        rstd = torch.empty_like(mean)
    rc = capi.lib().qqt_layernorm_forward(
        xr.data_ptr(), code, n, d, xr.stride(0), w.data_ptr(), None if b is None else b.data_ptr(),
        eps, y.data_ptr(), None if mean is None else mean.data_ptr(),
        None if rstd is None else rstd.data_ptr(), stream)
    if rc:
        capi.check(rc, "qqt_layernorm_forward")
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor, need_dx: bool = True, need_dw: bool = True):
    """(dx, dweight, dbias) for dL/dy = dy; dx has x's type, dweight and dbias
    are float32 of the weight's shape (None where not needed)."""
    code = _check(x, weight, None)
    if dy.shape != x.shape or dy.dtype is not x.dtype:
        raise ValueError("dy must have x's shape and type")
    d = weight.numel()
    n = x.numel() // d
    for t in (mean, rstd):
        if t.dim() != 1 or t.shape[0] != n or t.dtype is not _F32 or not t.is_contiguous():
            raise ValueError("mean and rstd must be the forward pass's")
    stream = capi.launch_stream(x, dy, mean, rstd, weight)
    L = capi.lib()
    xr, dyr, w = _rows(x, d), _rows(dy, d), weight.contiguous()
    dx = None
    if need_dx:
        dx = torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
    dw = db = work = None
    if need_dw:
        dw, db = torch.empty_like(w), torch.empty_like(w)
        work = w.new_empty(L.qqt_layernorm_work_bytes(n, d) // 4)
    rc = L.qqt_layernorm_backward(
        dyr.data_ptr(), dyr.stride(0), xr.data_ptr(), xr.stride(0), code, n, d, mean.data_ptr(),
        rstd.data_ptr(), w.data_ptr(), capi.ptr(dx), capi.ptr(dw), capi.ptr(db), capi.ptr(work),
        stream)
    if rc:
        capi.check(rc, "qqt_layernorm_backward")
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, mean, rstd, weight)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, mean, rstd, weight = ctx.saved_tensors
        nx, nw, nb = ctx.needs_input_grad[:3]
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, nx, nw or nb)
        return dx, dw if nw else None, db if nb else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the weight's trailing
    dimensions of x; differentiable in x, weight and bias (backward mode: a
    forward-mode tangent raises NotImplementedError)."""
    # (the Function sees to tangents, which set no requires_grad)
    if (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)) \
            and torch.is_grad_enabled() or forward_ad._current_level >= 0:
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_forward(x, weight, bias, eps, False)[0]


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
