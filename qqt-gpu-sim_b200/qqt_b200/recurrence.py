"""Gated linear recurrence on the kernels of csrc/recurrence.cu: a policy's
memory over the ticks of a rollout, or any long sequence.

    f = sigmoid(gate_t)
    h_t = f * (0 if reset_t else h_{t-1}) + (1 - f) * x_t

Sequences are time-major (T, N, D), as the rollout buffers are; a batch-first
tensor goes in as its `transpose(0, 1)` view, and so do the halves of one
wider projection: any strides with a unit innermost one are read in place.
x and gate are float32, float16 or bfloat16; states (h0, the last state and
what the backward pass recomputes) are float32.

`gated_recurrence` is differentiable; `gated_recurrence_forward` and
`gated_recurrence_backward` are its two halves; `gated_recurrence_step` is
one tick, for acting.
"""

from __future__ import annotations

import ctypes

import torch

from . import _capi as capi


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _seq(t: torch.Tensor | None):
    return None if t is None else ctypes.byref(capi.QqtSeq(t.data_ptr(), t.stride(0), t.stride(1)))


def _like(x: torch.Tensor) -> torch.Tensor:
    """An empty (T, N, D) in x's order: batch-first where x's time steps lie
    closer together than its sequences."""
    t, n, d = x.shape
    if t > 1 and n > 1 and x.stride(0) < x.stride(1):
        return torch.empty((n, t, d), dtype=x.dtype, device=x.device).transpose(0, 1)
    return torch.empty((t, n, d), dtype=x.dtype, device=x.device)


def _check(x, gate, h0, reset):
    capi.need(x.dtype in capi.DTYPES, f"x must be float32, float16 or bfloat16, got {x.dtype}",
              TypeError)
    capi.need(gate.dtype == x.dtype, "gate must have x's type", TypeError)
    capi.need(x.dim() == 3 and x.shape[2] > 0 and gate.shape == x.shape,
              f"x and gate must be (T, N, D) alike, got {tuple(x.shape)} and {tuple(gate.shape)}")
    _check_state(h0, x.shape[1:], "h0")
    if reset is not None:
        capi.need(reset.dtype in (torch.bool, torch.uint8), "reset must be bool or uint8",
                  TypeError)
        capi.need(reset.shape == x.shape[:2],
                  f"reset must be (T, N) = {tuple(x.shape[:2])}, got {tuple(reset.shape)}")


def _check_state(s, shape, what):
    if s is not None:
        capi.need(s.dtype == torch.float32, f"{what} must be float32", TypeError)
        capi.need(s.shape == shape, f"{what} must be (N, D) = {tuple(shape)}, got {tuple(s.shape)}")


def _work(L, t, n, d, dev):
    return torch.empty(int(L.qqt_recurrence_work_bytes(t, n, d)), dtype=torch.uint8, device=dev)


def gated_recurrence_forward(x: torch.Tensor, gate: torch.Tensor, h0: torch.Tensor | None = None,
                             reset: torch.Tensor | None = None, save: bool = True):
    """(h, h_last, saved): h (T, N, D) of x's type and order, h_last (N, D)
    float32, saved (chunks, N, D) float32 for `gated_recurrence_backward`
    (None with save=False).  h0 None is zero; reset (T, N) drops the state
    that would enter a tick."""
    _check(x, gate, h0, reset)
    capi.need_cuda(x, gate, h0, reset)
    t, n, d = x.shape
    dev, L = x.device, capi.lib()
    x, gate = _unit(x), _unit(gate)
    h0 = None if h0 is None else h0.contiguous()
    h = _like(x)
    last = torch.empty((n, d), dtype=torch.float32, device=dev)
    saved = None
    if save:
        saved = torch.empty((int(L.qqt_recurrence_chunks(t)), n, d), dtype=torch.float32,
                            device=dev)
    work = _work(L, t, n, d, dev)
    capi.check(L.qqt_recurrence_forward(
        _seq(x), _seq(gate), _seq(reset), capi.ptr(h0), capi.DTYPES[x.dtype], t, n, d, _seq(h),
        last.data_ptr(), capi.ptr(saved), work.data_ptr(), capi.stream_ptr(dev)),
        "qqt_recurrence_forward")
    return h, last, saved


def gated_recurrence_backward(dh: torch.Tensor | None, dh_last: torch.Tensor | None,
                              x: torch.Tensor, gate: torch.Tensor, saved: torch.Tensor,
                              reset: torch.Tensor | None = None):
    """(dx, dgate, dh0) for dL/dh = dh and dL/dh_last = dh_last (either may be
    None, zero); saved is the forward pass's."""
    _check(x, gate, None, reset)
    t, n, d = x.shape
    _check_state(dh_last, x.shape[1:], "dh_last")
    capi.need(dh is None or (dh.shape == x.shape and dh.dtype == x.dtype),
              "dh must have x's shape and type")
    L = capi.lib()
    capi.need(saved is not None and saved.dtype == torch.float32 and saved.is_contiguous()
              and saved.shape == (int(L.qqt_recurrence_chunks(t)), n, d),
              "saved must be the forward pass's")
    capi.need_cuda(x, gate, saved, dh, dh_last, reset)
    dev = x.device
    x, gate = _unit(x), _unit(gate)
    dh = None if dh is None else _unit(dh)
    dh_last = None if dh_last is None else dh_last.contiguous()
    dx, dg = _like(x), _like(x)
    dh0 = torch.empty((n, d), dtype=torch.float32, device=dev)
    work = _work(L, t, n, d, dev)
    capi.check(L.qqt_recurrence_backward(
        _seq(dh), capi.ptr(dh_last), _seq(x), _seq(gate), _seq(reset), saved.data_ptr(),
        capi.DTYPES[x.dtype], t, n, d, _seq(dx), _seq(dg), dh0.data_ptr(), work.data_ptr(),
        capi.stream_ptr(dev)), "qqt_recurrence_backward")
    return dx, dg, dh0


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, reset):
        h, last, saved = gated_recurrence_forward(x, gate, h0, reset)
        ctx.save_for_backward(x, gate, saved, reset)
        ctx.has_h0 = h0 is not None
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    def backward(ctx, dh, dh_last):
        x, gate, saved, reset = ctx.saved_tensors
        dx, dg, dh0 = gated_recurrence_backward(dh, dh_last, x, gate, saved, reset)
        return dx, dg, dh0 if ctx.has_h0 else None, None


def gated_recurrence(x: torch.Tensor, gate: torch.Tensor, h0: torch.Tensor | None = None,
                     reset: torch.Tensor | None = None):
    """(h, h_last) of the recurrence over x, gate (T, N, D); differentiable in
    x, gate and h0."""
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad
                                    or (h0 is not None and h0.requires_grad)):
        return _Recurrence.apply(x, gate, h0, reset)
    return gated_recurrence_forward(x, gate, h0, reset, save=False)[:2]


def gated_recurrence_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor,
                          reset: torch.Tensor | None = None,
                          state_out: torch.Tensor | None = None):
    """One tick: (h, new state) for x, gate (N, D), state (N, D) float32 and
    reset (N,).  state_out receives the new state (it may be `state` itself:
    the rollout's in-place form); by default it is a new tensor."""
    capi.need(x.dim() == 2, f"x must be (N, D), got {tuple(x.shape)}")
    x3, g3 = x[None], gate[None]
    r2 = None if reset is None else reset[None]
    _check(x3, g3, state, r2)
    capi.need(state is not None and state.is_contiguous(), "state must be contiguous")
    _check_state(state_out, x.shape, "state_out")
    capi.need(state_out is None or state_out.is_contiguous(), "state_out must be contiguous")
    capi.need_cuda(x, gate, state, reset, state_out)
    n, d = x.shape
    dev, L = x.device, capi.lib()
    x3, g3 = _unit(x3), _unit(g3)
    h = torch.empty((1, n, d), dtype=x.dtype, device=dev)
    out = torch.empty_like(state) if state_out is None else state_out
    work = _work(L, 1, n, d, dev)
    capi.check(L.qqt_recurrence_forward(
        _seq(x3), _seq(g3), _seq(r2), state.data_ptr(), capi.DTYPES[x.dtype], 1, n, d, _seq(h),
        out.data_ptr(), None, work.data_ptr(), capi.stream_ptr(dev)), "qqt_recurrence_forward")
    return h[0], out
