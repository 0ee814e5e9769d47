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
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _capi as capi


_F32 = torch.float32
_FLAGS = (torch.bool, torch.uint8)


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _like(x: torch.Tensor) -> torch.Tensor:
    """An output of x's shape and type, dense and with a unit innermost stride:
    in the order of x's strides where that leaves D innermost.  (It need not
    where x overlaps itself, as sliding windows do: several strides are 1.)"""
    out = torch.empty_like(x)
    return out if x.shape[-1] <= 1 or out.stride(-1) == 1 else x.new_empty(x.shape)


def _seqs(*tensors):
    """The tensors as one array of QqtSeq and its entries' addresses (None for
    a tensor that is None); the array has to live until the call is done."""
    v = []
    for t in tensors:
        if t is None:
            v += (0, 0, 0)
        else:
            st = t.stride()
            v += (t.data_ptr(), st[0], st[1])
    a = (ctypes.c_int64 * len(v))(*v)
    base = ctypes.addressof(a)
    return a, [None if t is None else base + 24 * i for i, t in enumerate(tensors)]


def _check(x, gate, state, reset, dims, what) -> int:
    """The element type's code; raises on arguments that do not go together.
    dims: x's dimensions (3, or 2 for one tick)."""
    code = capi.DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    if gate.dtype is not x.dtype:
        raise TypeError("gate must have x's type")
    shape = x.shape
    if len(shape) != dims or shape[-1] == 0 or gate.shape != shape:
        raise ValueError(f"x and gate must be {'(T, N, D)' if dims == 3 else '(N, D)'} alike, got "
                         f"{tuple(shape)} and {tuple(gate.shape)}")
    if state is not None:
        if state.dtype is not _F32:
            raise TypeError(f"{what} must be float32")
        if state.shape != shape[-2:]:
            raise ValueError(f"{what} must be (N, D) = {tuple(shape[-2:])}, got "
                             f"{tuple(state.shape)}")
    if reset is not None:
        if reset.dtype not in _FLAGS:
            raise TypeError("reset must be bool or uint8")
        if reset.shape != shape[:-1]:
            raise ValueError(f"reset must be {tuple(shape[:-1])}, got {tuple(reset.shape)}")
    return code


def _work(L, t, n, d, like):
    """(tensor, address) of the workspace, (None, None) where none is needed."""
    nb = L.qqt_recurrence_work_bytes(t, n, d)
    if nb == 0:
        return None, None
    w = like.new_empty(nb // 4)
    return w, w.data_ptr()


def gated_recurrence_forward(x: torch.Tensor, gate: torch.Tensor, h0: torch.Tensor | None = None,
                             reset: torch.Tensor | None = None, save: bool = True):
    """(h, h_last, saved): h (T, N, D) of x's type and order, h_last (N, D)
    float32, saved (chunks, N, D) float32 for `gated_recurrence_backward`
    (None with save=False).  h0 None is zero; reset (T, N) drops the state
    that would enter a tick."""
    code = _check(x, gate, h0, reset, 3, "h0")
    stream = capi.launch_stream(x, gate, h0, reset)
    t, n, d = x.shape
    L = capi.lib()
    x, gate = _unit(x), _unit(gate)
    h0 = None if h0 is None else h0.contiguous()
    h = _like(x)
    last = x.new_empty((n, d), dtype=_F32)
    saved = last.new_empty((L.qqt_recurrence_chunks(t), n, d)) if save else None
    work, wp = _work(L, t, n, d, last)
    keep, (xs, gs, rs, hs) = _seqs(x, gate, reset, h)
    rc = L.qqt_recurrence_forward(xs, gs, rs, None if h0 is None else h0.data_ptr(), code, t, n, d,
                                  hs, last.data_ptr(), capi.ptr(saved), wp, stream)
    if rc:
        capi.check(rc, "qqt_recurrence_forward")
    return h, last, saved


def gated_recurrence_backward(dh: torch.Tensor | None, dh_last: torch.Tensor | None,
                              x: torch.Tensor, gate: torch.Tensor, saved: torch.Tensor,
                              reset: torch.Tensor | None = None):
    """(dx, dgate, dh0) for dL/dh = dh and dL/dh_last = dh_last (either may be
    None, zero); saved is the forward pass's."""
    code = _check(x, gate, dh_last, reset, 3, "dh_last")
    t, n, d = x.shape
    if dh is not None and (dh.shape != x.shape or dh.dtype is not x.dtype):
        raise ValueError("dh must have x's shape and type")
    L = capi.lib()
    if saved is None or saved.dtype is not _F32 or not saved.is_contiguous() \
            or saved.shape != (L.qqt_recurrence_chunks(t), n, d):
        raise ValueError("saved must be the forward pass's")
    stream = capi.launch_stream(x, gate, saved, dh, dh_last, reset)
    x, gate = _unit(x), _unit(gate)
    dh = None if dh is None else _unit(dh)
    dh_last = None if dh_last is None else dh_last.contiguous()
    dx, dg = _like(x), _like(x)
    dh0 = saved.new_empty((n, d))
    work, wp = _work(L, t, n, d, saved)
    keep, (hs, xs, gs, rs, dxs, dgs) = _seqs(dh, x, gate, reset, dx, dg)
    rc = L.qqt_recurrence_backward(hs, capi.ptr(dh_last), xs, gs, rs, saved.data_ptr(), code, t, n,
                                   d, dxs, dgs, dh0.data_ptr(), wp, stream)
    if rc:
        capi.check(rc, "qqt_recurrence_backward")
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
    @once_differentiable
    def backward(ctx, dh, dh_last):
        x, gate, saved, reset = ctx.saved_tensors
        dx, dg, dh0 = gated_recurrence_backward(dh, dh_last, x, gate, saved, reset)
        return dx, dg, dh0 if ctx.has_h0 else None, None


def gated_recurrence(x: torch.Tensor, gate: torch.Tensor, h0: torch.Tensor | None = None,
                     reset: torch.Tensor | None = None):
    """(h, h_last) of the recurrence over x, gate (T, N, D); differentiable in
    x, gate and h0 (backward mode: a forward-mode tangent raises
    NotImplementedError)."""
    # (the Function sees to tangents, which set no requires_grad)
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (
            x.requires_grad or gate.requires_grad or (h0 is not None and h0.requires_grad)):
        return _Recurrence.apply(x, gate, h0, reset)
    return gated_recurrence_forward(x, gate, h0, reset, save=False)[:2]


def gated_recurrence_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor,
                          reset: torch.Tensor | None = None,
                          state_out: torch.Tensor | None = None):
    """One tick: (h, new state) for x, gate (N, D), state (N, D) float32 and
    reset (N,).  state_out receives the new state; it may be `state` itself
    (the rollout's in-place form) and overlaps no operand otherwise.  By default
    it is a new tensor.  Not differentiable."""
    code = _check(x, gate, state, reset, 2, "state")
    if state is None or not state.is_contiguous():
        raise ValueError("state must be contiguous")
    if state_out is None:
        out = torch.empty_like(state)
    elif state_out.dtype is not _F32:
        raise TypeError("state_out must be float32")
    elif state_out.shape != state.shape or not state_out.is_contiguous():
        raise ValueError(f"state_out must be a contiguous {tuple(state.shape)}")
    else:
        out = state_out
    stream = capi.launch_stream(x, gate, state, reset, out)
    n, d = x.shape
    x, gate = _unit(x), _unit(gate)
    h = x.new_empty((n, d))
    rc = capi.lib().qqt_recurrence_step(
        x.data_ptr(), x.stride(0), gate.data_ptr(), gate.stride(0),
        None if reset is None else reset.data_ptr(), 0 if reset is None else reset.stride(0),
        state.data_ptr(), code, n, d, h.data_ptr(), out.data_ptr(), stream)
    if rc:
        if rc == 1 and state_out is not None:      # (the entry's one refusal left)
            raise ValueError("state_out overlaps an operand")
        capi.check(rc, "qqt_recurrence_step")
    if state_out is not None:
        increment_version(out)             # autograd learns of the write
    return h, out
