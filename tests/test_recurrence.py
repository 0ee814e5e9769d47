"""Gated linear recurrence (csrc/recurrence.cu) against its definition in
float64, tick by tick.

Tolerances.  h_t is a convex combination of earlier x and h0, so one tick's
float32 roundings (a handful of units of 2^-24 of the operands) decay with
the state: against M, the largest |x| or |h0| of the channel, the sum over
ticks of what is left of each is at most 8 2^-24 M times the memory's length,
and the length of a memory with gates f is 1/(1 - f); the same holds for the
backward pass in the largest |dh| summed over that length.  The tests draw
gates whose mean memory is about ten ticks and hold values to
u |v| + 400 2^-24 times the largest magnitude that enters (u: the output
type's unit roundoff).
"""

from __future__ import annotations

import pytest
import torch

from qqt_b200.recurrence import (gated_recurrence, gated_recurrence_backward,
                                 gated_recurrence_forward, gated_recurrence_step)

gpu = pytest.mark.gpu
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
C = 400 * 2.0 ** -24


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _ref(x, g, h0, reset, dh=None, dh_last=None):
    t, n, d = x.shape
    dd = dict(dtype=torch.float64, device=x.device)
    x, f = x.double(), torch.sigmoid(g.double())
    h = torch.zeros((n, d), **dd) if h0 is None else h0.double()
    hs, prev = torch.empty((t, n, d), **dd), torch.empty((t, n, d), **dd)
    drop = torch.zeros((t, n, 1), dtype=torch.bool, device=x.device) if reset is None \
        else reset.bool()[..., None]
    for k in range(t):
        prev[k] = torch.where(drop[k], 0.0, h)
        h = f[k] * prev[k] + (1 - f[k]) * x[k]
        hs[k] = h
    if dh is None and dh_last is None:
        return hs, h
    e = torch.zeros((n, d), **dd) if dh_last is None else dh_last.double()
    dx, dg = torch.empty_like(hs), torch.empty_like(hs)
    for k in reversed(range(t)):
        if dh is not None:
            e = e + dh[k].double()
        dx[k] = (1 - f[k]) * e
        dg[k] = f[k] * (1 - f[k]) * e * (prev[k] - x[k])
        e = torch.where(drop[k], 0.0, f[k] * e)
    return hs, h, dx, dg, e


def _close(got, want, mag, dtype=torch.float32):
    if not want.numel():
        assert got.shape == want.shape
        return
    bound = UNIT[dtype] * want.abs() + C * mag
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all() and bool((err <= bound).all()), (err - bound).max().item()


def _data(t, n, d, dtype, seed, batch_first=False, resets=True):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(s, generator=g, device="cuda")

    a, b = (n, t) if batch_first else (t, n)
    both = r(a, b, 2 * d)
    both[..., d:] = 1.5 * both[..., d:] + 1.5
    both, dh = both.to(dtype), r(a, b, d).to(dtype)
    if batch_first:
        both, dh = both.transpose(0, 1), dh.transpose(0, 1)
    reset = (torch.rand((t, n), generator=g, device="cuda") < 0.05) if resets else None
    return both[..., :d], both[..., d:], r(n, d), reset, dh, r(n, d)


SIZES = [(1, 1, 1, False), (1, 64, 128, False), (2, 3, 5, True), (63, 2, 33, False),
         (64, 5, 64, True), (65, 1, 7, False), (128, 40, 128, False), (129, 6, 130, True),
         (200, 700, 36, False), (1000, 1, 1024, True), (4099, 2, 100, True), (20000, 1, 3, True),
         (9001, 1, 517, False), (127, 1, 4096, False)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,n,d,bf", SIZES)
def test_forward_and_backward_match_float64(t, n, d, bf, dtype):
    _need_cuda()
    x, g, h0, reset, dh, dl = _data(t, n, d, dtype, t + n + d, bf)
    h, last, saved = gated_recurrence_forward(x, g, h0, reset)
    dx, dg, dh0 = gated_recurrence_backward(dh, dl, x, g, saved, reset)
    rh, rl, rx, rg, r0 = _ref(x, g, h0, reset, dh, dl)
    m = max(x.abs().max().item(), h0.abs().max().item())
    _close(h, rh, m, dtype)
    _close(last, rl, m)
    me = max(rx.abs().max().item(), dl.abs().max().item(), dh.abs().max().item()) * 4
    _close(dx, rx, me, dtype)
    _close(dg, rg, me * m, dtype)
    _close(dh0, r0, me)


@gpu
@pytest.mark.parametrize("t,n,d", [(130, 9, 40), (5000, 1, 64)])
def test_optional_arguments(t, n, d):
    """No initial state, no resets, no gradient into the sequence or into the
    last state."""
    _need_cuda()
    x, g, h0, reset, dh, dl = _data(t, n, d, torch.float32, 5)
    h, last, saved = gated_recurrence_forward(x, g)
    rh, rl, rx, rg, r0 = _ref(x, g, None, None, dh, None)
    _close(h, rh, x.abs().max().item())
    dx, dg, dh0 = gated_recurrence_backward(dh, None, x, g, saved)
    me = 4 * rx.abs().max().item()
    _close(dx, rx, me)
    _close(dg, rg, me * 6)
    _close(dh0, r0, me)
    h, last, saved = gated_recurrence_forward(x, g, h0, reset)
    dx, dg, dh0 = gated_recurrence_backward(None, dl, x, g, saved, reset)
    _, _, rx, rg, r0 = _ref(x, g, h0, reset, None, dl)
    me = 4 * dl.abs().max().item()
    _close(dx, rx, me)
    _close(dg, rg, me * 6)
    _close(dh0, r0, me)
    assert gated_recurrence(x, g)[0].requires_grad is False


@gpu
def test_resets_cut_the_sequence():
    """A reset drops the state whatever it is, NaN and infinity included, and
    no gradient crosses it."""
    _need_cuda()
    x, g, h0, _, dh, dl = _data(100, 4, 32, torch.float32, 8, resets=False)
    reset = torch.zeros((100, 4), dtype=torch.uint8, device="cuda")
    reset[0, 0] = reset[40, 1] = reset[64, 2] = reset[99, 3] = 1
    h0[0] = float("nan")
    x = x.clone()
    x[39, 1] = float("inf")
    h, last, saved = gated_recurrence_forward(x, g, h0, reset)
    assert torch.isfinite(h[:, 0]).all() and torch.isfinite(h[40:, 1]).all()
    assert not torch.isfinite(h[39, 1]).any()
    dx, dg, dh0 = gated_recurrence_backward(dh, dl, x, g, saved, reset)
    assert not dh0[0].any() and torch.isfinite(dg[:, 0]).all()
    alone = gated_recurrence_forward(x[40:, 1:2].contiguous(), g[40:, 1:2].contiguous(), None, None)
    _close(h[40:, 1:2], alone[0].double(), x[40:, 1].abs().max().item())


@gpu
def test_extreme_gates():
    """Gates far out on both sides: f of 0 and 1 exactly or nearly, the state
    held or replaced, gradients finite; a NaN gate is not hidden."""
    _need_cuda()
    x, g, h0, reset, dh, dl = _data(200, 2, 64, torch.float32, 3)
    g = g.clone()
    g[:, :, 0], g[:, :, 1], g[:, :, 2], g[:, :, 3] = 200.0, -200.0, float("inf"), -float("inf")
    g[:, :, 4], g[:, :, 5] = torch.finfo(torch.float32).max, torch.finfo(torch.float32).min
    h, last, saved = gated_recurrence_forward(x, g, h0)
    for c in (0, 2, 4):
        assert torch.equal(h[:, :, c], h0[:, c].expand(200, 2))
    for c in (1, 3, 5):
        assert torch.equal(h[:, :, c], x[:, :, c])
    dx, dg, dh0 = gated_recurrence_backward(dh, dl, x, g, saved)
    assert all(torch.isfinite(v).all() for v in (dx, dg, dh0))
    g[150, 0, 10] = float("nan")
    h = gated_recurrence(x, g, h0)[0]
    assert torch.isfinite(h[:150]).all() and h[150:, 0, 10].isnan().all()
    assert torch.isfinite(h[:, 1]).all()


@gpu
def test_millions_of_ticks():
    """One channel over 2.2 million ticks: more segments of the least length
    than a grid's second dimension holds.  The reference walks the ticks on
    the host in 64 bits."""
    _need_cuda()
    t = 2200003
    x, g, h0, reset, dh, dl = _data(t, 1, 1, torch.float32, 77)
    h, last, saved = gated_recurrence_forward(x, g, h0, reset)
    dx, dg, dh0 = gated_recurrence_backward(dh, dl, x, g, saved, reset)
    xs, fs = x.double().flatten().tolist(), torch.sigmoid(g.double()).flatten().tolist()
    rs, ds = reset.flatten().tolist(), dh.double().flatten().tolist()
    s, hs, es, e = h0.item(), [], [0.0] * t, dl.item()
    for k in range(t):
        s = fs[k] * (0.0 if rs[k] else s) + (1 - fs[k]) * xs[k]
        hs.append(s)
    for k in range(t - 1, -1, -1):
        e += ds[k]
        es[k] = (1 - fs[k]) * e
        e = 0.0 if rs[k] else fs[k] * e
    m = max(x.abs().max().item(), abs(h0.item()))
    _close(h.flatten().cpu(), torch.tensor(hs, dtype=torch.float64), m)
    want = torch.tensor(es, dtype=torch.float64)
    _close(dx.flatten().cpu(), want, 4 * max(want.abs().max().item(), dh.abs().max().item()))
    assert abs(dh0.item() - e) <= C * 4 * max(abs(e), dh.abs().max().item())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_ticks_equal_the_sequence(dtype):
    """Acting tick by tick, in place, gives the sequence's states: the same
    operations in another order of composition, so within the bound above."""
    _need_cuda()
    t, n, d = 150, 33, 96
    x, g, h0, reset, _, _ = _data(t, n, d, dtype, 6)
    h, last, _ = gated_recurrence_forward(x, g, h0, reset)
    state = h0.clone()
    kept = state.data_ptr()
    for k in range(t):
        hk, state = gated_recurrence_step(x[k], g[k], state, reset[k], state_out=state)
        m = max(x.abs().max().item(), h0.abs().max().item())
        err = (hk.double() - h[k].double()).abs()
        assert bool((err <= 2 * UNIT[dtype] * h[k].double().abs() + C * m).all())
    assert state.data_ptr() == kept
    _close(state, last.double(), 6.0)
    before = h0.clone()
    _, new = gated_recurrence_step(x[0], g[0], h0, reset[0])
    assert torch.equal(h0, before) and new.data_ptr() != h0.data_ptr()


@gpu
def test_pieces_equal_the_whole():
    """Two calls joined by the carried state equal one call over both."""
    _need_cuda()
    x, g, h0, reset, _, _ = _data(300, 3, 50, torch.float32, 12)
    h, last, _ = gated_recurrence_forward(x, g, h0, reset)
    a, mid, _ = gated_recurrence_forward(x[:171], g[:171], h0, reset[:171])
    b, end, _ = gated_recurrence_forward(x[171:], g[171:], mid, reset[171:])
    _close(torch.cat([a, b]), h.double(), 6.0)
    _close(end, last.double(), 6.0)


@gpu
def test_gradients_through_autograd_and_differences():
    """Autograd gives the explicit backward's tensors, and a central difference
    along a random direction agrees: step h = 1e-2 leaves h^2/6 of a third
    derivative (order 1) and the outputs' rounding over h, 4e-4 of the scale
    together; 2e-3 is allowed."""
    _need_cuda()
    t, n, d = 140, 3, 24
    x, g, h0, reset, dh, dl = _data(t, n, d, torch.float32, 21)
    p = [v.clone().requires_grad_(True) for v in (x, g, h0)]

    def loss(x, g, h0):
        h, last = gated_recurrence(x, g, h0, reset)
        return (h.double() * dh.double()).sum() + (last.double() * dl.double()).sum()

    loss(*p).backward()
    _, _, saved = gated_recurrence_forward(x, g, h0, reset)
    want = gated_recurrence_backward(dh, dl, x, g, saved, reset)
    assert all(torch.equal(q.grad, v) for q, v in zip(p, want))
    gen = torch.Generator(device="cuda").manual_seed(2)
    for i in range(3):
        v = torch.randn(p[i].shape, generator=gen, device="cuda")
        f = []
        for s in (1e-2, -1e-2):
            q = [w.detach() for w in p]
            q[i] = q[i] + s * v
            f.append(loss(*q))
        num = ((f[0] - f[1]) / 2e-2).item()
        dot = p[i].grad.double() * v.double()
        assert abs(num - dot.sum().item()) <= 2e-3 * max(dot.square().sum().sqrt().item(),
                                                          abs(dot.sum().item()))


@gpu
def test_empty_repeatable_streams_and_graphs():
    _need_cuda()
    z = torch.empty((0, 3, 8), device="cuda")
    h0 = torch.randn((3, 8), device="cuda")
    h, last, saved = gated_recurrence_forward(z, z, h0)
    assert h.shape == (0, 3, 8) and torch.equal(last, h0) and saved.shape == (0, 3, 8)
    dx, dg, dh0 = gated_recurrence_backward(z, h0, z, z, saved)
    assert dx.shape == (0, 3, 8) and torch.equal(dh0, h0)
    z = torch.empty((5, 0, 8), device="cuda")
    assert gated_recurrence(z, z)[1].shape == (0, 8)
    for size in ((3000, 1, 70), (128, 50, 128)):
        x, g, h0, reset, dh, dl = _data(*size, torch.bfloat16, 9)
        h, last, saved = gated_recurrence_forward(x, g, h0, reset)
        grads = gated_recurrence_backward(dh, dl, x, g, saved, reset)
        want = (h, last, saved) + grads
        for _ in range(3):
            f = gated_recurrence_forward(x, g, h0, reset)
            got = f + gated_recurrence_backward(dh, dl, x, g, f[2], reset)
            assert all(torch.equal(p, q) for p, q in zip(want, got))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f = gated_recurrence_forward(x, g, h0, reset)
            got = f + gated_recurrence_backward(dh, dl, x, g, f[2], reset)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            f = gated_recurrence_forward(x, g, h0, reset)
            got = f + gated_recurrence_backward(dh, dl, x, g, f[2], reset)
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_refusals():
    x = torch.zeros(4, 2, 8)
    h0, reset = torch.zeros(2, 8), torch.zeros(4, 2, dtype=torch.bool)
    for bad in (dict(x=x.double()), dict(gate=x.half()), dict(h0=h0.half()),
                dict(reset=reset.float())):
        with pytest.raises(TypeError):
            gated_recurrence(**{**dict(x=x, gate=x, h0=h0, reset=reset), **bad})
    for bad in (dict(gate=x[:3]), dict(x=x[0], gate=x[0]), dict(h0=h0[:1]), dict(reset=reset[:3])):
        with pytest.raises(ValueError):
            gated_recurrence(**{**dict(x=x, gate=x, h0=h0, reset=reset), **bad})
    with pytest.raises(ValueError, match="CUDA"):
        gated_recurrence(x, x, h0, reset)
    with pytest.raises(ValueError):
        gated_recurrence_backward(x, h0, x, x, torch.zeros(3, 2, 8), reset)
    with pytest.raises(ValueError):
        gated_recurrence_backward(x[:3], h0, x, x, torch.zeros(1, 2, 8), reset)
    with pytest.raises(ValueError):
        gated_recurrence_step(x, x, h0)
    with pytest.raises(ValueError):
        gated_recurrence_step(x[0], x[0], h0, state_out=torch.zeros(8, 2).t())


def test_c_entry_refusals():
    import ctypes
    from qqt_b200 import _capi
    L = _capi.lib()
    P = 0x100000                 # never dereferenced
    s, null = _capi.QqtSeq(P, 16, 8), _capi.QqtSeq(None, 0, 0)
    r = ctypes.byref
    f = L.qqt_recurrence_forward
    assert f(r(s), r(s), None, P, 9, 4, 2, 8, r(s), P, P, P, None) == 1
    assert f(None, r(s), None, P, 0, 4, 2, 8, r(s), P, P, P, None) == 1
    assert f(r(s), r(s), None, P, 0, 4, 2, 0, r(s), P, P, P, None) == 1
    assert f(r(s), r(s), None, P, 0, -4, 2, 8, r(s), P, P, P, None) == 1
    assert f(r(null), r(s), None, P, 0, 4, 2, 8, r(s), P, P, P, None) == 1
    assert f(r(s), r(s), None, P, 0, 4, 0, 8, r(s), P, P, P, None) == 0
    assert f(r(s), r(s), None, P, 0, 4, 1 << 30, 8, r(s), P, P, P, None) == 3
    assert L.qqt_recurrence_step(P, 8, P, 8, None, 0, None, 0, 2, 8, P, P, None) == 1
    assert L.qqt_recurrence_step(P, 8, P, 8, None, 0, P, 4, 2, 8, P, P, None) == 1
    b = L.qqt_recurrence_backward
    assert b(r(s), P, r(s), r(s), None, None, 0, 4, 2, 8, r(s), r(s), P, P, None) == 1
    assert b(r(s), P, r(s), r(s), None, P, 0, 4, 2, 8, None, r(s), P, P, None) == 1
    assert L.qqt_recurrence_chunks(0) == 0 and L.qqt_recurrence_chunks(1) == 1


# Views that overlap themselves: a signal's sliding windows, ticks one sample
# apart; sequences one sample apart; (T, N, D, strides).
OVERLAPS = [(5, 3, 60, (1, 64, 1)), (4, 3, 8, (8, 1, 1)), (10, 3, 8, (50, 1, 1)),
            (3, 1, 16, (1, 16, 1)), (70, 2, 128, (1, 1, 1)), (6, 5, 8, (0, 8, 1))]


def _overlapping(t, n, d, strides, **kw):
    g = torch.Generator(device=kw.get("device", "cpu")).manual_seed(t + d)
    need = 1 + (t - 1) * strides[0] + (n - 1) * strides[1] + d - 1
    return [torch.randn(need, generator=g, device=kw.get("device", "cpu"))
            .to(kw.get("dtype", torch.float32)).as_strided((t, n, d), strides) for _ in range(2)]


@pytest.mark.parametrize("t,n,d,strides", OVERLAPS)
def test_outputs_are_dense_with_a_unit_innermost_stride(t, n, d, strides, monkeypatch):
    """What the kernels are given to write, with the library replaced by one
    that records it: d is innermost, and no two values share an address,
    whatever x's strides."""
    import ctypes
    from qqt_b200 import _capi, recurrence
    written = []

    def note(*operands):
        for p in operands:
            ts, ns = (ctypes.c_int64 * 3).from_address(p)[1:]
            at = (torch.arange(t)[:, None, None] * ts + torch.arange(n)[:, None] * ns
                  + torch.arange(d)).flatten()
            assert at.unique().numel() == t * n * d and at.max() < t * n * d
            written.append((ts, ns, 1))
        return 0

    class Lib:
        qqt_recurrence_chunks = staticmethod(lambda t: (t + 7) // 8)
        qqt_recurrence_work_bytes = staticmethod(lambda t, n, d: 0)
        qqt_recurrence_forward = staticmethod(lambda *a: note(a[8]))
        qqt_recurrence_backward = staticmethod(lambda *a: note(a[10], a[11]))

    monkeypatch.setattr(_capi, "lib", lambda: Lib)
    monkeypatch.setattr(_capi, "launch_stream", lambda *a: 0)
    x, g = _overlapping(t, n, d, strides)
    h, _, saved = recurrence.gated_recurrence_forward(x, g)
    dx, dg, _ = recurrence.gated_recurrence_backward(None, None, x, g, saved)
    assert [v.stride() for v in (h, dx, dg)] == written


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,n,d,strides", OVERLAPS)
def test_views_that_overlap_themselves(t, n, d, strides, dtype):
    """Sliding windows give what their copies give, bit for bit."""
    _need_cuda()
    x, g = _overlapping(t, n, d, strides, device="cuda", dtype=dtype)
    dh = torch.randn((t, n, d), device="cuda").to(dtype)
    h, last, saved = gated_recurrence_forward(x, g)
    got = (h, last, saved) + gated_recurrence_backward(dh, None, x, g, saved)
    xc, gc = x.contiguous(), g.contiguous()
    f = gated_recurrence_forward(xc, gc)
    want = f + gated_recurrence_backward(dh, None, xc, gc, f[2])
    assert all(torch.equal(p, q) for p, q in zip(got, want))



def test_c_step_refuses_a_state_out_that_overlaps():
    """A thread that wrote what another has yet to read would race: refused
    before anything is launched, on made-up addresses, from one byte of overlap
    on.  State and outputs are 5 x 8 floats (160 bytes)."""
    from qqt_b200 import _capi
    L = _capi.lib()
    X, G, S, R, H, OUT = (0x100000 * k for k in range(1, 7))

    def step(out=OUT, x=X, xs=8, dtype=0, reset=None, rs=0, h=H):
        return L.qqt_recurrence_step(x, xs, G, 8, reset, rs, S, dtype, 5, 8, h, out, None)

    for base in (X, G, S, H):
        for k in (4, 32, 156, -4, -32, -156):
            assert step(out=base + k) == 1, (base, k)
    assert step(out=H) == 1                                   # two outputs in one place
    assert step(out=X, dtype=1) == 1 and step(out=X, xs=16) == 1
    assert step(reset=OUT, rs=1) == 1 and step(reset=OUT + 159, rs=1) == 1
    assert step(reset=OUT - 4, rs=1) == 1 and step(reset=OUT, rs=0) == 1
    # rows of a wider buffer, 100 floats apart: each of them counts
    for row in range(5):
        for k in (-156, -4, 0, 28):
            assert step(x=X, xs=100, out=X + 400 * row + k) == 1, (row, k)
    assert step(x=OUT + 4, xs=0) == 1 and step(x=OUT + 1600, xs=-100) == 1


@gpu
def test_state_out_in_every_allowed_place():
    """The state itself, memory right before and after each operand, the gap
    between the rows of a wider one, x or gate themselves."""
    _need_cuda()
    n, d = 5, 8
    size = n * d
    g = torch.Generator(device="cuda").manual_seed(4)
    fresh = torch.randn(9 * size, generator=g, device="cuda")
    reset = torch.tensor([0, 1, 0, 0, 1], dtype=torch.uint8, device="cuda")

    def run(where, row=None):
        buf = fresh.clone()
        at = [buf[k * size:(k + 1) * size].view(n, d) for k in range(9)]
        x = buf[:(n - 1) * row + d].as_strided((n, d), (row, 1)) if row else at[1]
        want = gated_recurrence_step(x, at[5], at[3], reset)
        out = at[where] if row is None else buf[where:where + size].view(n, d)
        got = gated_recurrence_step(x, at[5], at[3], reset, state_out=out)
        assert got[1] is out and all(torch.equal(p, q) for p, q in zip(got, want))

    for where in (0, 1, 2, 3, 4, 5, 6):
        run(where)
    run(8, row=60)                       # x's rows at 0, 60, 120, ..: 8 to 59 is free
    run(20, row=60)
    with pytest.raises(ValueError, match="overlap"):
        run(21, row=60)
    state = fresh[:size].view(n, d)
    with pytest.raises(ValueError, match="overlap"):
        gated_recurrence_step(state, state, state, state_out=fresh[d:d + size].view(n, d))


def test_autograd_learns_of_a_state_written_in_place(monkeypatch):
    """A graph that saved the state before the tick refuses its backward pass
    instead of using the new one; the library is replaced by one that does
    nothing."""
    from qqt_b200 import _capi

    class Lib:
        qqt_recurrence_step = staticmethod(lambda *a: 0)

    monkeypatch.setattr(_capi, "lib", lambda: Lib)
    monkeypatch.setattr(_capi, "launch_stream", lambda *a: 0)
    x, state = torch.zeros(3, 4), torch.ones(3, 4)
    w = torch.ones(3, 4, requires_grad=True)
    loss = (w * state).sum()
    gated_recurrence_step(x, x, state)
    loss.backward()                                 # nothing was written over
    loss = (w * state).sum()
    gated_recurrence_step(x, x, state, state_out=state)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    with torch.inference_mode():
        s = torch.ones(3, 4)
        assert gated_recurrence_step(x, x, s, state_out=s)[1] is s


@gpu
def test_state_out_over_the_one_row_of_a_wider_tensor():
    """With one sequence a row's stride is any: x's own place is allowed."""
    _need_cuda()
    wide = torch.randn((1, 40), device="cuda")
    x, g, s = wide[:, :16], torch.randn((1, 16), device="cuda"), torch.randn((1, 16), device="cuda")
    assert x.stride(0) == 40
    want = gated_recurrence_step(x, g, s)
    got = gated_recurrence_step(x, g, s, state_out=x)
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and torch.equal(wide[:, :16], want[1])
