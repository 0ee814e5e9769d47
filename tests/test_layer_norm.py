"""Layer norm (csrc/layer_norm.cu) against its definition in float64.

Tolerances.  A value v held in the output type is off by at most u |v| (u the
type's unit roundoff).  Before that rounding every value is a handful of
float32 operations on sums of d (or n) terms added in trees and short chains:
a sum is off by at most C 2^-24 times the sum of its terms' magnitudes, with
C = 40 covering chains of up to 40 additions.  So forward and dx are held to
u |v| + 40 2^-24 M, where M is the row's largest product of magnitudes that
enters the value, and dw, db to 40 2^-24 times sum |dy xh|, sum |dy|.
"""

from __future__ import annotations

import pytest
import torch

from qqt_b200.norm import LayerNorm, layer_norm, layer_norm_backward, layer_norm_forward

gpu = pytest.mark.gpu
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
C = 40 * 2.0 ** -24
EPS = 1e-5


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _ref(x, w, b, dy=None):
    x, w = x.double(), w.double()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = 1 / ((c * c).mean(-1, keepdim=True) + EPS).sqrt()
    xh = c * rstd
    y = xh * w + (0 if b is None else b.double())
    # what one float32 rounding inside the row can do to y: |xh| and |mean| rstd, times w
    m = (xh.abs() + mean.abs() * rstd + 1) * w.abs() + (0 if b is None else b.double().abs())
    if dy is None:
        return y, m
    q = dy.double() * w
    qm = q.mean(-1, keepdim=True)
    qx = (q * xh).mean(-1, keepdim=True)
    dx = rstd * (q - qm - xh * qx)
    big = q.abs().amax(-1, keepdim=True)
    xm = xh.abs() + mean.abs() * rstd
    mx = rstd * (q.abs() + big + xm * (q.abs() * xm).mean(-1, keepdim=True) + xm * qx.abs())
    return y, m, dx, mx, (dy.double() * xh).sum(0), (dy.double().abs() * xm).sum(0), \
        dy.double().sum(0), dy.double().abs().sum(0)


def _close(got, want, mag, dtype):
    bound = UNIT[dtype] * want.abs() + C * mag
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25          # half the spacing of its subnormal numbers
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all() and bool((err <= bound).all()), (err - bound).max().item()


def _data(n, d, dtype, seed, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(s, generator=g, device="cuda")

    x = (r(n, d + pad) * (0.5 + r(n, 1).abs()) + 2 * r(n, 1)).to(dtype)[:, :d]
    return x, 1 + 0.3 * r(d), 0.5 * r(d), r(n, d + pad).to(dtype)[:, :d]


SIZES = [(1, 1, 0), (1, 128, 0), (3, 2, 1), (64, 128, 0), (63, 127, 0), (5, 129, 7), (1000, 128, 0),
         (4097, 64, 8), (257, 1352, 0), (130, 2704, 24), (33, 5408, 0), (37, 10816, 0),
         (9, 16385, 3), (3, 50001, 0), (2, 70000, 8), (20011, 96, 0), (100003, 7, 0)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,d,pad", SIZES)
def test_forward_and_backward_match_float64(n, d, pad, dtype):
    _need_cuda()
    x, w, b, dy = _data(n, d, dtype, 7 * n + d, pad)
    y, mean, rstd = layer_norm_forward(x, w, b, EPS)
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w)
    ry, my, rx, mx, rw, mw, rb, mb = _ref(x, w, b, dy)
    _close(y, ry, my, dtype)
    _close(dx, rx, mx, dtype)
    _close(dw, rw, mw, torch.float32)
    _close(db, rb, mb, torch.float32)


@gpu
def test_large_offset_keeps_its_digits():
    """The variance is taken around the mean: rows at 1000 with a spread of 1
    lose no more than the mean's own rounding."""
    _need_cuda()
    x, w, b, _ = _data(50, 512, torch.float32, 3)
    x = x + 1000.0
    _close(layer_norm(x, w, b), *_ref(x, w, b), torch.float32)


@gpu
def test_constant_rows_and_missing_bias():
    _need_cuda()
    x = torch.full((4, 300), 2.5, device="cuda")
    w = torch.rand(300, device="cuda")
    assert layer_norm(x, w).abs().max().item() <= 2.0 ** -24 * 2.5 / EPS ** 0.5 * 40
    b = torch.rand(300, device="cuda")
    assert torch.equal(layer_norm(torch.zeros_like(x), w, b), b.expand(4, 300))


@gpu
def test_nan_and_inf_stay_in_their_rows():
    _need_cuda()
    x, w, b, _ = _data(6, 260, torch.float32, 5)
    clean = layer_norm(x, w, b)
    x[1, 7], x[4, 200] = float("nan"), float("inf")
    y = layer_norm(x, w, b)
    assert y[1].isnan().all() and y[4].isnan().any()
    for r in (0, 2, 3, 5):
        assert torch.equal(y[r], clean[r])


@gpu
def test_layouts_give_the_same_values():
    """CNN-shaped weights, sliced rows, expanded rows, misaligned bases and a
    non-unit inner stride give what the contiguous tensor gives."""
    _need_cuda()
    x, w, b, _ = _data(24, 1352, torch.bfloat16, 9)
    want = layer_norm(x.contiguous(), w, b)
    assert torch.equal(layer_norm(x.view(4, 6, 8, 13, 13), w.view(8, 13, 13), b.view(8, 13, 13)),
                       want.view(4, 6, 8, 13, 13))
    for off in (1, 2, 4):
        wide = torch.zeros((24, 1352 + 11), dtype=x.dtype, device="cuda")
        wide[:, off:off + 1352] = x
        assert torch.equal(layer_norm(wide[:, off:off + 1352], w, b), want)
    assert torch.equal(layer_norm(x.t().contiguous().t(), w, b), want)
    assert torch.equal(layer_norm(x[:1].expand(5, -1), w, b), want[:1].expand(5, -1))


@gpu
def test_module_gradients_through_autograd_and_differences():
    """The module's gradients equal the explicit backward's, and a central
    difference of the loss along a random direction.  With step h the
    difference is off by h^2 / 6 times a third derivative (order 1 here) and
    by sum |c| y 2^-24 / h from the outputs' rounding: 1e-4 + 2e-4 of the
    directional derivative's scale for h = 1e-2; 2e-3 is allowed."""
    _need_cuda()
    ln = LayerNorm((5, 40)).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((30, 5, 40), generator=g, device="cuda", requires_grad=True)
    c = torch.randn((30, 5, 40), generator=g, device="cuda")
    with torch.no_grad():
        ln.weight.add_(0.2 * torch.randn((5, 40), generator=g, device="cuda"))
        ln.bias.add_(0.2 * torch.randn((5, 40), generator=g, device="cuda"))
    (ln(x) * c).sum().backward()
    _, mean, rstd = layer_norm_forward(x.detach(), ln.weight.detach(), ln.bias.detach())
    dx, dw, db = layer_norm_backward(c, x.detach(), mean, rstd, ln.weight.detach())
    assert torch.equal(x.grad, dx) and torch.equal(ln.weight.grad, dw) \
        and torch.equal(ln.bias.grad, db)
    for p in (x, ln.weight, ln.bias):
        v = torch.randn(p.shape, generator=g, device="cuda")
        h, at, f = 1e-2, p.detach().clone(), []
        for s in (h, -h):
            with torch.no_grad():
                p.copy_(at + s * v)
                f.append((ln(x).double() * c.double()).sum())
                p.copy_(at)
        num = ((f[0] - f[1]) / (2 * h)).item()
        want = (p.grad.double() * v.double()).sum().item()
        scale = (p.grad.double() * v.double()).square().sum().sqrt().item()
        assert abs(num - want) <= 2e-3 * max(scale, abs(want)), (num, want)


@gpu
def test_shared_input_gradient_adds_up():
    """A row used by several outputs (expanded) gets the sum of its gradients."""
    _need_cuda()
    x, w, b, dy = _data(7, 130, torch.float32, 11)
    one = x[:1].clone().requires_grad_(True)
    layer_norm(one.expand(7, -1), w, b).backward(dy)
    each = layer_norm_backward(dy, x[:1].expand(7, -1), *layer_norm_forward(
        x[:1].expand(7, -1), w, b)[1:], w)[0]
    assert torch.equal(one.grad, each.sum(0, keepdim=True))


@gpu
def test_empty_and_repeatable():
    _need_cuda()
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    x = torch.empty((0, 64), device="cuda", requires_grad=True)
    wp = w.clone().requires_grad_(True)
    y = layer_norm(x, wp, b)
    assert y.shape == (0, 64)
    y.sum().backward()
    assert x.grad.shape == (0, 64) and not wp.grad.any()
    x, w, b, dy = _data(30001, 100, torch.float32, 2)
    y, mean, rstd = layer_norm_forward(x, w, b)
    first = layer_norm_backward(dy, x, mean, rstd, w)
    for _ in range(3):
        again = layer_norm_backward(dy, x, mean, rstd, w)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


@gpu
def test_other_stream_and_graph_capture():
    _need_cuda()
    x, w, b, dy = _data(300, 128, torch.float32, 4)
    y, mean, rstd = layer_norm_forward(x, w, b)
    want = layer_norm_backward(dy, x, mean, rstd, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer_norm_backward(dy, x, mean, rstd, w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg, mg, rg = layer_norm_forward(x, w, b)
        gg = layer_norm_backward(dy, x, mg, rg, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(yg, y) and all(torch.equal(p, q) for p, q in zip(want, gg))


def test_refusals():
    """Bad arguments raise before anything is launched (host-side checks)."""
    x, w, b = torch.zeros(4, 8), torch.ones(8), torch.zeros(8)
    with pytest.raises(TypeError):
        layer_norm(x.double(), w, b)
    with pytest.raises(TypeError):
        layer_norm(x, w.half(), b)
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(7), b)
    with pytest.raises(ValueError):
        layer_norm(x, w, torch.zeros(2, 4))
    with pytest.raises(ValueError):
        layer_norm(x, w, b, eps=-1.0)
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm(x, w, b)
    with pytest.raises(ValueError):
        layer_norm_backward(x[:3], x, torch.zeros(4), torch.zeros(4), w)
    with pytest.raises(ValueError):
        layer_norm_backward(x, x, torch.zeros(3), torch.zeros(4), w)


def test_c_entry_refusals():
    from qqt_b200 import _capi
    L = _capi.lib()
    P = 0x100000                 # never dereferenced
    assert L.qqt_layernorm_forward(P, 7, 4, 8, 8, P, P, 1e-5, P, None, None, None) == 1
    assert L.qqt_layernorm_forward(P, 0, 4, 0, 8, P, P, 1e-5, P, None, None, None) == 1
    assert L.qqt_layernorm_forward(P, 0, -1, 8, 8, P, P, 1e-5, P, None, None, None) == 1
    assert L.qqt_layernorm_forward(None, 0, 4, 8, 8, P, P, 1e-5, P, None, None, None) == 1
    assert L.qqt_layernorm_forward(P, 0, 4, 8, 8, P, P, float("nan"), P, None, None, None) == 1
    assert L.qqt_layernorm_forward(P, 0, 1 << 40, 8, 8, P, P, 1e-5, P, None, None, None) == 3
    assert L.qqt_layernorm_forward(P, 0, 0, 8, 8, P, P, 1e-5, P, None, None, None) == 0
    assert L.qqt_layernorm_backward(P, 8, P, 8, 0, 4, 8, None, P, P, P, P, P, P, None) == 1
    assert L.qqt_layernorm_backward(P, 8, P, 8, 0, 4, 8, P, P, P, P, P, P, None, None) == 1
    assert L.qqt_layernorm_work_bytes(-1, 8) == 0


@gpu
@pytest.mark.parametrize("n,d,dtype", [(3000, 10816, torch.float16), (5000, 2704, torch.bfloat16),
                                       (2000, 1352, torch.float32), (5, 8192, torch.float32)])
def test_wait_expiry_ends_the_call(n, d, dtype):
    """A wait for a staged row that runs out (qqt_test_set_wait_polls: one on a
    barrier that nothing completes, with the first copies in flight) is
    reported, the call ends, and the next one is as before."""
    _need_cuda()
    from qqt_b200 import _capi
    x, w, b, dy = _data(n, d, dtype, 13)
    x, dy = x.contiguous(), dy.contiguous()
    y, mean, rstd = layer_norm_forward(x, w, b)
    want = (y, mean, rstd) + layer_norm_backward(dy, x, mean, rstd, w)
    assert _capi.device_error() == 0
    lib = _capi.lib()
    try:
        assert lib.qqt_test_set_wait_polls(64) == 0
        layer_norm_forward(x, w, b)
        assert _capi.device_error() == 1 << 3                  # QQT_DEV_TIMEOUT
        layer_norm_backward(dy, x, mean, rstd, w)
        assert _capi.device_error() == 1 << 3
    finally:
        lib.qqt_test_set_wait_polls(0)
    again = layer_norm_forward(x, w, b)
    again = again + layer_norm_backward(dy, x, again[1], again[2], w)
    assert _capi.device_error() == 0
    assert all(torch.equal(p, q) for p, q in zip(want, again))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 130, 512, 1352, 3001, 9000, 16392, 20001])
def test_variance_beyond_float32_and_of_zero(d, dtype):
    """Every path gives what 1 / sqrt(var + eps) is in float32: 0 for a variance
    past its range (y is the bias, dx 0), infinity for none and eps = 0 (0 times
    infinity: NaN); the rows beside are untouched."""
    _need_cuda()
    x, w, b, dy = _data(5, d, dtype, d)
    want = layer_norm_forward(x, w, b)
    wide = x.clone()
    wide[1] = torch.where(torch.arange(d, device="cuda") % 2 == 0, 1e30, -1e30).to(dtype)
    wide[3] = 0.0
    y, mean, rstd = layer_norm_forward(wide, w, b)
    assert rstd[1] == 0 and torch.equal(y[1], b.to(dtype)) and torch.equal(y[3], b.to(dtype))
    dx, _, _ = layer_norm_backward(dy, wide, mean, rstd, w)
    assert not dx[1].any() and torch.isfinite(dx).all()
    _, _, r0 = layer_norm_forward(wide, w, b, eps=0.0)
    y0 = layer_norm(wide, w, b, eps=0.0)
    assert r0[1] == 0 and r0[3] == float("inf") and y0[3].isnan().all()
    for r in (0, 2, 4):
        assert torch.equal(y[r], want[0][r]) and torch.isfinite(y0[r]).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,d", [(70, 8), (3001, 64), (999, 200), (700, 512), (300, 1352),
                                 (500, 2704), (60, 8192), (9, 14084), (7, 16384)])
def test_backward_of_whole_vectors_at_odd_places(n, d, dtype):
    """Rows made of whole 16-byte vectors whose strides or addresses are not on
    16 bytes, x's and dy's differing: the values of the aligned tensors, bit for
    bit, which are held to float64."""
    _need_cuda()
    x, w, b, dy = _data(n, d, dtype, n + d)
    x, dy = x.contiguous(), dy.contiguous()
    y, mean, rstd = layer_norm_forward(x, w, b, EPS)
    want = layer_norm_backward(dy, x, mean, rstd, w)
    ry, my, rx, mx, rw, mw, rb, mb = _ref(x, w, b, dy)
    _close(y, ry, my, dtype)
    _close(want[0], rx, mx, dtype)
    _close(want[1], rw, mw, torch.float32)
    _close(want[2], rb, mb, torch.float32)
    for xo, xp, yo, yp in ((1, 1, 0, 0), (0, 0, 3, 5), (5, 11, 2, 3), (0, 1, 0, 1)):
        wx = torch.full((n, d + xp + xo), float("nan"), dtype=dtype, device="cuda")
        wy = torch.full((n, d + yp + yo), float("nan"), dtype=dtype, device="cuda")
        wx[:, xo:xo + d], wy[:, yo:yo + d] = x, dy
        vx, vy = wx[:, xo:xo + d], wy[:, yo:yo + d]
        f = layer_norm_forward(vx, w, b, EPS)
        assert all(torch.equal(p, q) for p, q in zip(f, (y, mean, rstd)))
        got = layer_norm_backward(vy, vx, mean, rstd, w)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    wo = torch.empty(d + 1, device="cuda")[1:].copy_(w)      # the weight off 16 bytes
    got = layer_norm_backward(dy, x, mean, rstd, wo)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@gpu
@pytest.mark.parametrize("n,d", [(300, 14080), (301, 14081), (200, 14084), (9, 16383), (300, 16384)])
def test_float32_rows_where_the_plan_changes(n, d):
    """Two stages of x and dy no longer fit beside 14,080 float32 values a row."""
    _need_cuda()
    x, w, b, dy = _data(n, d, torch.float32, d)
    y, mean, rstd = layer_norm_forward(x, w, b, EPS)
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w)
    ry, my, rx, mx, rw, mw, rb, mb = _ref(x, w, b, dy)
    _close(y, ry, my, torch.float32)
    _close(dx, rx, mx, torch.float32)
    _close(dw, rw, mw, torch.float32)
    _close(db, rb, mb, torch.float32)
