"""Layer norm, forward and backward, against its definition in 64 bits.

Tolerances, with u = 2^-24 (half a step of float32) and L the longest chain of
additions that a row's sum may go through (a thread's share with 32 threads
to a row, and the tree that joins them):
  mean       |dmu| <= L u mean|x|
  rstd       the variance is a sum of squares of x - mu: relative error
             (L + 4) u from the sum and the squares, 2 r |dmu| from the mean's error
             in each deviation (a bound: to first order they cancel), and the
             root halves both
  y          |w| (r |dmu| + |xh| (relative error of r + 3 u)) + u |b| + 2 u |y|
  dx         c1 and c2 carry L u times the mean of their terms' magnitudes and a
             few u of their own; each product and difference adds one u of its result
  dw, db     sums over the rows: (rows + 160) u times the sum of magnitudes
  and the output's own rounding, eps / 2 relative to the value.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

import mcke  # noqa: E402

U = 2.0 ** -24
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def _chain(cols: int) -> int:
    return math.ceil(cols / 32) + 16


def _half_step(t) -> float:
    return torch.finfo(t).eps / 2


def _inputs(rows, cols, dtype, seed=0, offset=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=DEV) + offset * torch.randn(rows, 1, generator=g, device=DEV)
    x[:, ::7] *= 6
    w = 1 + 0.3 * torch.randn(cols, generator=g, device=DEV)
    b = 0.5 * torch.randn(cols, generator=g, device=DEV)
    dy = torch.randn(rows, cols, generator=g, device=DEV)
    return x.to(dtype), w, b, dy.to(dtype)


def _want(x, w, b, eps):
    d = x.double()
    mu = d.mean(1, keepdim=True)
    r = 1 / ((d - mu).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (d - mu) * r
    y = xh * (1 if w is None else w.double()) + (0 if b is None else b.double())
    return y, mu, r, xh


def _check_forward(x, w, b, y, mean, rstd, eps=1e-5):
    want, mu, r, xh = _want(x, w, b, eps)
    n = _chain(x.shape[1])
    dmu = n * U * x.double().abs().mean(1, keepdim=True) + U * mu.abs()
    dr = ((n + 4) * U + 2 * r * dmu) / 2 + 3 * U
    aw = 1.0 if w is None else w.double().abs()
    tol = aw * (r * dmu + xh.abs() * (dr + 3 * U)) + (0 if b is None else U * b.double().abs()) + 2 * U * want.abs()
    tol = tol + _half_step(y.dtype) * (want.abs() + tol) + 1e-38
    assert ((y.double() - want).abs() <= tol).all()
    if mean is not None:
        assert ((mean.double() - mu.squeeze(1)).abs() <= dmu.squeeze(1) + 1e-38).all()
        assert ((rstd.double() - r.squeeze(1)).abs() <= (dr * r).squeeze(1)).all()


COLS = [1, 2, 3, 5, 8, 31, 33, 127, 128, 255, 256, 257, 520, 1000, 1024, 1537, 2048, 2049, 4096, 4097, 4104, 5120, 6001,
        8192, 8200, 12288, 16384, 16392, 20001, 32768, 40008, 65536]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", COLS)
def test_forward(cols, dtype):
    for rows in (1, 5):
        x, w, b, _ = _inputs(rows, cols, dtype, seed=cols)
        y, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True)
        assert y.dtype == dtype and y.shape == x.shape and mean.shape == rstd.shape == (rows,)
        _check_forward(x, w, b, y, mean, rstd)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols", [(1000, 768), (4097, 256), (700, 1000), (333, 4096), (160, 16384), (2000, 33)])
def test_forward_of_many_rows(rows, cols, dtype):
    x, w, b, _ = _inputs(rows, cols, dtype, seed=3)
    _check_forward(x, w, b, *mcke.layer_norm(x, w, b, save_stats=True))


@pytest.mark.parametrize("w, b", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forward_without_weight_or_bias(dtype, w, b):
    for cols in (515, 1024, 8192):
        x, weight, bias, _ = _inputs(6, cols, dtype, seed=4)
        weight, bias = weight if w else None, bias if b else None
        y = mcke.layer_norm(x, weight, bias, eps=1e-3)
        _check_forward(x, weight, bias, y, None, None, eps=1e-3)


def _check_backward(x, w, mean, rstd, dy, dx, dw, db):
    d, g0 = x.double(), dy.double()
    rows, cols = d.shape
    mu, r = mean.double()[:, None], rstd.double()[:, None]
    xh = (d - mu) * r
    g = g0 if w is None else g0 * w.double()
    c1, c2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    want = r * (g - c1 - xh * c2)
    n = _chain(cols)
    # x - mu rounds relative to the difference; the other factors one u each
    dc1 = (n + 2) * U * g.abs().mean(1, keepdim=True)
    dc2 = (n + 6) * U * (g * xh).abs().mean(1, keepdim=True)
    tol = r * (4 * U * (g.abs() + c1.abs() + (xh * c2).abs()) + dc1 + xh.abs() * dc2 + 4 * U * (xh * c2).abs())
    tol = tol + 2 * U * want.abs()
    tol = tol + _half_step(dx.dtype) * (want.abs() + tol) + 1e-38
    assert ((dx.double() - want).abs() <= tol).all()
    if dw is None:
        return
    m = (rows + 160) * U
    for got, terms in ((dw, g0 * xh), (db, g0)):
        assert got.dtype == F32 and got.shape == (cols,)
        assert ((got.double() - terms.sum(0)).abs() <= (m + 4 * U) * terms.abs().sum(0) + 1e-38).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", COLS)
def test_backward(cols, dtype):
    for rows in (1, 7):
        x, w, _, dy = _inputs(rows, cols, dtype, seed=cols + 1)
        _, mean, rstd = mcke.layer_norm(x, w, save_stats=True)
        dx, dw, db = mcke.layer_norm_backward(dy, x, mean, rstd, w)
        assert dx.dtype == dtype and dx.shape == x.shape
        _check_backward(x, w, mean, rstd, dy, dx, dw, db)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols", [(147, 1024), (148, 1024), (149, 1024), (1000, 768), (2053, 136), (700, 1001),
                                        (333, 4096), (300, 16384), (297, 8192), (900, 33)])
def test_backward_of_many_rows(rows, cols, dtype):
    x, w, _, dy = _inputs(rows, cols, dtype, seed=5)
    _, mean, rstd = mcke.layer_norm(x, w, save_stats=True)
    dx, dw, db = mcke.layer_norm_backward(dy, x, mean, rstd, w)
    _check_backward(x, w, mean, rstd, dy, dx, dw, db)
    again = mcke.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))  # the same bits on every run


@pytest.mark.parametrize("cols", [515, 1024, 20001])
def test_backward_without_weight_and_without_parameters(cols):
    x, w, _, dy = _inputs(9, cols, BF16, seed=6)
    _, mean, rstd = mcke.layer_norm(x, save_stats=True)
    dx, dw, db = mcke.layer_norm_backward(dy, x, mean, rstd)
    _check_backward(x, None, mean, rstd, dy, dx, dw, db)
    only = mcke.layer_norm_backward(dy, x, mean, rstd, param_grads=False)
    _check_backward(x, None, mean, rstd, dy, only, None, None)
    # one of the two sums alone, through the C-ABI
    ws = torch.empty(mcke.layer_norm_backward_workspace_bytes(9, cols), dtype=torch.uint8, device=DEV)
    for dwp, dbp in ((True, False), (False, True)):
        got = torch.full((cols,), -7.0, device=DEV)
        rc = mcke.lib().mcke_sm100_layer_norm_backward(
            dy.data_ptr(), cols, x.data_ptr(), cols, None, mean.data_ptr(), rstd.data_ptr(), only.data_ptr(), cols,
            got.data_ptr() if dwp else None, got.data_ptr() if dbp else None, 9, cols, mcke.DTYPE["bf16"],
            ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        assert rc == mcke.OK
        assert torch.equal(got, dw if dwp else db)


def test_no_rows_give_zero_parameter_gradients():
    x = torch.empty(0, 300, device=DEV)
    y, mean, rstd = mcke.layer_norm(x, save_stats=True)
    assert y.shape == (0, 300) and mean.shape == (0,)
    dx, dw, db = mcke.layer_norm_backward(x, x, mean, rstd)
    assert dx.shape == (0, 300) and not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols, pad, shift", [(1024, 8, 0), (1024, 1, 0), (1024, 0, 1), (520, 3, 5), (4096, 4096, 4096),
                                              (16384, 2, 2), (33, 0, 7)])
def test_strided_and_unaligned_rows(cols, pad, shift, dtype):
    rows, stride = 11, cols + pad + shift
    x, w, b, dy = _inputs(rows, cols, dtype, seed=8)

    def view(values):
        buf = torch.full((rows * stride + shift + 16,), 77.0, dtype=dtype, device=DEV)
        v = torch.as_strided(buf, (rows, cols), (stride, 1), shift)
        v.copy_(values)
        return buf, v

    _, xv = view(x)
    buf, yv = view(torch.zeros_like(x))
    ws = torch.randn(cols + 1, device=DEV)
    ws[1:] = w  # a weight that starts off a 16-byte boundary
    y, mean, rstd = mcke.layer_norm(xv, ws[1:], b, out=yv, save_stats=True)
    _check_forward(x, w, b, yv, mean, rstd)
    gbuf, dxv = view(torch.zeros_like(x))
    _, dyv = view(dy)
    dx, dw, db = mcke.layer_norm_backward(dyv, xv, mean, rstd, ws[1:], out=dxv)
    _check_backward(x, w, mean, rstd, dy, dxv, dw, db)
    outside = torch.ones_like(buf, dtype=torch.bool)
    torch.as_strided(outside, (rows, cols), (stride, 1), shift).fill_(False)
    assert (buf[outside] == 77).all() and (gbuf[outside] == 77).all()  # what lies between the rows stays


def test_windows_of_one_buffer_and_broadcast_rows():
    cols = 512
    x, w, b, dy = _inputs(6, cols, BF16, seed=9)
    buf = torch.zeros(6, 2 * cols, dtype=BF16, device=DEV)
    buf[:, :cols] = x
    mcke.layer_norm(buf[:, :cols], w, b, out=buf[:, cols:])
    _check_forward(x, w, b, buf[:, cols:], None, None)
    one = x[:1].expand(6, cols)  # row stride 0
    _check_forward(one.contiguous(), w, b, *mcke.layer_norm(one, w, b, save_stats=True))
    _, mean, rstd = mcke.layer_norm(x, w, save_stats=True)
    up = dy[:1].expand(6, cols)
    _check_backward(x, w, mean, rstd, up.contiguous(), *mcke.layer_norm_backward(up, x, mean, rstd, w))


def test_leading_dimensions():
    x, w, b, dy = _inputs(12, 256, F32, seed=10)
    y, mean, rstd = mcke.layer_norm(x.view(3, 4, 256), w, b, save_stats=True)
    assert y.shape == (3, 4, 256)
    _check_forward(x, w, b, y.view(12, 256), mean, rstd)
    dx, dw, db = mcke.layer_norm_backward(dy.view(3, 4, 256), x.view(3, 4, 256), mean, rstd, w)
    _check_backward(x, w, mean, rstd, dy, dx.view(12, 256), dw, db)


@pytest.mark.parametrize("cols", [64, 1024, 1025, 16384, 40000])
def test_values_at_the_edges(cols):
    # constant rows: no variance, rstd = 1 / sqrt(eps), y = b exactly where the mean is exact
    x = torch.full((3, cols), 4.0, device=DEV)
    b = torch.randn(cols, device=DEV)
    y, mean, rstd = mcke.layer_norm(x, None, b, eps=0.25, save_stats=True)
    assert (mean == 4).all() and (rstd == 2).all() and torch.equal(y, b.expand(3, cols))
    # a large offset: the variance is not lost in it (values exact in float32)
    x = (1024.0 + torch.randint(0, 3, (4, cols), device=DEV)).float()
    _check_forward(x, None, None, *mcke.layer_norm(x, save_stats=True))
    # NaN and infinity stay in their rows
    x = torch.randn(4, cols, device=DEV)
    ok = mcke.layer_norm(x)
    x[1, cols // 2] = float("nan")
    x[2, 0] = float("inf")
    y = mcke.layer_norm(x)
    assert y[1].isnan().all() and y[2].isnan().any() and torch.equal(y[0], ok[0]) and torch.equal(y[3], ok[3])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient_against_differences(dtype):
    """Directional derivatives of the definition in 64 bits, by central differences
    of step 1e-5 (error about 1e-10 of the values), against the kernel's gradients;
    the kernel's own error is at most a relative 1e-3 of the terms' magnitude
    (bf16: a half step 2^-9 of each dx element, adding over the columns)."""
    x, w, b, dy = _inputs(5, 600, dtype, seed=11)
    _, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True)
    dx, dw, db = (t.double() for t in mcke.layer_norm_backward(dy, x, mean, rstd, w))
    g = torch.Generator(device=DEV).manual_seed(12)
    loss = lambda x_, w_, b_: (_want(x_, w_, b_, 1e-5)[0] * dy.double()).sum()  # noqa: E731
    h = 1e-5
    x, w, b = x.double(), w.double(), b.double()
    for which, grad in enumerate((dx, dw, db)):
        for _ in range(3):
            args = [x, w, b]
            v = torch.randn(args[which].shape, generator=g, device=DEV, dtype=torch.float64)
            hi, lo = list(args), list(args)
            hi[which], lo[which] = args[which] + h * v, args[which] - h * v
            diff = (loss(*hi) - loss(*lo)) / (2 * h)
            bound = (2 ** -8 if which == 0 and dtype == BF16 else 2 ** -16) * (grad * v).abs().sum()
            assert (diff - (grad * v).sum()).abs() <= bound + 1e-5
