"""Layer norm of rows whose sums leave float32's range: the same answer from every
kernel that a width, a type or a number of rows chooses.

  a row that holds an infinity        mean infinite, rstd and y NaN
  squared deviations past the range   rstd 0, y = bias, dx = 0, nothing for dweight
  values whose sum is past the range  mean infinite, rstd 0, y NaN
"""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

import mcke  # noqa: E402
import test_gpu_layer_norm as ln  # noqa: E402

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")

SHAPES = [(6, 33), (6, 64), (6, 512), (6, 515), (6, 4096), (600, 1024), (600, 515), (600, 4096), (600, 8192), (600, 8193),
          (6, 12288), (6, 16384), (6, 16385), (6, 20000), (6, 32768), (6, 32769), (6, 40000)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_forward(rows, cols, dtype):
    x, w, b, _ = ln._inputs(rows, cols, dtype, seed=cols)
    clean = mcke.layer_norm(x, w, b, save_stats=True)
    x[1, cols // 2] = INF
    x[2, cols - 1] = -INF
    x[3, ::2], x[3, 1::2] = 1e25, -1e25
    x[4] = 3e38
    y, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True)
    assert mean[1] == INF and mean[2] == -INF
    assert rstd[1:3].isnan().all() and y[1:3].isnan().all()
    # one value is left over in an odd row; the sum goes through the chain's additions
    assert (mean[3].double() - x[3].double().mean()).abs() <= ln._chain(cols) * ln.U * 1e25 + ln.U * 1e25
    assert rstd[3] == 0 and torch.equal(y[3], b.to(dtype))
    assert mean[4] == INF and rstd[4] == 0 and y[4].isnan().all()
    others = torch.ones(rows, dtype=torch.bool, device=DEV)
    others[1:5] = False
    assert all(torch.equal(got[others], was[others]) for got, was in zip((y, mean, rstd), clean))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_backward(rows, cols, dtype):
    x, w, _, dy = ln._inputs(rows, cols, dtype, seed=cols + 1)
    # 1e36: the sum of dy w (x - mean) is past the range in wide rows, and has to be, times rstd = 0, nothing
    x[3, ::2], x[3, 1::2] = 1e36, -1e36
    _, mean, rstd = mcke.layer_norm(x, w, save_stats=True)
    assert rstd[3] == 0
    dx, dw, db = mcke.layer_norm_backward(dy, x, mean, rstd, w)
    ln._check_backward(x, w, mean, rstd, dy, dx, dw, db)
    assert not dx[3].any()
    assert torch.equal(dx, mcke.layer_norm_backward(dy, x, mean, rstd, w, param_grads=False))
