"""Layer norm of very wide rows, whose statistics must not get worse with the width.

Rows beyond what a block or a cluster holds are added up in fours (2 u of the magnitudes,
u = 2^-24) and the fours of 32 threads in float64; a warp's sum is rounded (u), eight warps'
are joined in seven additions, and the mean is divided by a width that is itself rounded
(2 u): 12 u in all.  A square adds its own u.  The bounds are those of the narrow rows'
tests with a chain of 16 whatever the width."""
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


@pytest.fixture(autouse=True)
def chain(monkeypatch):
    monkeypatch.setattr(ln, "_chain", lambda cols: 16)


@pytest.mark.parametrize("cols", [40000, (1 << 22) + 5, 1 << 24, (1 << 26) + 1])
@pytest.mark.parametrize("value", [1.1, -0.3])
def test_a_constant_row_has_its_value_for_mean_and_no_variance(cols, value):
    x = torch.full((1, cols), value, device=DEV)
    y, mean, rstd = mcke.layer_norm(x, save_stats=True)
    # the error of the mean, squared, is all the variance there is: 6.2e-13 beside eps = 1e-5 for 12 u of 1.1
    assert (mean.double() - x[0, 0].double()).abs() <= 12 * ln.U * abs(value)
    assert (rstd.double() - 1e-5 ** -0.5).abs() <= 4 * ln.U * 1e-5 ** -0.5
    # off by as much as the mean, times rstd
    assert float(y.abs().max()) <= 12 * ln.U * abs(value) * 317


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols", [(3, 32776), (2, 40001), (2, (1 << 22) + 5), (1, 1 << 24)])
def test_forward_and_backward(rows, cols, dtype):
    x, w, b, dy = ln._inputs(rows, cols, dtype, seed=cols, offset=8.0)
    y, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True)
    ln._check_forward(x, w, b, y, mean, rstd)
    dy += 1  # a sum that does not cancel
    ln._check_backward(x, w, mean, rstd, dy, *mcke.layer_norm_backward(dy, x, mean, rstd, w))
