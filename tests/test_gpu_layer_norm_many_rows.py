"""The parameters' gradients of layer norm over very many rows, where a row that is
dropped or counted twice has to show.

With statistics mean 0 and rstd 1 and small whole numbers for dy and x, every
product and partial sum is a whole number below 2^24, so dweight and dbias are
exact in float32 in any order, and have to be equal."""
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

SHAPES = [(300007, 16), (300007, 17), (100001, 520), (100003, 515), (20011, 1024), (20000, 2049), (20001, 4096), (5003, 8192),
          (5003, 8193), (3001, 12288), (2003, 20000), (2003, 20001), (1501, 32768), (1501, 40000), (1187, 40001)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_whole_numbers_add_up_exactly(rows, cols, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    # |dy x| <= 5 * 4 and 300007 rows of it stay below 2^24; dy leans to one side, and dy x too
    dy = torch.randint(-2, 6, (rows, cols), generator=g, device=DEV, dtype=torch.int8)
    x = torch.randint(-1, 5, (rows, cols), generator=g, device=DEV, dtype=torch.int8)
    db = dy.sum(0, dtype=torch.int64)
    dw = sum((a.short() * b.short()).sum(0, dtype=torch.int64) for a, b in zip(dy.split(4096), x.split(4096)))
    assert int(db.min()) > rows and int(dw.min()) > rows  # each about twice the rows: one row matters, zeros differ
    mean, rstd = torch.zeros(rows, device=DEV), torch.ones(rows, device=DEV)
    got = mcke.layer_norm_backward(dy.to(dtype), x.to(dtype), mean, rstd)
    assert torch.equal(got[1].long(), dw) and torch.equal(got[2].long(), db)
    mcke.check_device_errors()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols", [(300007, 16), (300007, 17), (60000, 1024), (40001, 1001), (5003, 12288)])
def test_sums_that_do_not_cancel(rows, cols, dtype):
    """The longest chain of additions is a slab's rows, a 148th of them (a 74th over pairs of
    blocks: 68 of 5003, which the 160 holds too), and the join of groups and slabs:
    (rows / 148 + 160) u of the sum of magnitudes, and 6 u for the terms."""
    x, w, _, dy = ln._inputs(rows, cols, dtype, seed=3)
    y, mean, rstd = mcke.layer_norm(x, w, save_stats=True)
    dy = (dy + 1 + y.float()).to(dtype)
    _, dw, db = mcke.layer_norm_backward(dy, x, mean, rstd, w)
    d = dy.double()
    for got, terms in ((dw, d * (x.double() - mean.double()[:, None]) * rstd.double()[:, None]), (db, d)):
        want, bound = terms.sum(0), (rows / 148 + 166) * ln.U * terms.abs().sum(0)
        assert ((got.double() - want).abs() <= bound).all()
        assert (want.abs() > 100 * bound).float().mean() > 0.9  # most columns: zeros would not pass
