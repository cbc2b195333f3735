"""The gradient norm and clipping against their definitions in 64 bits.

The squares are added in double, so the norm is off by its rounding to float
(u = 2^-24) and the double sum's last bits: 2 u.  The coefficient adds the sum
norm + 1e-6, the quotient and the norm's own error: 4 u; the product one more,
and the output's rounding eps / 2.
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


def _grads(sizes, dtypes, seed=0, scale=1e-2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(scale * 4.0 ** (i % 5) * torch.randn(n, generator=g, device=DEV)).to(dtypes[i % len(dtypes)])
            for i, n in enumerate(sizes)]


def _norm(grads):
    return math.sqrt(math.fsum(float(x.double().square().sum()) for x in grads))


def _check_clip(before, after, max_norm, norm, got):
    assert got.dtype == F32 and got.dim() == 0 and abs(float(got) - norm) <= 2 * U * norm
    c = min(1.0, max_norm / (norm + 1e-6))
    for x, y in zip(before, after):
        want = x.double() * c
        tol = 5 * U * want.abs() + torch.finfo(y.dtype).eps / 2 * want.abs() * (1 + 5 * U) + 1e-38
        assert ((y.double() - want).abs() <= tol).all()


SIZES = {
    "one element": [1],
    "short": [1, 2, 3, 7, 8, 9, 15, 16, 17],
    "around a chunk": [4095, 4096, 4097, 8191, 8192, 8193, 8200],
    "empty ones": [0, 5, 0, 0, 4096, 0],
    "mixed": [100003, 1, 64, 262144, 33, 1000000, 12288],
    "many": [1 + 37 * (i % 11) for i in range(200)],
    "over one table": [3 + i % 5 for i in range(1003)],
    "over two tables": [1 + i % 3 for i in range(2001)],
    "large": [3000001, 2097152],
}


@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F32, BF16]])
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES.keys())
def test_norm_and_clip(sizes, dtypes):
    grads = _grads(sizes, dtypes, seed=len(sizes))
    norm = _norm(grads)
    assert abs(float(mcke.grad_norm(grads)) - norm) <= 2 * U * norm
    for max_norm in (0.3 * norm, 3 * norm):
        # in place
        mine = [x.clone() for x in grads]
        got = mcke.clip_grad_norm(mine, max_norm)
        _check_clip(grads, mine, max_norm, norm, got)
        if max_norm > norm:
            assert all(torch.equal(a, b) for a, b in zip(grads, mine))
        # into other tensors, of the same types and of float32
        for out in ([torch.full_like(x, 7) for x in grads], [torch.full(x.shape, 7.0, device=DEV) for x in grads]):
            keep = [x.clone() for x in grads]
            got = mcke.clip_grad_norm(grads, max_norm, out=out)
            _check_clip(grads, out, max_norm, norm, got)
            assert all(torch.equal(a, b) for a, b in zip(grads, keep))
        # by a norm that is given
        mine = [x.clone() for x in grads]
        mcke.clip_grads(mine, max_norm, torch.tensor(norm, device=DEV))
        _check_clip(grads, mine, max_norm, norm, torch.tensor(norm))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_that_start_anywhere(dtype):
    flat = _grads([60000], [dtype], seed=3)[0]
    keep = flat.clone()
    cuts = [0, 1, 4, 9, 4100, 4101, 12345, 30001, 60000]
    parts = [flat[a:b] for a, b in zip(cuts, cuts[1:])][1:-1]  # the first and last stay out
    norm = _norm(parts)
    before = [p.clone() for p in parts]
    _check_clip(before, parts, 0.5 * norm, norm, mcke.clip_grad_norm(parts, 0.5 * norm))
    assert torch.equal(flat[:1], keep[:1]) and torch.equal(flat[30001:], keep[30001:])
    # outputs at another offset than the gradients
    buf = torch.full((60016,), 3.0, device=DEV).to(dtype)
    outs = [buf[a + 3:b + 3] for a, b in zip(cuts, cuts[1:])]
    grads = [keep[a:b] for a, b in zip(cuts, cuts[1:])]
    norm = _norm(grads)
    _check_clip(grads, outs, 0.5 * norm, norm, mcke.clip_grad_norm(grads, 0.5 * norm, out=outs))
    assert (buf[:3] == 3).all() and (buf[60003:] == 3).all()
    if dtype == BF16:
        wide = torch.full((60016,), 3.0, device=DEV)
        outs = [wide[a + 1:b + 1] for a, b in zip(cuts, cuts[1:])]
        _check_clip(grads, outs, 0.5 * norm, norm, mcke.clip_grad_norm(grads, 0.5 * norm, out=outs))


def test_range_of_values():
    # squares that leave float's range, at both ends, next to one another
    for values in ([1e30, -2e30], [1e-30, 3e-30], [1e-30, 1e30], [3e38, 0.0], [1e-45, 0.0]):
        x = torch.tensor(values * 50, device=DEV)
        norm = _norm([x])
        if norm < 3.4e38:
            got = float(mcke.grad_norm([x]))
            assert abs(got - norm) <= 2 * U * norm + 1.4e-45
    assert float(mcke.grad_norm([torch.full((100,), 3e38, device=DEV)])) == math.inf  # the norm itself does
    # many small next to one large: each is below half a step of the sum in float
    x = torch.full((1 << 22,), 1e-4, device=DEV)
    x[5] = 1.0
    assert abs(float(mcke.grad_norm([x])) - _norm([x])) <= 2 * U * _norm([x])


def test_nan_infinity_and_zero():
    x = torch.ones(5000, device=DEV)
    x[77] = float("nan")
    y = torch.ones(30, device=DEV, dtype=BF16)
    assert mcke.clip_grad_norm([x, y], 1.0).isnan() and x.isnan().all() and y.isnan().all()
    x = torch.ones(5000, device=DEV)
    x[77] = math.inf
    assert mcke.clip_grad_norm([x], 1.0) == math.inf
    assert x[77].isnan() and not x[:77].any()
    z = [torch.zeros(300, device=DEV), torch.zeros(0, device=DEV)]
    assert mcke.clip_grad_norm(z, 1.0) == 0 and not z[0].any()
    w = torch.ones(300, device=DEV)
    mcke.clip_grad_norm([w], 0.0)
    assert not w.any()


def test_only_empty_tensors():
    norm = mcke.grad_norm([torch.zeros(0, device=DEV)] * 3)
    assert norm == 0
    assert mcke.clip_grad_norm([torch.zeros(0, device=DEV)], 1.0) == 0


def test_the_same_tensor_twice():
    x = torch.randn(3000, device=DEV)
    n = _norm([x, x])
    assert abs(float(mcke.grad_norm([x, x])) - n) <= 2 * U * n  # counts twice
    with pytest.raises(mcke.MckeError, match="overlaps"):
        mcke.clip_grad_norm([x, x], 1.0)
    out = [torch.empty_like(x), torch.empty_like(x)]
    _check_clip([x, x], out, 1.0, n, mcke.clip_grad_norm([x, x], 1.0, out=out))


def test_norm_of_shards():
    grads = _grads([50000, 3001], [F32, BF16], seed=6)
    shards = [[g[: g.numel() // 3] for g in grads], [g[g.numel() // 3:] for g in grads]]
    norm = torch.stack([mcke.grad_norm(s) for s in shards]).square().sum().sqrt()
    keep = [g.clone() for g in grads]
    for s in shards:
        mcke.clip_grads(s, 0.1, norm)
    want = _norm(keep)
    c = 0.1 / (want + 1e-6)
    for g, k in zip(grads, keep):
        # the norm of two rounded norms: 4 u more
        assert ((g.double() - k.double() * c).abs() <= (9 * U + torch.finfo(g.dtype).eps / 2 * 1.001) * c * k.double().abs()).all()


def test_refusals():
    x = torch.zeros(8, 8, device=DEV)
    with pytest.raises(ValueError, match="contiguous"):
        mcke.grad_norm([x.t()[1:, 1:]])
    with pytest.raises(ValueError, match="shape"):
        mcke.clip_grad_norm([x], 1.0, out=[x.view(-1)])
    with pytest.raises(ValueError, match="float32"):
        mcke.clip_grad_norm([x], 1.0, out=[x.half()])
    with pytest.raises(ValueError, match="norm"):
        mcke.clip_grads([x], 1.0, torch.zeros(2, device=DEV))
    with pytest.raises(mcke.MckeError, match="bf16"):
        mcke.clip_grad_norm([x], 1.0, out=[x.bfloat16()])
    with pytest.raises(mcke.MckeError, match="max_norm"):
        mcke.clip_grad_norm([x], -1.0)
