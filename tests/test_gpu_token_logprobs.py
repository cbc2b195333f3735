"""Token log probabilities, entropy, alternatives and their gradient, against
their definitions in 64 bits.

Tolerances, with u = 2^-24, d = x - max (|d| its distance), L = cols / 256 + 40
the longest chain of additions (256 threads or more to a row) and E the mean
under p:
  e^d           relative 4 u + 2 |d| u (the exponential, and the rounding of d and of
                its scaled form)
  ln s          absolute (L + 8) u + 2 u E|d|
  lse, lp       that, plus 2 u of the parts they are added from
  H             that, plus (L + 12) u E|d| + 2 u E d^2
  dx_j          p_j's relative error (8 + 2 |q|) u (q = x_j - lse) on each term
  and the output's own rounding, eps / 2 relative to the value.
Ids are equal.
"""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

import mcke  # noqa: E402

U = 2.0 ** -24
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


def _logits(rows, cols, dtype, seed=0, masked=0, scale=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = scale * torch.randn(rows, cols, generator=g, device=DEV) + 4 * torch.randn(rows, 1, generator=g, device=DEV)
    if masked:
        x[torch.rand(rows, cols, generator=g, device=DEV) < masked] = -INF
    t = torch.randint(0, cols, (rows,), generator=g, device=DEV)
    return x.to(dtype), t


def _check(x, t, r, top_k):
    """r (a TokenLogprobs) of finite or -inf logits with something left in each row."""
    d = x.double()
    rows, cols = d.shape
    m = d.amax(1, keepdim=True)
    dist = d - m
    e = dist.exp()
    s = e.sum(1, keepdim=True)
    p = e / s
    far = torch.where(p > 0, dist.abs(), 0.0)
    e1, e2 = (p * far).sum(1), (p * far * far).sum(1)
    ln_s = s.log().squeeze(1)
    n = cols / 256 + 40
    tol_ln = (n + 8) * U + 2 * U * e1
    lse = m.squeeze(1) + ln_s
    assert ((r.lse.double() - lse).abs() <= tol_ln + 2 * U * (m.squeeze(1).abs() + ln_s.abs())).all()
    if r.entropy is not None:
        ent = ln_s + e1
        assert ((r.entropy.double() - ent).abs() <= tol_ln + (n + 12) * U * e1 + 2 * U * e2 + 4 * U * ent.abs()).all()
    lp = dist - ln_s[:, None]
    lp[lp.float() == -INF] = -INF  # lowest - max of the type is -6.8e38: no float32 but -inf is near it
    tol_lp = tol_ln[:, None] + 2 * U * (torch.where(lp == -INF, 0.0, lp.abs()) + ln_s.abs()[:, None])
    if r.logprobs is not None:
        at = t.clamp(0, cols - 1)[:, None]
        want = torch.where(t < 0, 0.0, lp.gather(1, at).squeeze(1))
        got = r.logprobs.double()
        assert torch.equal(got == -INF, want == -INF)
        off = torch.where(want == -INF, 0.0, got - want).abs()
        assert (off <= tol_lp.gather(1, at).squeeze(1)).all()
    if top_k:
        order = torch.sort(d, dim=1, descending=True, stable=True).indices[:, :top_k]
        assert r.top_ids.dtype == torch.int64 and torch.equal(r.top_ids, order)
        want, got = lp.gather(1, order), r.top_logprobs.double()
        assert torch.equal(got == -INF, want == -INF)
        assert (torch.where(want == -INF, 0.0, got - want).abs() <= tol_lp.gather(1, order)).all()


COLS = [1, 2, 7, 8, 9, 31, 100, 255, 256, 257, 1000, 1024, 2048, 2051, 4096, 8191, 16384, 16391, 32768, 50257, 65535,
        131072, 200001]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", COLS)
def test_forward(cols, dtype):
    for rows, k in ((1, min(cols, 20)), (3, min(cols, 5)), (17, 0)):
        x, t = _logits(rows, cols, dtype, seed=cols)
        _check(x, t, mcke.token_logprobs(x, t, top_k=k, entropy=True), k)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols, k", [(1000, 1024, 4), (700, 33, 32), (2100, 257, 1), (600, 32768, 8), (400, 50257, 5),
                                           (149, 16384, 32), (75, 131072, 2), (37, 65536, 20), (5000, 2000, 0)])
def test_forward_of_many_rows(rows, cols, k, dtype):
    x, t = _logits(rows, cols, dtype, seed=2, masked=0.1)
    t[::9] = -100
    r = mcke.token_logprobs(x, t, top_k=k, entropy=True)
    _check(x, t, r, k)
    again = mcke.token_logprobs(x, t, top_k=k, entropy=True)
    assert all(torch.equal(a, b) for a, b in zip(r, again) if a is not None)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [40, 3000, 70000])
def test_parts_alone(cols, dtype):
    x, t = _logits(4, cols, dtype, seed=3)
    whole = mcke.token_logprobs(x, t, top_k=4, entropy=True)
    lse = mcke.token_logprobs(x)
    assert lse.logprobs is lse.entropy is lse.top_ids is lse.top_logprobs is None
    _check(x, t, lse, 0)
    _check(x, t, mcke.token_logprobs(x, t), 0)
    top = mcke.token_logprobs(x, top_k=4)
    assert torch.equal(top.top_ids, whole.top_ids) and top.logprobs is None
    _check(x, t, top, 4)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [64, 1000, 5000, 50257, 140000])
def test_equal_values_go_by_index(cols, dtype):
    g = torch.Generator(device=DEV).manual_seed(4)
    few = torch.randint(0, 3, (3, cols), generator=g, device=DEV).float()  # thirds of a row are equal
    one = torch.zeros(3, cols, device=DEV)
    zeros = one.clone()
    zeros[:, 1::2] = -0.0  # -0 is 0
    rising = torch.arange(cols, device=DEV).div(cols / 100.0, rounding_mode="floor").expand(3, cols).contiguous()
    for x in (few, one, zeros, rising, -rising):
        x = x.to(dtype)
        t = torch.zeros(3, dtype=torch.int64, device=DEV)
        _check(x, t, mcke.token_logprobs(x, t, top_k=32, entropy=True), 32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [40, 1024, 4099, 65536])
def test_masks(cols, dtype):
    x, t = _logits(8, cols, dtype, seed=5)
    low = torch.finfo(dtype).min
    x[0] = -INF                       # nothing left
    x[1] = -INF; x[1, cols - 1] = 3   # one token left  # noqa: E702
    x[2, ::2] = low                   # masked by the type's lowest value
    x[3] = low                        # all of them: a uniform row
    x[4, 1:] = low
    x[4, 0] = torch.finfo(dtype).max  # the whole range of the type
    x[5, : cols // 2] = -INF
    t[0], t[1], t[5] = 3, 5, 0        # given tokens that are masked
    r = mcke.token_logprobs(x, t, top_k=4, entropy=True)
    assert r.lse[0] == -INF and r.logprobs[0] == -INF and r.entropy[0] == 0
    assert (r.top_logprobs[0] == -INF).all() and r.top_ids[0].tolist() == [0, 1, 2, 3]
    assert r.logprobs[1] == -INF and r.entropy[1] == 0 and r.top_logprobs[1].tolist() == [0] + [-INF] * 3
    assert r.top_ids[1].tolist() == [cols - 1, 0, 1, 2] and r.logprobs[5] == -INF
    rest = mcke.TokenLogprobs(*(v[1:] for v in r))
    _check(x[1:], t[1:], rest, 4)
    gl = torch.ones(8, device=DEV)
    dx = mcke.token_logprobs_backward(x, r.lse, t, gl, r.entropy, gl, gl)
    assert not dx[0].any() and dx.isfinite().all()
    _check_backward(x[1:], t[1:], r.lse[1:], r.entropy[1:], gl[1:], gl[1:], gl[1:], dx[1:])


@pytest.mark.parametrize("cols", [40, 5000, 66000])
def test_bad_values_stay_in_their_rows(cols):
    x, t = _logits(6, cols, F32, seed=6)
    good = mcke.token_logprobs(x, t, top_k=3, entropy=True)
    x[1, cols // 3] = float("nan")
    x[3, cols - 1] = INF
    x[4] = -INF
    x[4, 7] = float("nan")
    t[5] = cols  # past the end
    r = mcke.token_logprobs(x, t, top_k=3, entropy=True)
    for row in (1, 3, 4):
        for v in (r.logprobs, r.lse, r.entropy):
            assert v[row].isnan()
        assert r.top_logprobs[row].isnan().all()
    assert r.top_ids[1, 0] == cols // 3 and r.top_ids[3, 0] == cols - 1 and r.top_ids[4, 0] == 7
    assert r.logprobs[5].isnan() and r.lse[5] == good.lse[5]
    for v, w in zip(r, good):
        assert torch.equal(v[0], w[0]) and torch.equal(v[2], w[2])
    gl = torch.ones(6, device=DEV)
    dx = mcke.token_logprobs_backward(x, r.lse, t, gl)
    assert all(dx[row].isnan().all() for row in (1, 3, 4, 5)) and dx[0].isfinite().all() and dx[2].isfinite().all()
    # without grad_logprobs the target takes no part
    assert mcke.token_logprobs_backward(x, r.lse, grad_lse=gl)[5].isfinite().all()


def _check_backward(x, t, lse, ent, gl, ge, gz, dx):
    d, cols = x.double(), x.shape[1]
    q = d - lse.double()[:, None]
    p = torch.where(q == -INF, 0.0, q.exp())
    q = torch.where(p > 0, q, 0.0)
    col = lambda v: (torch.zeros(len(d), dtype=torch.float64, device=DEV) if v is None else v.double())[:, None]  # noqa: E731
    g, h, z, hh = col(gl), col(ge), col(gz), col(ent)
    if gl is not None:
        g = torch.where(t[:, None] < 0, 0.0, g)
    terms = z.abs() + g.abs() + h.abs() * (q.abs() + hh.abs())
    want = p * (z - g - h * (q + hh))
    if gl is not None:
        hot = torch.zeros_like(d).scatter_(1, t.clamp(min=0)[:, None], 1.0) * (t[:, None] >= 0)
        want = want + g * hot
    tol = p * terms * (12 + 2 * q.abs()) * U + 2 * U * want.abs()
    tol = tol + torch.finfo(dx.dtype).eps / 2 * (want.abs() + tol) + 1e-37
    assert dx.dtype == x.dtype and ((dx.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", COLS)
def test_backward(cols, dtype):
    for rows in (1, 19):
        x, t = _logits(rows, cols, dtype, seed=cols + 7)
        t[2::5] = -1
        r = mcke.token_logprobs(x, t, entropy=True)
        g = torch.Generator(device=DEV).manual_seed(cols)
        gl, ge, gz = torch.randn(3, rows, generator=g, device=DEV).unbind(0)
        dx = mcke.token_logprobs_backward(x, r.lse, t, gl, r.entropy, ge, gz)
        _check_backward(x, t, r.lse, r.entropy, gl, ge, gz, dx)
        _check_backward(x, t, r.lse, None, gl, None, None, mcke.token_logprobs_backward(x, r.lse, t, gl))
        _check_backward(x, t, r.lse, r.entropy, None, ge, None,
                        mcke.token_logprobs_backward(x, r.lse, entropy=r.entropy, grad_entropy=ge))
        mine = x.clone()
        assert mcke.token_logprobs_backward(mine, r.lse, t, gl, r.entropy, ge, gz, out=mine) is mine
        assert torch.equal(mine, dx)  # in place


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols, pad, shift", [(1024, 64, 0), (1000, 24, 0), (1001, 0, 3), (4096, 1, 0), (70001, 2, 1),
                                              (9, 0, 0)])
def test_strided_and_unaligned_rows(cols, pad, shift, dtype):
    rows, stride = 7, cols + pad
    x, t = _logits(rows, cols, dtype, seed=9)
    buf = torch.full((rows * stride + shift,), 9e4, device=DEV).to(dtype)  # larger than any logit
    v = torch.as_strided(buf, (rows, cols), (stride, 1), shift)
    v.copy_(x)
    k = min(cols, 6)
    r = mcke.token_logprobs(v, t, top_k=k, entropy=True)
    _check(x, t, r, k)
    gl, ge = torch.randn(2, rows, device=DEV).unbind(0)
    want = mcke.token_logprobs_backward(x, r.lse, t, gl, r.entropy, ge)
    _check_backward(x, t, r.lse, r.entropy, gl, ge, None, want)
    assert torch.equal(mcke.token_logprobs_backward(v, r.lse, t, gl, r.entropy, ge), want)
    out = torch.full((rows * stride + 3,), 5.0, device=DEV).to(dtype)
    ov = torch.as_strided(out, (rows, cols), (stride, 1), 2)
    mcke.token_logprobs_backward(v, r.lse, t, gl, r.entropy, ge, out=ov)
    assert torch.equal(ov, want)
    outside = torch.ones_like(out, dtype=torch.bool)
    torch.as_strided(outside, (rows, cols), (stride, 1), 2).fill_(False)
    assert (out[outside] == 5).all()
    mcke.token_logprobs_backward(v, r.lse, t, gl, r.entropy, ge, out=v)
    assert torch.equal(v, want)
    assert torch.equal(buf[: shift], torch.full((shift,), 9e4, device=DEV).to(dtype))


def test_leading_dimensions_and_no_rows():
    x, t = _logits(6, 300, F32, seed=10)
    r = mcke.token_logprobs(x.view(2, 3, 300), t.view(2, 3), top_k=2, entropy=True)
    assert r.logprobs.shape == r.lse.shape == r.entropy.shape == (2, 3) and r.top_ids.shape == (2, 3, 2)
    _check(x, t, mcke.TokenLogprobs(*(v.flatten(0, 1) for v in r)), 2)
    empty = mcke.token_logprobs(x[:0], t[:0], top_k=2, entropy=True)
    assert empty.lse.shape == (0,) and empty.top_ids.shape == (0, 2)
    assert mcke.token_logprobs_backward(x[:0], empty.lse, t[:0], empty.lse).shape == (0, 300)


def test_peaked_and_flat_rows():
    # near certainty: 1 - p of 1e-4 .. 1e-9 has to come from s, not from lse's last bits
    for gap in (9.0, 14.0, 20.0):
        x = torch.zeros(2, 5, device=DEV)
        x[:, 2] = gap + 40.0
        x[:, [0, 1, 3, 4]] = 40.0
        t = torch.tensor([2, 0], device=DEV)
        _check(x, t, mcke.token_logprobs(x, t, top_k=5, entropy=True), 5)
    for scale in (1e-3, 60.0, 1e4):
        x, t = _logits(5, 3001, F32, seed=11, scale=scale)
        _check(x, t, mcke.token_logprobs(x, t, top_k=3, entropy=True), 3)


def test_gradient_against_differences():
    """Central differences (step 1e-5) of the definitions in 64 bits; the kernel's
    error is within 2^-16 of its terms' magnitude for f32."""
    x, t = _logits(4, 700, F32, seed=12)
    t[1] = -1
    r = mcke.token_logprobs(x, t, entropy=True)
    g = torch.Generator(device=DEV).manual_seed(13)
    gl, ge, gz = torch.randn(3, 4, generator=g, device=DEV).unbind(0)
    dx = mcke.token_logprobs_backward(x, r.lse, t, gl, r.entropy, ge, gz).double()

    def loss(d):
        lp = torch.log_softmax(d, 1)
        given = lp.gather(1, t.clamp(min=0)[:, None]).squeeze(1) * (t >= 0)
        return (gl * given - ge * (lp.exp() * lp).sum(1) + gz * torch.logsumexp(d, 1)).sum()

    d, h = x.double(), 1e-5
    for _ in range(4):
        v = torch.randn(d.shape, generator=g, device=DEV, dtype=torch.float64)
        diff = (loss(d + h * v) - loss(d - h * v)) / (2 * h)
        assert (diff - (dx * v).sum()).abs() <= 2 ** -16 * (dx * v).abs().sum() + 1e-6
