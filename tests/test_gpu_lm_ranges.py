"""The language-model operators over the rest of their ranges: every kernel that a
size chooses (rows over clusters of blocks, rows to a warp, rows by the element),
offsets past 32 bits, very many rows, and those kernels in captured graphs and on
several streams at once.  Oracles and tolerances are those of the operators' own
tests."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

import mcke  # noqa: E402
import test_gpu_grad_norm as gn  # noqa: E402
import test_gpu_layer_norm as ln  # noqa: E402
import test_gpu_token_logprobs as lp  # noqa: E402

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols", [(593, 8), (2000, 512), (1201, 520), (900, 1544), (1000, 2048), (777, 2056), (640, 4096),
                                        (600, 5128), (999, 6144), (595, 8192), (601, 8200), (777, 12288), (650, 16384),
                                        (600, 20000), (613, 24576), (594, 32768), (600, 8193), (1300, 4097), (700, 127),
                                        (600, 40000)])
def test_layer_norm_of_many_rows(rows, cols, dtype):
    x, w, b, dy = ln._inputs(rows, cols, dtype, seed=rows)
    y, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True)
    ln._check_forward(x, w, b, y, mean, rstd)
    again, _, _ = mcke.layer_norm(x, w, b, save_stats=True)
    assert torch.equal(y, again)
    dx, dw, db = mcke.layer_norm_backward(dy, x, mean, rstd, w)
    ln._check_backward(x, w, mean, rstd, dy, dx, dw, db)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), mcke.layer_norm_backward(dy, x, mean, rstd, w)))
    mcke.check_device_errors()  # no wait of the posted sums ran out


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols", [(600, 8193), (601, 12289), (149, 12287), (1, 8201), (297, 16383), (600, 16385),
                                        (299, 20001), (3, 24577), (65, 24575), (595, 32767), (40, 32769), (2, 20001)])
def test_layer_norm_of_wide_odd_rows(rows, cols, dtype):
    x, w, b, dy = ln._inputs(rows, cols, dtype, seed=cols)
    y, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True)
    ln._check_forward(x, w, b, y, mean, rstd)
    dx, dw, db = mcke.layer_norm_backward(dy, x, mean, rstd, w)
    ln._check_backward(x, w, mean, rstd, dy, dx, dw, db)
    # rows of another stride: the same kernel, the same bits
    apart = torch.full((rows, cols + 3), float("nan"), dtype=dtype, device=DEV)
    apart[:, :cols] = x
    out = torch.full_like(apart, 7.0)
    again = mcke.layer_norm_backward(dy, apart[:, :cols], mean, rstd, w, out=out[:, :cols])
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))
    assert bool((out[:, cols:] == 7.0).all())
    # whole units that start off a 16-byte boundary
    odd = torch.empty(rows * (cols // 8 * 8) + 1, dtype=dtype, device=DEV)[1:].view(rows, cols // 8 * 8)
    odd.copy_(x[:, : cols // 8 * 8])
    y, mean, rstd = mcke.layer_norm(odd, save_stats=True)
    ln._check_forward(odd, None, None, y, mean, rstd)
    mcke.check_device_errors()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols", [(1, 16392), (2, 17408), (3, 24576), (75, 20000), (149, 20000), (400, 16400),
                                        (30, 8200), (1, 12288), (33, 24584), (1, 32768), (599, 18440)])
def test_layer_norm_of_few_wide_rows(rows, cols, dtype):
    x, w, b, dy = ln._inputs(rows, cols, dtype, seed=cols + rows)
    y, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True)
    ln._check_forward(x, w, b, y, mean, rstd)
    out = torch.full((rows, cols + 8), 7.0, dtype=dtype, device=DEV)
    mcke.layer_norm(x, w, b, out=out[:, :cols])
    assert torch.equal(out[:, :cols], y) and bool((out[:, cols:] == 7.0).all())
    ln._check_backward(x, w, mean, rstd, dy, *mcke.layer_norm_backward(dy, x, mean, rstd, w))
    mcke.check_device_errors()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols, k", [(18, 200000, 32), (19, 200000, 32), (74, 131072, 9), (149, 70001, 8),
                                           (1184, 2048, 5), (1183, 2048, 5), (1500, 4096, 32), (1500, 4104, 32),
                                           (3000, 24, 20), (888, 40000, 0), (889, 40000, 1), (2, 1 << 22, 4)])
def test_token_logprobs_by_size(rows, cols, k, dtype):
    x, t = lp._logits(rows, cols, dtype, seed=rows + k, masked=0.02)
    t[1::7] = -5
    r = mcke.token_logprobs(x, t, top_k=k, entropy=True)
    lp._check(x, t, r, k)
    gl, ge = torch.randn(2, rows, device=DEV).unbind(0)
    dx = mcke.token_logprobs_backward(x, r.lse, t, gl, r.entropy, ge)
    lp._check_backward(x, t, r.lse, r.entropy, gl, ge, None, dx)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, cols, k", [(1184, 5920, 8), (1184, 5921, 0), (1300, 4736, 1), (3277, 16384, 8), (3300, 16385, 8),
                                           (8000, 4999, 3), (1200, 4500, 20), (5, 4500, 32), (1, 300, 32), (2000, 257, 9),
                                           (3, 33, 32), (40, 8191, 31), (1200, 64, 32), (300, 2560, 20),
                                           (300, 2815, 20), (1300, 5632, 20), (90, 5633, 20), (70, 1152, 8), (1200, 2304, 8)])
def test_token_logprobs_of_rows_to_a_warp(rows, cols, k, dtype):
    x, t = lp._logits(rows, cols, dtype, seed=rows + cols, masked=0.02)
    lp._check(x, t, mcke.token_logprobs(x, t, top_k=k, entropy=True), k)
    if k:
        # all equal, nothing but a few left, a NaN: the first of the equal come first
        flat = torch.full((3, cols), 0.5, dtype=dtype, device=DEV)
        flat[1, 2:] = float("-inf")
        flat[2, cols // 2] = float("nan")
        ids = mcke.token_logprobs(flat, top_k=k).top_ids
        assert ids[0].tolist() == list(range(k)) and ids[1].tolist() == list(range(k))
        assert ids[2].tolist() == [cols // 2] + [i for i in range(k) if i != cols // 2][: k - 1]


def test_offsets_past_32_bits():
    stride = (1 << 31) + 24
    buf = torch.empty(2 * stride, dtype=BF16, device=DEV)
    for cols in (4096, 4097, 16384):
        view = torch.as_strided(buf, (2, cols), (stride, 1))
        x, w, b, dy = ln._inputs(2, cols, BF16, seed=cols)
        view.copy_(x)
        y, mean, rstd = mcke.layer_norm(view, w, b, save_stats=True)
        ln._check_forward(x, w, b, y, mean, rstd)
        out = torch.as_strided(buf, (2, cols), (stride, 1), 1 << 20)
        mcke.layer_norm_backward(dy, view, mean, rstd, w, out=out)
        assert torch.equal(out, mcke.layer_norm_backward(dy, x, mean, rstd, w)[0])
        t = torch.tensor([3, cols - 1], device=DEV)
        r = mcke.token_logprobs(view, t, top_k=3, entropy=True)
        lp._check(x, t, r, 3)
        g = torch.ones(2, device=DEV)
        want = mcke.token_logprobs_backward(x, r.lse, t, g)
        assert torch.equal(mcke.token_logprobs_backward(view, r.lse, t, g, out=out), want)
        assert torch.equal(mcke.token_logprobs_backward(view, r.lse, t, g, out=view), want)
    # one tensor of more than 2^31 elements
    buf.zero_()
    buf[-1] = 3.0
    buf[5] = 4.0
    assert mcke.grad_norm([buf]) == 5.0
    mcke.clip_grad_norm([buf], 2.5)
    assert buf[-1] == 1.5 and buf[5] == 2.0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_very_many_rows(dtype):
    rows = 300007
    x, w, b, dy = ln._inputs(rows, 16, dtype, seed=2)
    y, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True)
    ln._check_forward(x, w, b, y, mean, rstd)
    ln._check_backward(x, w, mean, rstd, dy, *mcke.layer_norm_backward(dy, x, mean, rstd, w))
    t = torch.randint(0, 16, (rows,), device=DEV)
    r = mcke.token_logprobs(x, t, top_k=2, entropy=True)
    lp._check(x, t, r, 2)
    g = torch.randn(rows, device=DEV)
    lp._check_backward(x, t, r.lse, None, g, None, None, mcke.token_logprobs_backward(x, r.lse, t, g))


def _wide(seed):
    """Calls that run over clusters of blocks and with alternatives."""
    x, w, b, dy = ln._inputs(600, 16384, BF16, seed=seed)
    z, t = lp._logits(3, 100000, BF16, seed=seed)
    grads = gn._grads([3000001, 17, 70000], [F32, BF16], seed=seed)
    outs = [torch.empty_like(g) for g in grads]

    def run(stream=None):
        y, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True, stream=stream)
        dx, dw, db = mcke.layer_norm_backward(dy, x, mean, rstd, w, stream=stream)
        r = mcke.token_logprobs(z, t, top_k=20, entropy=True, stream=stream)
        n = mcke.clip_grad_norm(grads, 0.1, out=outs, stream=stream)
        return [y, mean, rstd, dx, dw, db, *r, n, *outs]

    return run


def test_wide_calls_captured_and_at_once():
    calls = [_wide(s) for s in (1, 2, 3)]
    want = [[v.clone() for v in c()] for c in calls]
    torch.cuda.synchronize()
    graphs, got = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(c())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    del graphs
    eager = []
    for _ in range(3):
        eager = [c(stream=s) for c, s in zip(calls, streams)]
    torch.cuda.synchronize()
    for a, b in zip(eager, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    mcke.check_device_errors()
    # the default stream by its handle
    with torch.cuda.stream(streams[0]):
        out = calls[0](stream=0)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, want[0]))


def test_a_workspace_of_the_callers():
    x, w, b, dy = ln._inputs(700, 1024, BF16, seed=9)
    _, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True)
    want = mcke.layer_norm_backward(dy, x, mean, rstd, w)
    ws = torch.full((mcke.layer_norm_backward_workspace_bytes(700, 1024),), 255, dtype=torch.uint8, device=DEV)  # NaNs
    got = mcke.layer_norm_backward(dy, x, mean, rstd, w, workspace=ws)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(mcke.MckeError, match="workspace"):
        mcke.layer_norm_backward(dy, x, mean, rstd, w, workspace=ws[:64])
    grads = [x, w]
    ws = torch.full((mcke.grad_norm_workspace_bytes(2),), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(mcke.grad_norm(grads, workspace=ws), mcke.grad_norm(grads))
    out = torch.zeros((), device=DEV)
    assert mcke.grad_norm(grads, norm=out) is out and out > 0


def test_refusals_of_the_binding():
    x, w, b, dy = ln._inputs(6, 64, F32, seed=1)
    _, mean, rstd = mcke.layer_norm(x, w, b, save_stats=True)
    need = mcke.layer_norm_backward_workspace_bytes(6, 64)
    for ws in (torch.empty(1, dtype=torch.uint8, device=DEV).expand(need),  # one byte, listed need times
               torch.empty(2 * need, dtype=torch.uint8, device=DEV)[::2], torch.empty(need, dtype=torch.uint8)):
        with pytest.raises(ValueError, match="workspace"):
            mcke.layer_norm_backward(dy, x, mean, rstd, w, workspace=ws)
    need = mcke.grad_norm_workspace_bytes(1)
    for f in (mcke.grad_norm, lambda g, workspace: mcke.clip_grad_norm(g, 1.0, workspace=workspace)):
        with pytest.raises(ValueError, match="workspace"):
            f([x], workspace=torch.empty(1, dtype=torch.uint8, device=DEV).expand(need))
    for k in (33, 1 << 40, -1):
        with pytest.raises(mcke.MckeError, match="top_k"):
            mcke.token_logprobs(x, top_k=k)
    with pytest.raises(mcke.MckeError, match="no statistics"):
        mcke.layer_norm(x[:, :0], save_stats=True)
    assert mcke.layer_norm(x[:, :0]).shape == (6, 0)
    assert mcke.layer_norm(x[:0], save_stats=True)[1].shape == (0,)
