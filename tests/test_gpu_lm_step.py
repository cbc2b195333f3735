"""The language-model operators as they are used together: the end of a training
step (layer norm -> product -> token log probabilities, their gradients, clipping),
captured into a CUDA graph, on other streams, and several at a time."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

import mcke  # noqa: E402

DEV = "cuda"
ROWS, WIDTH, VOCAB = 96, 256, 1000
NAMES = ("loss rows", "entropy", "dhidden", "dgamma", "dbeta", "dhead", "norm")


def _inputs(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(ROWS, WIDTH, generator=g, device=DEV)
    gamma, beta = 1 + 0.1 * torch.randn(WIDTH, generator=g, device=DEV), 0.1 * torch.randn(WIDTH, generator=g, device=DEV)
    head = 0.2 * torch.randn(WIDTH, VOCAB, generator=g, device=DEV)
    t = torch.randint(0, VOCAB, (ROWS,), generator=g, device=DEV)
    t[::10] = -100
    return [x, gamma, beta, head, t]


def _step(x, gamma, beta, head, targets, max_norm=0.05, stream=None):
    """Gradients, clipped to max_norm, of the mean of -logprobs - 0.01 * entropy."""
    kept = (targets >= 0).sum()
    g_lp = (-1.0 / kept).expand(ROWS).contiguous()
    g_h = torch.full((ROWS,), -0.01 / ROWS, device=x.device)
    h, mean, rstd = mcke.layer_norm(x, gamma, beta, save_stats=True, stream=stream)
    logits = mcke.gemm(h, head, stream=stream)
    r = mcke.token_logprobs(logits, targets, entropy=True, stream=stream)
    dlogits = mcke.token_logprobs_backward(logits, r.lse, targets, g_lp, r.entropy, g_h, out=logits, stream=stream)
    dh = mcke.gemm(dlogits, head.t().contiguous(), stream=stream)
    dhead = mcke.gemm(h.t().contiguous(), dlogits, stream=stream)
    dx, dgamma, dbeta = mcke.layer_norm_backward(dh, x, mean, rstd, gamma, stream=stream)
    norm = mcke.clip_grad_norm([dx, dgamma, dbeta, dhead], max_norm, stream=stream)
    return r.logprobs, r.entropy, dx, dgamma, dbeta, dhead, norm


def _want(x, gamma, beta, head, targets, max_norm=0.05):
    leaves = [v.double().requires_grad_() for v in (x, gamma, beta, head)]
    h = torch.nn.functional.layer_norm(leaves[0], (WIDTH,), leaves[1], leaves[2])
    lp = torch.log_softmax(h @ leaves[3], 1)
    given = lp.gather(1, targets.clamp(min=0)[:, None]).squeeze(1) * (targets >= 0)
    ent = -(lp.exp() * lp).sum(1)
    (-given.sum() / (targets >= 0).sum() - 0.01 * ent.mean()).backward()
    grads = [v.grad for v in leaves]
    norm = torch.sqrt(sum(g.square().sum() for g in grads))
    c = min(1.0, max_norm / (float(norm) + 1e-6))
    return [given.detach(), ent.detach()] + [g * c for g in grads] + [norm]


def _close(got, want):
    # the products are f32 with a relative error of a few 2^-20 per element (3xTF32
    # over 256 and 1000 terms); logits of magnitude 10 pass an absolute 1e-5 on to p.
    # 2^-13 of each result's 2-norm holds that with a wide margin for what follows.
    for name, a, b in zip(NAMES, got, want):
        err = (a.double() - b).norm() / b.norm()
        assert err <= 2 ** -13, (name, float(err))


def test_step_against_autograd_in_64_bits():
    for seed in (0, 1):
        ins = _inputs(seed)
        _close(_step(*ins), _want(*ins))


def test_step_in_bf16():
    """The same run on bf16 activations: rounding h, logits and their gradients to
    bf16 (2^-9 each, relative) moves the results by a few of those."""
    x, gamma, beta, head, t = _inputs(2)
    xb, hb = x.bfloat16(), head.bfloat16()
    h, mean, rstd = mcke.layer_norm(xb, gamma, beta, save_stats=True)
    logits = mcke.gemm(h, hb, out_dtype=torch.bfloat16)
    r = mcke.token_logprobs(logits, t, top_k=3, entropy=True)
    g = torch.full((ROWS,), -1.0 / int((t >= 0).sum()), device=DEV)
    dlogits = mcke.token_logprobs_backward(logits, r.lse, t, g)
    dh = mcke.gemm(dlogits, hb.t().contiguous(), out_dtype=torch.bfloat16)
    dx, dgamma, dbeta = mcke.layer_norm_backward(dh, xb, mean, rstd, gamma)
    leaves = [v.double().requires_grad_() for v in (xb, gamma, beta)]
    lp = torch.log_softmax(torch.nn.functional.layer_norm(leaves[0], (WIDTH,), leaves[1], leaves[2]) @ hb.double(), 1)
    given = lp.gather(1, t.clamp(min=0)[:, None]).squeeze(1) * (t >= 0)
    (-given.sum() / (t >= 0).sum()).backward()
    assert (r.logprobs.double() - given).norm() <= 2 ** -6 * given.norm()
    for got, leaf in zip((dx, dgamma, dbeta), leaves):
        assert (got.double() - leaf.grad).norm() <= 2 ** -5 * leaf.grad.norm()


def test_step_in_a_captured_graph():
    ins = _inputs(3)
    eager = [v.clone() for v in _step(*ins)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*ins)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(*ins)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, eager))
    fresh = _inputs(4)
    want = [v.clone() for v in _step(*fresh)]
    for a, b in zip(ins, fresh):
        a.copy_(b)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_graphs_at_once():
    """Each capture has its own buffers and workspaces: replayed side by side they
    give what they give alone."""
    sets = [_inputs(5), _inputs(6)]
    want = [[v.clone() for v in _step(*ins)] for ins in sets]
    graphs, outs = [], []
    for ins in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(*ins))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_explicit_streams_and_eager_calls_at_once():
    sets = [_inputs(s) for s in (7, 8, 9)]
    want = [[v.clone() for v in _step(*ins)] for ins in sets]
    torch.cuda.synchronize()
    for raw in (False, True):
        streams = [torch.cuda.Stream() for _ in sets]
        got = []
        for _ in range(5):
            got = []
            for ins, s in zip(sets, streams):
                with torch.cuda.stream(s):
                    got.append(_step(*ins, stream=s.cuda_stream if raw else s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))
    # a stream that is not the current one, for one call
    s = torch.cuda.Stream()
    x, gamma, beta, _, _ = sets[0]
    y = mcke.layer_norm(x, gamma, beta, stream=s)
    s.synchronize()
    assert torch.equal(y, mcke.layer_norm(x, gamma, beta))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_device():
    ins = _inputs(10)
    want = _step(*ins)
    other = [v.to("cuda:1") for v in ins]
    x, gamma, beta = other[:3]
    y, mean, rstd = mcke.layer_norm(x, gamma, beta, save_stats=True)
    r = mcke.token_logprobs(y, top_k=3)
    n = mcke.grad_norm([x])
    assert torch.cuda.current_device() == 0 and y.device == r.lse.device == n.device == x.device
    assert torch.equal(y.cpu(), mcke.layer_norm(*ins[:3]).cpu()) and want[0].device.index == 0


def test_mixed_devices_are_refused():
    x = torch.randn(4, 64, device=DEV)
    for bad in (torch.ones(64), torch.ones(63, device=DEV), torch.ones(64, device=DEV, dtype=torch.float64)):
        with pytest.raises(ValueError, match="weight"):
            mcke.layer_norm(x, bad)
    with pytest.raises(ValueError, match="targets"):
        mcke.token_logprobs(x, torch.zeros(4, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="contiguous"):
        mcke.token_logprobs(x.t())
    with pytest.raises(ValueError, match="float32"):
        mcke.layer_norm(x.half())
    with pytest.raises(ValueError, match="shape"):
        mcke.layer_norm(x, out=x.new_empty(4, 63))
    with pytest.raises(mcke.MckeError, match="top_k"):
        mcke.token_logprobs(x, top_k=33)
    with pytest.raises(mcke.MckeError, match="overlaps"):
        mcke.layer_norm(x, out=x)


def test_programmatic_launches_change_nothing():
    ins = _inputs(11)
    on = [v.clone() for v in _step(*ins)]
    was = mcke.set_programmatic_launch(False)
    try:
        off = [v.clone() for v in _step(*ins)]
    finally:
        mcke.set_programmatic_launch(was)
    assert all(torch.equal(a, b) for a, b in zip(on, off))
