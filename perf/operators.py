"""Cases of the language-model operators: layer norm (forward, backward), the log
probabilities of given tokens (forward, backward) and gradient clipping.

With ``own`` false, run() computes an operator in elementary torch operations;
with ``own`` true it makes the calls of the mcke package.
"""
import functools
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # the norm of one decoded token (the width of the benchmark's DAG): launch latency
        {"name": "ln_fwd_token", "op": "ln_fwd", "rows": 1, "cols": 4096, "type": "bf16"},
        # a batch of prompts, rows as wide as the DAG's input
        {"name": "ln_fwd_bf16", "op": "ln_fwd", "rows": 8192, "cols": 4096, "type": "bf16"},
        # f32 rows of an odd width, whose rows start at every alignment
        {"name": "ln_fwd_f32_odd", "op": "ln_fwd", "rows": 5003, "cols": 1537, "type": "f32"},
        # a small f32 model's step: few rows, where the columns' sums have little to split
        {"name": "ln_bwd_f32_small", "op": "ln_bwd", "rows": 250, "cols": 1024, "type": "f32"},
        # the training step of the same rows
        {"name": "ln_bwd_bf16", "op": "ln_bwd", "rows": 8192, "cols": 4096, "type": "bf16"},
        # the widest rows of the framework's tables
        {"name": "ln_bwd_bf16_wide", "op": "ln_bwd", "rows": 4096, "cols": 16384, "type": "bf16"},
        # one decoded token: its log probability, the entropy and twenty alternatives
        {"name": "lp_fwd_token", "op": "lp_fwd", "rows": 1, "cols": 131072, "type": "bf16", "top_k": 20, "masked": 1000},
        # a training batch: the given tokens' log probabilities and the entropy
        {"name": "lp_fwd_bf16", "op": "lp_fwd", "rows": 8192, "cols": 32768, "type": "bf16", "top_k": 0, "masked": 0},
        # prompt scoring with alternatives over an odd vocabulary of f32 logits
        {"name": "lp_fwd_f32_odd", "op": "lp_fwd", "rows": 1023, "cols": 50257, "type": "f32", "top_k": 5, "masked": 100},
        # the gradient of a training batch's log probabilities and entropies
        {"name": "lp_bwd_bf16", "op": "lp_bwd", "rows": 4096, "cols": 50257, "type": "bf16", "masked": 57},
        # a large model's step: bf16 gradients of matrices and vectors, clipped into other buffers
        {"name": "clip_bf16", "op": "clip", "tensors": 60, "largest": 33554432, "type": "bf16", "clipped": True},
        # a small model's step, whose norm is below the limit: clipped in place
        {"name": "clip_f32_small", "op": "clip", "tensors": 37, "largest": 1048577, "type": "f32", "clipped": False},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm; odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "lp_fwd", "lp_bwd", "clip"])
    kind = rng.choice(["f32", "bf16"])
    if op == "clip":
        return {"op": op, "tensors": _between(rng, 3, 60), "largest": _between(rng, 1000, 20000000), "type": kind,
                "clipped": rng.random() < 0.5}
    if op in ("ln_fwd", "ln_bwd"):
        cols = _between(rng, 64, 20000)
        if rng.random() < 0.6:  # most widths are round
            cols = max(64, cols // 64 * 64)
        return {"op": op, "rows": _between(rng, 1, min(16384, 2 ** 25 // cols)), "cols": cols, "type": kind}
    cols = _between(rng, 1000, 200000)
    if rng.random() < 0.5:
        cols = max(1024, cols // 128 * 128)
    case = {"op": op, "rows": _between(rng, 1, min(8192, 2 ** 27 // cols)), "cols": cols, "type": kind,
            "masked": rng.choice([0, 1, 64, cols // 10])}
    if op == "lp_fwd":
        case["top_k"] = rng.choice([0, 1, 3, 8, 20])
    return case


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _sizes(case):
    """Tensor sizes of a step: every fourth a matrix, the rest vectors and smaller matrices, none of them round."""
    n, top = case["tensors"], case["largest"]
    parts = [1.0, 0.001, 0.03, 0.0005]
    return [max(1, int(top * parts[i % 4]) - 3 * (i % 5)) for i in range(n)]


def prepare(case, seed):
    g = _gen(seed)
    op, t = case["op"], TYPES[case["type"]]
    if op == "clip":
        # gradients of a step: each tensor has a scale of its own
        sizes = _sizes(case)
        scales = (_randn(g, len(sizes)).exp() * 1e-3).tolist()
        grads = [(_randn(g, n) * s).to(t) for n, s in zip(sizes, scales)]
        norm = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
        # the limit that the user sets: half of this step's norm, or twice
        state = {"grads": grads, "max_norm": norm * (0.5 if case["clipped"] else 2.0)}
        state["out"] = [torch.empty_like(x) for x in grads] if case["clipped"] else None
        return {"op": op, **state}
    rows, cols = case["rows"], case["cols"]
    if op in ("ln_fwd", "ln_bwd"):
        # activations of a residual stream: a mean that is not zero and a few loud channels
        x = _randn(g, rows, cols)
        x[:, ::61] *= 8.0
        x = (x + _randn(g, rows, 1)).to(t)
        state = {"x": x, "weight": 1.0 + 0.1 * _randn(g, cols), "bias": 0.1 * _randn(g, cols)}
        if op == "ln_bwd":
            state["dy"] = (_randn(g, rows, cols) * 1e-2).to(t)
            d = x.double()
            mean = d.mean(1, keepdim=True)
            var = (d - mean).square_().mean(1)
            state["mean"], state["rstd"] = mean.squeeze(1).float(), (var + EPS).rsqrt().float()
        return {"op": op, **state}
    # logits: a wide spread, a row's own offset, the given token among the likelier ones, some tokens forbidden
    x = _randn(g, rows, cols).mul_(2.5)
    x += 3.0 * _randn(g, rows, 1)
    targets = torch.randint(0, cols - case["masked"], (rows,), generator=g, device=DEV)
    x[torch.arange(rows, device=DEV), targets] += 6.0
    if case["masked"]:
        x[:, cols - case["masked"]:] = -math.inf
    x = x.to(t)
    if rows > 8:
        targets[torch.rand(rows, generator=g, device=DEV) < 0.05] = -100  # padding
    state = {"logits": x, "targets": targets}
    if op == "lp_fwd":
        state["top_k"] = case["top_k"]
    else:
        state["lse"], state["entropy"] = (v.float() for v in _stats64(x))
        state["grad_logprobs"] = _randn(g, rows) / rows
        state["grad_entropy"] = 0.01 * _randn(g, rows) / rows
    return {"op": op, **state}


def _rows_at_once(cols):
    return max(1, 2 ** 26 // cols)


def _stats64(x):
    """lse and entropy of the rows of x in 64 bits."""
    lse, ent = [], []
    for part in x.split(_rows_at_once(x.shape[1])):
        p = part.double()
        l = torch.logsumexp(p, 1, keepdim=True)
        q = p - l
        lse.append(l.squeeze(1))
        ent.append(-(q.exp() * torch.where(q == -math.inf, 0.0, q)).sum(1))
    return torch.cat(lse), torch.cat(ent)


# ---- one pass ------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


@functools.cache
def _mcke():
    pkg = os.path.join(os.getcwd(), "mini-cuda-kernel-engine_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mcke

    return mcke


def _run_own(s):
    mcke = _mcke()
    if s["op"] == "ln_fwd":
        y, mean, rstd = mcke.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, save_stats=True)
        return {"y": y, "mean": mean, "rstd": rstd}
    if s["op"] == "ln_bwd":
        dx, dw, db = mcke.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
        return {"dx": dx, "dweight": dw, "dbias": db}
    if s["op"] == "lp_fwd":
        r = mcke.token_logprobs(s["logits"], s["targets"], top_k=s["top_k"], entropy=True)
        out = {"logprobs": r.logprobs, "lse": r.lse, "entropy": r.entropy}
        if s["top_k"]:
            out.update(top_logprobs=r.top_logprobs, top_ids=r.top_ids)
        return out
    if s["op"] == "lp_bwd":
        return {"dlogits": mcke.token_logprobs_backward(s["logits"], s["lse"], s["targets"],
                                                        grad_logprobs=s["grad_logprobs"], entropy=s["entropy"],
                                                        grad_entropy=s["grad_entropy"])}
    norm = mcke.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"])
    return [norm] + (s["out"] or s["grads"])


def _run_plain(s):
    return {"ln_fwd": _plain_ln_fwd, "ln_bwd": _plain_ln_bwd, "lp_fwd": _plain_lp_fwd, "lp_bwd": _plain_lp_bwd,
            "clip": _plain_clip}[s["op"]](s)


def _plain_ln_fwd(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = (xc.square().mean(1, keepdim=True) + EPS).rsqrt()
    y = xc * rstd * s["weight"] + s["bias"]
    return {"y": y.to(s["x"].dtype), "mean": mean.squeeze(1), "rstd": rstd.squeeze(1)}


def _plain_ln_bwd(s):
    x, dy = s["x"].float(), s["dy"].float()
    rstd = s["rstd"][:, None]
    xh = (x - s["mean"][:, None]) * rstd
    g = dy * s["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dweight": (dy * xh).sum(0), "dbias": dy.sum(0)}


def _plain_lp_fwd(s):
    x = s["logits"].float()
    m = x.amax(1, keepdim=True)
    d = x - m
    e = d.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    t = s["targets"]
    given = d.gather(1, t.clamp(min=0)[:, None]) - log_total
    out = {"logprobs": torch.where(t >= 0, given.squeeze(1), 0.0),
           "lse": (m + log_total).squeeze(1),
           "entropy": (log_total - (e * torch.where(d == -math.inf, 0.0, d)).sum(1, keepdim=True) / total).squeeze(1)}
    if s["top_k"]:
        value, at = torch.sort(d, dim=1, descending=True, stable=True)
        out.update(top_logprobs=value[:, :s["top_k"]] - log_total, top_ids=at[:, :s["top_k"]].contiguous())
    return out


def _plain_lp_bwd(s):
    x, t = s["logits"].float(), s["targets"]
    q = x - s["lse"][:, None]
    p = q.exp()
    g = torch.where(t >= 0, s["grad_logprobs"], 0.0)
    dx = p * (-g[:, None] - s["grad_entropy"][:, None] * (torch.where(q == -math.inf, 0.0, q) + s["entropy"][:, None]))
    dx.scatter_add_(1, t.clamp(min=0)[:, None], g[:, None])
    return {"dlogits": dx.to(s["logits"].dtype)}


def _plain_clip(s):
    squares = torch.stack([x.float().square().sum() for x in s["grads"]])
    norm = squares.sum().sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    to = s["out"] or s["grads"]
    done = [o.copy_(x.float() * coef) for x, o in zip(s["grads"], to)]
    return [norm] + done


# ---- bytes and operations that a pass cannot do without ----------------------------------


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "clip":
        n = sum(_sizes(case))
        # clipped: one read and one write; below the limit the tensors stay as they are
        return {"bytes": n * size * (2 if case["clipped"] else 1) + 4, "flops": n * (3 if case["clipped"] else 2)}
    rows, cols = case["rows"], case["cols"]
    n = rows * cols
    if case["op"] == "ln_fwd":
        return {"bytes": 2 * n * size + 8 * cols + 8 * rows, "flops": 8 * n}
    if case["op"] == "ln_bwd":
        return {"bytes": 3 * n * size + 12 * cols + 8 * rows, "flops": 15 * n}
    if case["op"] == "lp_fwd":
        return {"bytes": n * size + rows * (20 + 12 * case["top_k"]), "flops": 6 * n}
    return {"bytes": 2 * n * size + 24 * rows, "flops": 7 * n}


# ---- the definitions in 64 bits --------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        total = math.fsum(float((x.double() ** 2).sum()) for x in s["grads"])
        norm = math.sqrt(total)
        c = min(1.0, s["max_norm"] / (norm + 1e-6))
        return [torch.tensor(norm, dtype=torch.float64)] + [x.double() * c for x in s["grads"]]
    if op == "ln_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        y = (x - mean[:, None]) / torch.sqrt(var[:, None] + EPS) * s["weight"].double() + s["bias"].double()
        return {"y": y, "mean": mean, "rstd": 1.0 / torch.sqrt(var + EPS)}
    if op == "ln_bwd":
        x, dy, w = s["x"].double(), s["dy"].double(), s["weight"].double()
        mean, rstd, n = s["mean"].double(), s["rstd"].double(), case["cols"]
        z = (x - mean[:, None]) * rstd[:, None]
        dz = dy * w
        a, b = dz.sum(1) / n, torch.einsum("rc,rc->r", dz, z) / n
        return {"dx": (dz - a[:, None] - z * b[:, None]) * rstd[:, None],
                "dweight": torch.einsum("rc,rc->c", dy, z), "dbias": dy.sum(0)}
    x, t = s["logits"], s["targets"]
    parts = []
    for at in range(0, x.shape[0], _rows_at_once(x.shape[1])):
        rows = slice(at, at + _rows_at_once(x.shape[1]))
        d, tt = x[rows].double(), t[rows]
        hit = tt >= 0
        if op == "lp_bwd":
            lse, h = s["lse"][rows].double()[:, None], s["entropy"][rows].double()[:, None]
            g = (s["grad_logprobs"][rows].double() * hit)[:, None]
            ge = s["grad_entropy"][rows].double()[:, None]
            lp = d - lse
            p = lp.exp()
            dx = p * lp.clamp(min=-1e6) * -ge - p * (g + ge * h)
            dx[torch.arange(len(tt), device=dx.device), tt.clamp(min=0)] += g.squeeze(1)
            parts.append({"dlogits": dx.to(torch.float64)})
            continue
        lp = torch.log_softmax(d, dim=1)
        got = {"logprobs": lp[torch.arange(len(tt), device=lp.device), tt.clamp(min=0)] * hit,
               "lse": torch.logsumexp(d, dim=1), "entropy": -(lp.exp() * lp.clamp(min=-1e6)).sum(1)}
        if case["top_k"]:
            # value first, lowest index first among equals
            order = torch.argsort(d, dim=1, descending=True, stable=True)[:, :case["top_k"]]
            got.update(top_logprobs=lp.gather(1, order), top_ids=order.contiguous())
        parts.append(got)
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
