"""Refusals of the language-model operators (layer norm, token log probabilities,
gradient norm and clipping) through the C-ABI: every check comes before a
device is touched, so this runs without a GPU."""
from __future__ import annotations

import ctypes
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mini-cuda-kernel-engine_b200")

NAN, INF = float("nan"), float("inf")
A, B, C, D, E, F = (0x100000 * (i + 1) for i in range(6))  # never dereferenced: 1 MB apart
WS = 0x10000000


@pytest.fixture(scope="module")
def mcke():
    import mcke as m
    if not os.path.exists(m.LIB_PATH):
        subprocess.run([sys.executable, os.path.join(PKG, "build.py")], check=True)
    return m


def _refused(mcke, rc, text):
    assert rc == mcke.INVALID_ARGUMENT
    msg = mcke.lib().mcke_sm100_last_error_string().decode()
    assert text in msg, msg


def _forward(mcke, x=A, xs=64, w=None, b=None, y=B, ys=64, mean=None, rstd=None, rows=4, cols=64, eps=1e-5, dtype=0):
    return mcke.lib().mcke_sm100_layer_norm(x, xs, w, b, y, ys, mean, rstd, rows, cols, eps, dtype, None)


@pytest.mark.parametrize("args, text", [
    (dict(x=None), "null"),
    (dict(y=None), "null"),
    (dict(rows=-1), "negative"),
    (dict(cols=-1), "negative"),
    (dict(cols=1 << 31, xs=1 << 31, ys=1 << 31), "INT32_MAX"),
    (dict(dtype=1), "dtype"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=NAN), "eps"),
    (dict(eps=INF), "eps"),
    (dict(ys=63), "row stride"),
    (dict(xs=-64), "row stride"),
    (dict(xs=1 << 60), "2^40"),
    (dict(x=A + 2), "x is not element-aligned"),
    (dict(w=C + 2), "weight is not element-aligned"),
    (dict(mean=C + 1), "mean is not element-aligned"),
    (dict(rows=(1 << 31) - 1, xs=0, ys=64), "INT32_MAX"),
    (dict(y=A), "overlaps"),
    (dict(y=A + 4 * 63), "overlaps"),
    (dict(mean=A), "mean overlaps x"),
    (dict(mean=C, rstd=C + 12), "rstd overlaps mean"),
    (dict(w=B), "y overlaps weight"),
    # two windows of one buffer that share a column
    (dict(x=A, y=A + 4 * 63, xs=128, ys=128), "overlaps"),
])
def test_layer_norm_refuses(mcke, args, text):
    _refused(mcke, _forward(mcke, **args), text)


def test_layer_norm_of_nothing(mcke):
    assert _forward(mcke, x=None, y=None, rows=0) == mcke.OK
    assert _forward(mcke, x=None, y=None, cols=0) == mcke.OK


def _backward(mcke, dy=A, x=B, dx=C, dys=64, xs=64, dxs=64, w=None, mean=D, rstd=D + 0x1000, dw=E, db=E + 0x1000,
              rows=4, cols=64, dtype=0, ws=WS, nbytes=None):
    need = mcke.layer_norm_backward_workspace_bytes(rows, cols)
    return mcke.lib().mcke_sm100_layer_norm_backward(dy, dys, x, xs, w, mean, rstd, dx, dxs, dw, db, rows, cols, dtype,
                                                     ws, need if nbytes is None else nbytes, None)


@pytest.mark.parametrize("args, text", [
    (dict(dy=None), "null"), (dict(x=None), "null"), (dict(dx=None), "null"), (dict(mean=None), "null"),
    (dict(rstd=None), "null"), (dict(rows=-1), "negative"), (dict(dtype=3), "dtype"),
    (dict(ws=None), "workspace"), (dict(nbytes=16), "workspace"), (dict(ws=WS + 8), "workspace"),
    (dict(dxs=32), "row stride"), (dict(dx=B), "dx overlaps x"), (dict(dx=A), "dx overlaps dy"),
    (dict(dw=A), "dweight overlaps dy"), (dict(db=E), "dbias overlaps dweight"), (dict(ws=A), "workspace overlaps dy"),
    (dict(dx=C + 1), "aligned"),
])
def test_layer_norm_backward_refuses(mcke, args, text):
    _refused(mcke, _backward(mcke, **args), text)


def _logprobs(mcke, x=A, stride=64, rows=4, cols=64, dtype=0, targets=B, lp=C, lse=C + 0x1000, ent=C + 0x2000, k=3,
              top=D, ids=E):
    return mcke.lib().mcke_sm100_token_logprobs(x, stride, rows, cols, dtype, targets, lp, lse, ent, k, top, ids, None)


@pytest.mark.parametrize("args, text", [
    (dict(x=None), "null"), (dict(targets=None), "null"), (dict(top=None), "null"), (dict(ids=None), "null"),
    (dict(rows=-4), "negative"), (dict(cols=0), "no columns"), (dict(dtype=1), "dtype"),
    (dict(k=-1), "top_k"), (dict(k=33), "top_k"), (dict(k=5, cols=4), "top_k"),
    (dict(stride=-1), "row stride"), (dict(x=A + 3), "aligned"), (dict(targets=B + 4), "targets is not"),
    (dict(cols=(1 << 22) + 1, stride=1 << 23), "top_k of more than"), (dict(ids=E + 4), "top_ids is not"),
    (dict(lp=A), "logprobs overlaps logits"), (dict(lse=C + 4), "lse overlaps logprobs"),
    (dict(ids=D), "top_ids overlaps top_logprobs"), (dict(ent=B), "entropy overlaps targets"),
])
def test_token_logprobs_refuses(mcke, args, text):
    _refused(mcke, _logprobs(mcke, **args), text)


def test_token_logprobs_of_nothing(mcke):
    assert _logprobs(mcke, x=None, rows=0) == mcke.OK
    assert _logprobs(mcke, lp=None, lse=None, ent=None, k=0) == mcke.OK


def _logprobs_backward(mcke, x=A, stride=64, rows=4, cols=64, dtype=0, lse=B, targets=C, g=D, ent=E, ge=E + 0x1000,
                       gl=None, dx=F, dxs=64):
    return mcke.lib().mcke_sm100_token_logprobs_backward(x, stride, rows, cols, dtype, lse, targets, g, ent, ge, gl, dx,
                                                         dxs, None)


@pytest.mark.parametrize("args, text", [
    (dict(x=None), "null"), (dict(lse=None), "null"), (dict(dx=None), "null"), (dict(targets=None), "null"),
    (dict(ent=None), "null"), (dict(g=None, ge=None), "no gradient"), (dict(dxs=63), "row stride"),
    (dict(dx=A + 4), "overlaps"), (dict(dx=A, dxs=80), "overlaps"), (dict(dx=D), "dlogits overlaps grad_logprobs"),
    (dict(dx=F + 2), "aligned"), (dict(rows=1 << 31), "INT32_MAX"),
])
def test_token_logprobs_backward_refuses(mcke, args, text):
    _refused(mcke, _logprobs_backward(mcke, **args), text)


def _list(mcke, *grads):
    arr = (mcke.Grad * max(len(grads), 1))(*grads)
    return ctypes.cast(arr, ctypes.c_void_p), len(grads), arr


BF16, F32 = 2, 0


@pytest.mark.parametrize("grads, text", [
    ([(A, A, -1, F32, F32)], "negative"),
    ([(A, A, 8, 1, F32)], "dtype"),
    ([(A, B, 8, F32, BF16)], "not clipped into bf16"),
    ([(None, A, 8, F32, F32)], "null"),
    ([(A, None, 8, F32, F32)], "null"),
    ([(A + 2, B, 8, F32, F32)], "aligned"),
    ([(A, A, 8, F32, F32), (A, A, 8, F32, F32)], "overlaps"),              # the same tensor twice, in place
    ([(A, A, 8, F32, F32), (A + 28, A + 28, 8, F32, F32)], "overlaps"),    # the last element shared
    ([(A, B, 8, F32, F32), (A, B + 16, 8, F32, F32)], "overlaps"),         # outputs share bytes
    ([(A, A, 8, BF16, F32)], "overlaps"),                                  # in place, but of another size
    ([(A, A + 4, 8, F32, F32)], "overlaps"),
    ([(A, C, 1 << 41, F32, F32)], "too large"),
    ([(A, WS, 8, F32, F32)], "overlaps"),
    ([(A, D, 8, F32, F32)], "overlaps"),                                   # the norm's own place
])
def test_clip_grad_norm_refuses(mcke, grads, text):
    p, n, _ = _list(mcke, *grads)
    _refused(mcke, mcke.lib().mcke_sm100_clip_grad_norm(p, n, 1.0, D, WS, 1 << 20, None), text)


def test_clip_arguments(mcke):
    l = mcke.lib()
    p, n, _ = _list(mcke, (A, A, 8, F32, F32))
    for bad in (-1.0, NAN, INF):
        _refused(mcke, l.mcke_sm100_clip_grad_norm(p, n, bad, D, WS, 1 << 20, None), "max_norm")
        _refused(mcke, l.mcke_sm100_clip_grads(p, n, bad, D, None), "max_norm")
    _refused(mcke, l.mcke_sm100_clip_grad_norm(p, n, 1.0, None, WS, 1 << 20, None), "norm")
    _refused(mcke, l.mcke_sm100_clip_grad_norm(p, n, 1.0, D, WS, 64, None), "workspace")
    _refused(mcke, l.mcke_sm100_clip_grad_norm(p, n, 1.0, D, WS + 8, 1 << 20, None), "workspace")
    _refused(mcke, l.mcke_sm100_clip_grad_norm(None, 2, 1.0, D, WS, 1 << 20, None), "null list")
    _refused(mcke, l.mcke_sm100_grad_norm(p, -1, D, WS, 1 << 20, None), "negative")
    _refused(mcke, l.mcke_sm100_grad_norm(p, n, A, WS, 1 << 20, None), "overlaps")
    _refused(mcke, l.mcke_sm100_clip_grads(p, n, 1.0, A + 4, None), "overlaps")
    _refused(mcke, l.mcke_sm100_clip_grads(p, n, 1.0, D + 2, None), "aligned")
    assert l.mcke_sm100_clip_grads(None, 0, 1.0, D, None) == mcke.OK


def test_workspace_queries(mcke):
    assert mcke.layer_norm_backward_workspace_bytes(0, 64) == 0
    assert mcke.layer_norm_backward_workspace_bytes(64, 0) == 0
    assert mcke.layer_norm_backward_workspace_bytes(3, 64) >= 2 * 64 * 4
    # the workspace does not grow with the rows
    assert mcke.layer_norm_backward_workspace_bytes(1 << 20, 64) == mcke.layer_norm_backward_workspace_bytes(1 << 21, 64)
    assert mcke.grad_norm_workspace_bytes(1) == mcke.grad_norm_workspace_bytes(1000)
    assert mcke.grad_norm_workspace_bytes(1001) == 2 * mcke.grad_norm_workspace_bytes(1)


def test_python_checks_need_no_device(mcke):
    import torch
    x = torch.zeros(4, 8)
    for call in (lambda: mcke.layer_norm(x), lambda: mcke.layer_norm_backward(x, x, x, x),
                 lambda: mcke.token_logprobs(x), lambda: mcke.token_logprobs_backward(x, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="empty"):
        mcke.grad_norm([])
    with pytest.raises(ValueError, match="CUDA"):
        mcke.grad_norm([x])
    with pytest.raises(ValueError, match="outputs"):
        mcke.clip_grad_norm([x], 1.0, out=[])
