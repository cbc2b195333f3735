"""A stream of another device than the tensors' is refused by the language-model
operators, before anything is launched."""
from __future__ import annotations

import types

import pytest

torch = pytest.importorskip("torch")

import mcke  # noqa: E402

OTHER = types.SimpleNamespace(cuda_stream=7, device=torch.device("cuda", 1))


def test_a_stream_of_another_device_is_refused():
    t = types.SimpleNamespace(device=torch.device("cuda", 0), get_device=lambda: 0)
    with pytest.raises(ValueError, match="stream is on cuda:1, the tensors on cuda:0"):
        with mcke._on(t, OTHER):
            pass


def _calls(device):
    x = torch.randn(4, 64, device=device)
    mean = rstd = lse = x.new_zeros(4)
    norm = x.new_ones(())
    return [lambda s: mcke.layer_norm(x, stream=s), lambda s: mcke.layer_norm_backward(x, x, mean, rstd, stream=s),
            lambda s: mcke.token_logprobs(x, stream=s), lambda s: mcke.token_logprobs_backward(x, lse, grad_lse=lse, stream=s),
            lambda s: mcke.grad_norm([x], stream=s), lambda s: mcke.clip_grad_norm([x], 1.0, stream=s),
            lambda s: mcke.clip_grads([x], 1.0, norm, stream=s)]


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")
def test_every_operator_refuses_it():
    for call in _calls("cuda:0"):
        with pytest.raises(ValueError, match="stream is on cuda:1"):
            call(OTHER)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two CUDA devices")
def test_every_operator_refuses_a_real_one():
    other = torch.cuda.Stream("cuda:1")
    for call in _calls("cuda:0"):
        with pytest.raises(ValueError, match="stream is on cuda:1"):
            call(other)
