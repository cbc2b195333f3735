"""The layer norm's bounded wait: one that runs out is reported on the host, under its
own name, and the context stays usable."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU container
    pytest.skip("needs a CUDA device", allow_module_level=True)

import mcke  # noqa: E402
import test_gpu_layer_norm as ln  # noqa: E402


def test_a_wait_that_runs_out_is_reported_and_the_context_survives():
    mcke.check_device_errors()  # start clean
    x, w, b, dy = ln._inputs(7, 12288, torch.bfloat16, seed=1)  # rows over clusters: their sums are waited for
    want = mcke.layer_norm(x, w, b, save_stats=True)
    stream = torch.cuda.current_stream().cuda_stream
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    assert mcke.lib().mcke_sm100_layer_norm_watchdog_selftest(stream) == mcke.OK
    end.record()
    with pytest.raises(mcke.MckeError) as e:
        mcke.check_device_errors()
    # both passes wait in the same way, so neither is named
    assert e.value.code == mcke.INTERNAL and "layer norm:" in e.value.message and "backward" not in e.value.message
    assert 15 < begin.elapsed_time(end) < 39  # 20 ms once: behind it the next wait does not wait
    mcke.check_device_errors()  # the word was cleared
    got = mcke.layer_norm(x, w, b, save_stats=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    ln._check_backward(x, w, got[1], got[2], dy, *mcke.layer_norm_backward(dy, x, got[1], got[2], w))
    mcke.check_device_errors()
