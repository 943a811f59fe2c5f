"""A paged attention call whose waits run out: it reports so, ends, and leaves
an engine that works again once cleared. Bounds as in test_gpu_attention.py."""
import pytest
import torch

from test_gpu_attention import Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("lengths", [[(1, 3000), (1, 40)], [(90, 900), (1, 500), (300, 300)]])
def test_waits_that_run_out(cuda_device, native_lib, lengths, weights, dim):
    from leanstream_b200 import _native as N

    call = Call(lengths, dim=dim, weights=weights, page=32)
    engine = call.engine()
    engine.run(**call.kwargs(), timeout_ns=1)  # no load ends within a nanosecond
    torch.cuda.synchronize()
    assert engine.error() == N.ATTN_TIMEOUT
    engine.clear_error()
    if weights:
        call.weights.copy_(call.weights_before)
    engine.run(**call.kwargs())
    torch.cuda.synchronize()
    assert engine.error() == 0
    call.check()
