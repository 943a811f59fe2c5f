"""A paged attention call with the shortest bound on its waits: it ends, and
either says that a wait gave up or is right (one poll of a barrier may itself
sleep until the load is there); the engine works again once cleared. Bounds as
in test_gpu_attention.py."""
import pytest
import torch

from test_gpu_attention import Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("lengths", [[(1, 3000), (1, 40)], [(90, 900), (1, 500), (300, 300)]])
def test_waits_that_may_run_out(cuda_device, native_lib, lengths, weights, dim):
    from leanstream_b200 import _native as N

    call = Call(lengths, dim=dim, weights=weights, page=32)
    engine = call.engine()
    engine.run(**call.kwargs(), timeout_ns=1)
    torch.cuda.synchronize()
    assert engine.error() in (0, N.ATTN_TIMEOUT)
    if engine.error() == 0:
        call.check()
    engine.clear_error()
    if weights:
        call.weights.copy_(call.weights_before)
    engine.run(**call.kwargs())
    torch.cuda.synchronize()
    assert engine.error() == 0
    call.check()
