"""Waits of the attention over a cache in 8 bits that give up: the kernels end and
say so, the cache is as it was, and the engine works again once cleared; and a call
that takes longer than its bound, which is of each wait, is none of these."""
import pytest
import torch

from test_gpu_attention_expiry import SMALL
from test_gpu_attention_int8 import Call8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", SMALL)
def test_expired_waits(cuda_device, native_lib, name, dim, page):
    from leanstream_b200 import _native as N

    call = Call8(SMALL[name], dim=dim, page=page)
    engine = call.engine()
    old = [t.clone() for t in (call.k_pages, call.v_pages, call.exponents)]
    for _ in range(3):
        engine.run(**call.kwargs(), timeout_ns=1)
    torch.cuda.synchronize()
    assert engine.error() in (0, N.ATTN_TIMEOUT)
    assert all(torch.equal(a, b) for a, b in zip(old, (call.k_pages, call.v_pages, call.exponents)))
    engine.clear_error()
    engine.run(**call.kwargs())
    torch.cuda.synchronize()
    assert engine.error() == 0
    call.check()


def long_call(q, dim, page, batch=16):
    """More than the L2 cache holds, in pages that the sequences share."""
    c = Call8([(q, 16 + q)] * batch, dim=dim, page=page, dtype=torch.bfloat16)
    pool = 200000 // page
    g = torch.Generator(device="cuda").manual_seed(dim + q)
    c.k_pages, c.v_pages = (torch.randint(-127, 128, (pool, page, 2, dim), generator=g, device="cuda",
                                          dtype=torch.int8) for _ in range(2))
    c.exponents = torch.randint(-8, -5, (pool, 2, page // 16, 2), generator=g, device="cuda", dtype=torch.int8)
    c.page_table = torch.randint(0, pool, (batch, 120000 // page), generator=g, device="cuda").int()
    c.lengths = [(q, 110000 + 131 * b) for b in range(batch)]
    c.kv_len = torch.tensor([n for _, n in c.lengths], dtype=torch.int32, device="cuda")
    return c


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q", [1, 3, 6, 200])
def test_expired_waits_over_a_long_cache(cuda_device, native_lib, q, dim, page):
    from leanstream_b200 import _native as N

    call = long_call(q, dim, page)
    engine = call.engine()
    for _ in range(5):
        engine.run(**call.kwargs(), timeout_ns=1)
    torch.cuda.synchronize()
    assert engine.error() == N.ATTN_TIMEOUT
    engine.clear_error()
    got = []
    for use in (engine, call.engine()):
        call.output.fill_(7)
        use.run(**call.kwargs())
        torch.cuda.synchronize()
        assert use.error() == 0
        got.append((call.output.clone(), call.lse.clone()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert torch.isfinite(got[0][0]).all()


@pytest.mark.parametrize("q,bound_us", [(1, 60), (2048, 1000)])
def test_call_longer_than_the_bound(cuda_device, native_lib, q, bound_us):
    call = long_call(q, 128, 64, batch=64 if q == 1 else 4)
    engine, got = call.engine(), []
    for bound in (0, bound_us * 1000):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        engine.run(**call.kwargs(), timeout_ns=bound)
        end.record()
        torch.cuda.synchronize()
        assert begin.elapsed_time(end) > 2e-3 * bound_us
        assert engine.error() == 0
        got.append((call.output.clone(), call.lse.clone()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
