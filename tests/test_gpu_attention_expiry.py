"""Waits of the paged attention that give up: the kernels end, say so, leave no
row in the cache that is not a new token's, and work again once cleared. Whether
the waits of a small call run out under a bound of 1 ns depends on how long one
try of a barrier sleeps; over a cache that streams from memory they do. Bounds of
the results as in test_gpu_attention.py."""
import pytest
import torch

from test_gpu_attention import Call

pytestmark = pytest.mark.gpu

SMALL = {
    "decode_one": [(1, 700)],
    "decode": [(1, 3000), (1, 40), (1, 1), (1, 20000)],
    "draft": [(4, 90), (3, 2000), (1, 17)],
    "chunk": [(90, 900), (1, 500), (300, 300)],
    "long_chunk": [(700, 9000)],
}


def bits(t):
    return t.contiguous().view(torch.int16)


def check_cache(call, old):
    """Every row is as before, or, in a new token's slot, its key or value (each head on its own)."""
    fresh = torch.zeros(old[0].shape[:2], dtype=torch.bool, device="cuda")
    at = 0
    for b, (q, n) in enumerate(call.lengths):
        for i in range(max(0, n - q), n):
            where, token = int(call.page_table[b, i // call.page]), at + i - (n - q)
            fresh[where, i % call.page] = True
            for before, pool, new in zip(old, (call.k_pages, call.v_pages), (call.k_new, call.v_new)):
                row = bits(pool[where, i % call.page])
                as_new = (row == bits(new[token])).all(-1)
                assert (as_new | (row == before[where, i % call.page]).all(-1)).all()
        at += q
    for before, pool in zip(old, (call.k_pages, call.v_pages)):
        assert torch.equal(bits(pool)[~fresh], before[~fresh])


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", SMALL)
def test_expired_waits(cuda_device, native_lib, name, dim, weights, window):
    from leanstream_b200 import _native as N

    call = Call(SMALL[name], dim=dim, weights=weights, page=32, window=window, sinks=3 if window else 0)
    engine = call.engine()
    old = [bits(t).clone() for t in (call.k_pages, call.v_pages)]
    for _ in range(3):
        engine.run(**call.kwargs(), timeout_ns=1)
    torch.cuda.synchronize()
    assert engine.error() in (0, N.ATTN_TIMEOUT)
    check_cache(call, old)
    engine.clear_error()
    if weights:
        call.weights.copy_(call.weights_before)
    engine.run(**call.kwargs())
    torch.cuda.synchronize()
    assert engine.error() == 0
    call.check()


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q", [1, 4, 200])
def test_expired_waits_over_a_long_cache(cuda_device, native_lib, q, dim, weights):
    """More than the L2 cache holds: against the same call with the default bound."""
    from leanstream_b200 import _native as N

    call = Call([(q, 16 + q)] * 16, dim=dim, weights=weights, page=64)
    call.lengths = [(q, 60000 // dim * 64 + 131 * b) for b in range(16)]
    columns = -(-max(n for _, n in call.lengths) // 64)
    g = torch.Generator(device="cuda").manual_seed(dim + q)
    pool = (16 * columns, 64, 2, dim)
    call.k_pages, call.v_pages = (torch.randn(pool, generator=g, device="cuda").half() for _ in range(2))
    call.page_table = torch.randperm(pool[0], generator=g, device="cuda").int().reshape(16, columns)
    call.kv_len = torch.tensor([n for _, n in call.lengths], dtype=torch.int32, device="cuda")
    if weights:
        call.weights = torch.rand(16, 2, columns * 64, generator=g, device="cuda")
    old, before = [bits(t).clone() for t in (call.k_pages, call.v_pages)], call.weights
    assert 2 * call.k_pages.numel() * 2 > 2 ** 28

    engine = call.engine()
    if weights:
        call.weights = before.clone()
    for _ in range(5):
        engine.run(**call.kwargs(), timeout_ns=1)
    torch.cuda.synchronize()
    assert engine.error() == N.ATTN_TIMEOUT
    check_cache(call, old)
    engine.clear_error()
    got = []
    for use in (engine, call.engine()):
        if weights:
            call.weights = before.clone()
        call.output.fill_(7)
        use.run(**call.kwargs())
        torch.cuda.synchronize()
        assert use.error() == 0
        got.append((call.output.clone(), call.lse.clone(), call.weights))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert not weights or torch.equal(got[0][2], got[1][2])
    assert torch.isfinite(got[0][0]).all()
