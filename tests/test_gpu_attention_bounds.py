"""timeout_ns bounds every wait of a paged attention call, not the call: calls
that take several times as long as their bound, over sequences that share their
pages, give the results of the default bound."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE, POOL = 32, 8, 128, 64, 2048


@pytest.mark.parametrize("batch,q,slots,weights,bound_us", [
    (16, 1, 1 << 19, False, 1000),   # about 5 ms
    (1, 2048, 1 << 17, False, 1000),  # about 4.5 ms
    (1, 2048, 1 << 17, True, 1000)], ids=["decode", "chunk", "chunk_weights"])
def test_call_longer_than_the_bound(cuda_device, native_lib, batch, q, slots, weights, bound_us):
    from leanstream_b200 import PagedAttention

    g = torch.Generator(device="cuda").manual_seed(slots + q)
    half = dict(dtype=torch.bfloat16, device="cuda")
    tokens = batch * q
    k_pages, v_pages = (torch.randn(POOL, PAGE, KV_HEADS, DIM, generator=g, **half) for _ in range(2))
    args = dict(q=torch.randn(tokens, HEADS, DIM, generator=g, **half), k_pages=k_pages, v_pages=v_pages,
                page_table=torch.randint(0, POOL, (batch, slots // PAGE), generator=g, device="cuda").int(),
                q_start=torch.arange(batch + 1, device="cuda").int() * q, max_q=q,
                kv_len=torch.full((batch,), slots, dtype=torch.int32, device="cuda"))
    engine = PagedAttention(HEADS, KV_HEADS, DIM, page_size=PAGE, dtype="bfloat16", max_sequences=batch,
                            max_tokens=tokens, max_queries=q, max_weights_length=slots if weights else 0)
    got = []
    for bound in (0, bound_us * 1000):
        out, lse = torch.full((tokens, HEADS, DIM), 7.0, **half), torch.full((tokens, HEADS), 7.0, device="cuda")
        mass = torch.zeros(batch, KV_HEADS, slots, device="cuda") if weights else None
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        engine.run(output=out, lse=lse, weights=mass, timeout_ns=bound, **args)
        end.record()
        torch.cuda.synchronize()
        assert begin.elapsed_time(end) > 2e-3 * bound_us
        assert engine.error() == 0
        got.append((out, lse, mass))
    assert torch.isfinite(got[0][0]).all() and torch.isfinite(got[0][1]).all()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert not weights or torch.equal(got[0][2], got[1][2])
