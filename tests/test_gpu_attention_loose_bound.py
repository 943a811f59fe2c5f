"""max_q is a bound: a call of very many sequences with a bound far above their
new tokens, of which most have none. Bounds of the results as in
test_gpu_attention.py."""
import pytest
import torch

from test_gpu_attention import Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bound", [64, 1 << 16, 1 << 20])
@pytest.mark.parametrize("batch", [3, 40, 1 << 14])
def test_loose_bound(cuda_device, native_lib, batch, bound):
    from leanstream_b200 import PagedAttention

    lengths = [(0, 9), (40, 300), (1, 77)] + [(0, 0)] * (batch - 3)
    lengths[-1] = lengths[-1] if batch == 3 else (17, 50)
    c = Call(lengths, 8, 2, 64, page=32)
    engine = PagedAttention(8, 2, 64, page_size=32, max_sequences=batch, max_tokens=c.q.shape[0], max_queries=bound)
    engine.run(**{**c.kwargs(), "max_q": bound})
    torch.cuda.synchronize()
    assert engine.error() == 0
    c.check()


def test_more_tokens_than_append_blocks(cuda_device, native_lib):
    """One sequence whose new tokens' rows are copied by blocks that go round."""
    tokens, slots = 1 << 18, (1 << 18) + 100
    from leanstream_b200 import PagedAttention

    g = torch.Generator(device="cuda").manual_seed(7)
    half = dict(dtype=torch.float16, device="cuda")
    columns = -(-slots // 64)
    table = torch.randperm(columns, generator=g, device="cuda").int()[None]
    k_pages, v_pages = torch.zeros(columns, 64, 1, 64, **half), torch.zeros(columns, 64, 1, 64, **half)
    q, k_new, v_new = (torch.randn(tokens, 1, 64, generator=g, **half) for _ in range(3))
    out = torch.empty_like(q)
    engine = PagedAttention(1, 1, 64, page_size=64, max_sequences=1, max_tokens=tokens, max_queries=tokens)
    engine.run(q=q, output=out, k_pages=k_pages, v_pages=v_pages, page_table=table,
               q_start=torch.tensor([0, tokens], dtype=torch.int32, device="cuda"),
               kv_len=torch.tensor([slots], dtype=torch.int32, device="cuda"), max_q=tokens, k_new=k_new,
               v_new=v_new, window=64)
    torch.cuda.synchronize()
    assert engine.error() == 0
    for pool, new in ((k_pages, k_new), (v_pages, v_new)):
        rows = pool[table[0].long()].reshape(-1, 1, 64)[:slots]
        assert torch.equal(rows[100:], new) and (rows[:100] == 0).all()
