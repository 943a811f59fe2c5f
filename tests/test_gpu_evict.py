"""Eviction from a paged cache (leanstream_b200.evict_cache) on the GPU: what
is kept, and where, is exact."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def expected_slots(w, n, budget, sinks, recent):
    if n <= budget:
        return list(range(n))
    value = [-math.inf if math.isnan(x) else x for x in w[:n].tolist()]
    middle = sorted(range(sinks, n - recent), key=lambda i: (-value[i], i))
    return list(range(sinks)) + sorted(middle[:budget - sinks - recent]) + list(range(n - recent, n))


def evict(lengths, budget, sinks=0, recent=0, kv_heads=2, dim=128, page=16, dtype=torch.float16, weights=None, seed=0,
          layout="nhd"):
    from leanstream_b200 import evict_cache

    g = torch.Generator(device="cuda").manual_seed(seed)
    batch, columns, rows = len(lengths), max(-(-max(lengths) // page), 1), -(-budget // page)
    pages = batch * (columns + rows)
    shape = (pages, page, kv_heads, dim) if layout == "nhd" else (pages, kv_heads, page, dim)
    k, v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    if layout == "hnd":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table, new = order[:batch * columns].reshape(batch, columns), order[batch * columns:].reshape(batch, rows)
    w = torch.rand(batch, kv_heads, columns * page, generator=g, device="cuda")
    if weights is not None:
        w = weights(w)
    kv_len = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    new_len = torch.full((batch,), -9, dtype=torch.int32, device="cuda")
    kept = torch.full((batch, kv_heads, budget), -9, dtype=torch.int32, device="cuda")
    new_w = torch.full((batch, kv_heads, budget), -9.0, device="cuda")
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    want_k, want_v = k.clone(), v.clone()
    evict_cache(k_pages=k, v_pages=v, page_table=table, kv_len=kv_len, weights=w, budget=budget, sinks=sinks,
                recent=recent, new_table=new, new_len=new_len, kept=kept, new_weights=new_w, error=error)
    torch.cuda.synchronize()
    assert error.item() == 0
    assert new_len.tolist() == [min(n, budget) for n in lengths]
    for b, n in enumerate(lengths):
        for h in range(kv_heads):
            slots = expected_slots(w[b, h].cpu(), n, budget, sinks, recent)
            assert kept[b, h].tolist() == slots + [-1] * (budget - len(slots))
            i, j = torch.tensor(slots, device="cuda").long(), torch.arange(len(slots), device="cuda")
            assert torch.equal(new_w[b, h, :len(slots)].nan_to_num(5.0), w[b, h, i].nan_to_num(5.0))
            assert (new_w[b, h, len(slots):] == 0).all()
            for pool in (want_k, want_v):
                pool[new[b].long()[j // page], j % page, h] = pool[table[b].long()[i // page], i % page, h]
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


@pytest.mark.parametrize("dim,kv_heads,dtype", [(64, 1, torch.float16), (128, 3, torch.bfloat16)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_sizes(cuda_device, native_lib, page, dim, kv_heads, dtype):
    for seed, (lengths, budget, sinks, recent) in enumerate([
            ([1], 1, 0, 0), ([0, 1, 2, 5], 2, 1, 1), ([17, 16, 15, 300], 16, 2, 5), ([1025, 1024, 1023], 1024, 4, 100),
            ([5000, 2500, 60], 777, 0, 0), ([3000], 2999, 4, 0), ([2048, 4099], 40, 40, 0), ([2048, 4099], 40, 0, 40),
            ([2049], 40, 20, 20)]):
        evict(lengths, budget, sinks, recent, kv_heads, dim, page, dtype, seed=seed)


def test_ties_signs_and_non_finite_weights(cuda_device, native_lib):
    evict([3000, 1500], 1000, 4, 50, weights=lambda w: (w * 4).floor())
    evict([3000, 1500], 1000, 4, 50, weights=lambda w: torch.zeros_like(w))
    evict([3000], 1000, weights=lambda w: torch.where(w < 0.5, -0.0, 0.0))
    evict([3000], 1000, weights=lambda w: w - 0.5)

    def wild(w):
        w = w.clone()
        w[w < 0.2] = math.nan
        w[(w > 0.2) & (w < 0.3)] = -math.inf
        w[w > 0.9] = math.inf
        w[(w > 0.8) & (w < 0.85)] = 1e-42
        return w

    evict([3000, 999], 700, 3, 3, weights=wild)
    evict([3000], 2900, weights=wild)


def test_head_major_pages(cuda_device, native_lib):
    evict([400, 90], 100, 4, 10, layout="hnd")


def test_long(cuda_device, native_lib):
    evict([70001], 9000, 4, 512, kv_heads=2, page=64)


def test_bad_lengths_are_reported(cuda_device, native_lib):
    from leanstream_b200 import _native as N, evict_cache

    k = torch.zeros(8, 16, 1, 64, dtype=torch.float16, device="cuda")
    int32 = dict(dtype=torch.int32, device="cuda")
    table, new = torch.tensor([[0, 1], [2, 3]], **int32), torch.tensor([[4], [5]], **int32)
    error, new_len, kept = torch.zeros(1, **int32), torch.zeros(2, **int32), torch.zeros(2, 1, 8, **int32)
    w = torch.rand(2, 1, 32, device="cuda")
    common = dict(k_pages=k, v_pages=k.clone(), weights=w, budget=8, new_len=new_len, kept=kept, error=error)
    evict_cache(page_table=table, new_table=new, kv_len=torch.tensor([33, 20], **int32), **common)
    torch.cuda.synchronize()
    assert error.item() == N.ATTN_LENGTH and new_len.tolist() == [0, 8] and (kept[0] == -1).all()
    error.zero_()
    evict_cache(page_table=torch.tensor([[0, 1], [2, 8]], **int32), new_table=new,
                kv_len=torch.tensor([4, 32], **int32), **{**common, "weights": torch.ones_like(w).cumsum(-1)})
    torch.cuda.synchronize()
    assert error.item() == N.ATTN_PAGE
