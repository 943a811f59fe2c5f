"""The paged cache calls in CUDA graphs: chunks, drafts, weights and evictions,
replayed with lengths and pages that changed on the device since the capture.
Bounds of the results as in test_gpu_attention.py."""
import pytest
import torch

from test_gpu_attention import Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[(1, 500), (1, 77)], [(4, 90), (3, 700)], [(90, 900), (1, 500)], [(300, 2000)]])
def test_attention(cuda_device, native_lib, lengths, dim, weights):
    c = Call(lengths, dim=dim, weights=weights)
    engine = c.engine()
    engine.run(**c.kwargs())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        engine.run(**c.kwargs())
    # another call of the same shape, in the captured buffers
    other = Call([(q, n - 5) for q, n in lengths], dim=dim, weights=weights, seed=3)
    for name in ("k_pages", "v_pages"):
        getattr(c, name)[:other.k_pages.shape[0]] = getattr(other, name)
    c.page_table.zero_()
    c.page_table[:, :other.page_table.shape[1]] = other.page_table
    c.q.copy_(other.q), c.k_new.copy_(other.k_new), c.v_new.copy_(other.v_new), c.kv_len.copy_(other.kv_len)
    for _ in range(2):
        c.output.fill_(7), c.lse.fill_(7)
        if weights:
            w = other.weights_before.shape[2]
            c.weights.zero_()
            c.weights[:, :, :w] = other.weights_before[:, :, :c.weights.shape[2]]
        graph.replay()
        torch.cuda.synchronize()
        assert engine.error() == 0
        other.output, other.lse, other.k_pages, other.v_pages = c.output, c.lse, c.k_pages, c.v_pages
        if weights:
            other.weights = c.weights[:, :, :w]
        other.check()


def test_evict(cuda_device, native_lib):
    from leanstream_b200 import evict_cache

    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(200, 16, 2, 64, generator=g, device="cuda").half() for _ in range(2))
    int32 = dict(dtype=torch.int32, device="cuda")
    order = torch.randperm(200, generator=g, device="cuda").int()
    table, new = order[:130].reshape(2, 65), order[130:146].reshape(2, 8)
    kv_len, w = torch.tensor([1040, 700], **int32), torch.rand(2, 2, 1040, generator=g, device="cuda")
    out = dict(new_len=torch.zeros(2, **int32), kept=torch.zeros(2, 2, 128, **int32),
               new_weights=torch.zeros(2, 2, 128, device="cuda"), error=torch.zeros(1, **int32))
    call = dict(page_table=table, kv_len=kv_len, weights=w, budget=128, new_table=new, sinks=3, recent=20)
    evict_cache(k_pages=k, v_pages=v, **call, **out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        evict_cache(k_pages=k, v_pages=v, **call, **out)
    kv_len.copy_(torch.tensor([90, 1000], **int32))
    w.copy_(torch.rand(w.shape, generator=g, device="cuda"))
    want = {n: torch.full_like(t, -9) for n, t in out.items() if n != "error"}
    pools = k.clone(), v.clone()
    evict_cache(k_pages=pools[0], v_pages=pools[1], **call, **want, error=out["error"])
    graph.replay()
    torch.cuda.synchronize()
    assert out["error"].item() == 0 and out["new_len"].tolist() == [90, 128]
    for name, t in want.items():
        assert torch.equal(out[name], t)
    assert torch.equal(k, pools[0]) and torch.equal(v, pools[1])
