"""examples/bounded_cache.py: every attention call and every eviction of a run,
prompts in chunks to decoding past several evictions, against the formulas in
64 bits on what the cache's pages hold.

Bounds as in test_gpu_attention.py: float16's unit roundoff 2^-11 on the result
and on each probability, 2e-5 of the probabilities for logits and exponentials;
the weights 2e-5 of the probabilities that a call adds, plus the 32-bit sum's
rounding."""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = pytest.mark.gpu


def slots(pages, row, n, page):
    at = torch.arange(n, device="cuda")
    return pages[row[at // page].long(), at % page].double()


def watch_attention(layer, seen):
    run = layer.attention.run

    def checked(**a):
        before = a["weights"].clone()
        run(**a)
        starts, q = a["q_start"].tolist(), a["q"].double()
        group, u = layer.q_heads // layer.kv_heads, 2.0 ** -11
        for b, n in enumerate(a["kv_len"].tolist()):
            t0, t1 = starts[b:b + 2]
            if t0 == t1:
                assert torch.equal(a["weights"][b], before[b])
                continue
            assert n == layer.lengths[b]
            k, v = (slots(a[x], a["page_table"][b], n, layer.page).repeat_interleave(group, 1)
                    for x in ("k_pages", "v_pages"))
            assert torch.equal(k[n - (t1 - t0):, ::group], a["k_new"][t0:t1].double())
            s = torch.einsum("qhd,khd->hqk", q[t0:t1], k) * layer.head_dim ** -0.5
            future = torch.arange(n, device="cuda")[None] > torch.arange(n - (t1 - t0), n, device="cuda")[:, None]
            p = s.masked_fill(future, -torch.inf).softmax(-1)
            want, area = torch.einsum("hqk,khd->qhd", p, v), torch.einsum("hqk,khd->qhd", p, v.abs())
            err = (a["output"][t0:t1].double() - want).abs()
            assert (err <= u * (want.abs() + area) + 2e-5 * area + 2.0 ** -24).all()
            mass = p.view(layer.kv_heads, group, t1 - t0, n).sum((1, 2))
            old = before[b, :, :n].double()
            old[:, n - (t1 - t0):] = 0
            err = (a["weights"][b, :, :n].double() - old - mass).abs()
            assert (err <= 2e-5 * mass + 2.0 ** -22 * (old + mass) + 1e-30).all()
        seen.append(a["max_q"])

    layer.attention.run = checked


def watch_evict(module, seen):
    evict = module.evict_cache

    def checked(**a):
        held = [[slots(a[x], a["page_table"][b], n, a[x].shape[1]) for x in ("k_pages", "v_pages")]
                for b, n in enumerate(a["kv_len"].tolist())]
        w = a["weights"].clone()
        evict(**a)
        budget, sinks, recent = a["budget"], a["sinks"], a["recent"]
        for b, n in enumerate(a["kv_len"].tolist()):
            m = min(n, budget)
            assert a["new_len"][b].item() == m
            for h in range(a["kept"].shape[1]):
                kept = a["kept"][b, h, :m].long()
                if n <= budget:
                    assert torch.equal(kept, torch.arange(n, device="cuda"))
                else:
                    middle = w[b, h, sinks:n - recent].sort(descending=True, stable=True).indices + sinks
                    middle = middle[:budget - sinks - recent].sort().values
                    want = torch.cat([torch.arange(sinks, device="cuda"), middle,
                                      torch.arange(n - recent, n, device="cuda")])
                    assert torch.equal(kept, want)
                assert torch.equal(a["new_weights"][b, h, :m], w[b, h, kept])
                for x, rows in zip(("k_pages", "v_pages"), held[b]):
                    assert torch.equal(slots(a[x], a["new_table"][b], m, a[x].shape[1])[:, h], rows[kept, h])
        seen.append(max(a["kv_len"].tolist()))

    return checked


@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 4, 128)])
def test_prompt_to_decode(cuda_device, native_lib, monkeypatch, heads):
    import bounded_cache

    calls, cuts = [], []
    monkeypatch.setattr(bounded_cache, "evict_cache", watch_evict(bounded_cache, cuts))
    layer = bounded_cache.BoundedLayer(3, 300, hidden=512, q_heads=heads[0], kv_heads=heads[1], head_dim=heads[2],
                                       budget=90, slack=9, sinks=3, recent=20, chunk=130, seed=heads[0])
    watch_attention(layer, calls)
    x = layer.prompt([torch.randn(n, 512, device="cuda").half() for n in (300, 131, 40)])
    for _ in range(21):
        x = layer.step(torch.nn.functional.rms_norm(x, (512,)))
        assert torch.isfinite(x).all()
    layer.check()
    assert calls == [130, 130, 40] + [1] * 21
    assert cuts == [300, 99, 99]
