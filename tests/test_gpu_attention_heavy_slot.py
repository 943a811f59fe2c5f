"""A slot that draws nearly all of a row's weight and whose value is near zero:
the output is what the other slots add up to, each with a small probability.

Bound: that of test_gpu_attention.py, plus what 16-bit probabilities can lose at
the low end. float16 holds them to u of their value, or to half its smallest step,
2^-25, where that is more. The kernels scale them so that the row's largest is at
least 2^7 (2^15 in the decode kernel): at most 2^-32 (2^-40) of it per slot,
times the sum of |v|. bfloat16 reaches to 2^-133."""
import pytest
import torch

from test_gpu_attention import UNIT, Call

pytestmark = pytest.mark.gpu

SLOTS, DIM = 6000, 64


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("value", [1.0, 300.0])
@pytest.mark.parametrize("gap", [12.0, 16.5, 17.5, 20.0])
@pytest.mark.parametrize("q,at", [(1, 0), (4, 0), (1, 3333), (90, 0), (300, 0), (90, 3333)])
def test_small_probabilities(cuda_device, native_lib, q, at, gap, value, dtype):
    heads, kv_heads = 8, 2
    c = Call([(q, SLOTS)], heads, kv_heads, DIM, page=64, dtype=dtype, seed=q + at, append=False)
    g = torch.Generator(device="cuda").manual_seed(int(gap * 2) + q)
    # queries along one direction, `gap` above the others in the heavy slot
    e = torch.zeros(DIM, device="cuda")
    e[0] = 1.0
    queries = 0.5 * torch.randn(q, heads, DIM, generator=g, device="cuda")
    queries[..., 0] = 8.0
    c.q.copy_(queries)
    keys = torch.randn(SLOTS, kv_heads, DIM, generator=g, device="cuda")
    keys[..., 0] = 0
    keys[at] = e * (gap * DIM ** 0.5 / 8.0)
    values = value * (1 + 0.25 * torch.randn(SLOTS, kv_heads, DIM, generator=g, device="cuda"))
    values[at] = 0
    c.keys, c.values = [keys.to(dtype)], [values.to(dtype)]
    slot = torch.arange(SLOTS, device="cuda")
    pages = c.page_table[0].long()
    c.k_pages[pages[slot // c.page], slot % c.page] = c.keys[0]
    c.v_pages[pages[slot // c.page], slot % c.page] = c.values[0]
    engine = c.engine()
    engine.run(**c.kwargs())
    torch.cuda.synchronize()
    assert engine.error() == 0
    want, area, lse, _, _ = c.expected()
    u = UNIT[dtype]
    floor = 0.0 if dtype is torch.bfloat16 else 2.0 ** (-40 if q * heads // kv_heads <= 16 else -32)
    lost = floor * c.values[0].double().abs().sum(0).repeat_interleave(heads // kv_heads, 0)
    err = (c.output.double() - want).abs()
    tol = u * (want.abs() + area) + 2e-5 * area + 2.0 ** -24 + lost
    assert (err <= tol).all(), f"output off by {(err / tol).max().item():.3g} of its bound"
    assert (c.lse.double() - lse).abs().max().item() <= 2e-5
