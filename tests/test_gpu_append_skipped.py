"""Tokens that append_cache skips, beside others of their block, in a cache of 8 bits.
Bounds as in test_gpu_append.py."""
import pytest
import torch

from test_gpu_append import RANGE, Case

pytestmark = pytest.mark.gpu


def check_rows(c, block, slots, skipped, older):
    """The block's exponents are of its written rows (and no smaller than older rows'), whose codes are
    right; the codes of `skipped` slots are as they were."""
    page = int(c.page_table[0, block])
    lowest = RANGE[c.dtype][0]
    for kv, (pages, new) in enumerate(((c.k_pages, c.k_new), (c.v_pages, c.v_new))):
        rows = [(new[t].double(), torch.zeros_like(new[t], dtype=torch.float64)) if kv else
                c.turned(new[t], int(c.positions[t])) for t, _ in slots]
        x, slack = torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows])
        for h in range(c.hk):
            e, was = int(c.exponents[page, h, 0, kv]), int(c.before[2][page, h, 0, kv])
            least = max(lowest, was) if older else lowest
            top, give = float(x[:, h].abs().max()), float(slack[:, h].max())
            assert e >= least and top - give <= 127 * 2.0 ** e
            assert e == least or top + give > 127 * 2.0 ** (e - 1)
            got = pages[page, [s % 16 for _, s in slots], h].double()
            assert ((got * 2.0 ** e - x[:, h]).abs() <= 0.5 * 2.0 ** e + slack[:, h]).all()
        for s in skipped:
            assert torch.equal(pages[page, s % 16], c.before[kv][page, s % 16])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_skipped_beside_written(cuda_device, native_lib, dim, dtype):
    from leanstream_b200 import _native as N, append_cache

    # slots 13 to 37: an older block, a new one, and one of which nothing is written
    c = Case([(25, 38)], dim=dim, dtype=dtype, int8=True, positions=True)
    bad = [14, 16, 20] + list(range(32, 38))
    c.positions[[s - 13 for s in bad]] = torch.tensor([-1, 1 << 20] * 4 + [-5], dtype=torch.int32, device="cuda")
    c.exponents[int(c.page_table[0, 2])] = -128
    c.keep()
    append_cache(**c.kwargs())
    torch.cuda.synchronize()
    assert c.error.item() == N.ATTN_POSITION
    check_rows(c, 0, [(0, 13), (2, 15)], [14], older=True)
    check_rows(c, 1, [(s - 13, s) for s in range(16, 32) if s not in bad], [16, 20], older=False)
    page = int(c.page_table[0, 2])
    for now, was in zip((c.k_pages, c.v_pages, c.exponents), c.before):
        assert torch.equal(now[page], was[page])
    written = torch.ones(25, dtype=torch.bool, device="cuda")
    written[[s - 13 for s in bad]] = False
    assert (c.q_out[~written] == 7).all()
    for t in written.nonzero()[:, 0].tolist():
        c.near(c.q_out[t], *c.turned(c.q[t], int(c.positions[t])))
