"""Sequences beside one whose lengths or pages do not fit the call: their outputs,
lse, weights and appended rows are right, and the refused one's are as they were.
Bounds as in test_gpu_attention.py."""
import pytest
import torch

from test_gpu_attention import UNIT, Call

pytestmark = pytest.mark.gpu

LONG = {1: [(1, 200), (1, 150), (1, 333)], 50: [(50, 200), (50, 150), (50, 333)]}


def compare(c, bad, expected):
    out, area, lse, weights, mass = expected
    rows = torch.ones(c.q.shape[0], dtype=torch.bool, device="cuda")
    at = 0
    for b, (q, n) in enumerate(c.lengths):
        if b == bad:
            rows[at:at + q] = False
        else:
            for i in range(n - q, n):
                page, token = int(c.page_table[b, i // c.page]), at + i - (n - q)
                assert torch.equal(c.k_pages[page, i % c.page], c.k_new[token])
                assert torch.equal(c.v_pages[page, i % c.page], c.v_new[token])
            err = (c.weights[b].double() - weights[b]).abs()
            assert (err <= 2e-5 * mass[b] + 2.0 ** -22 * weights[b].abs() + 1e-30).all()
        at += q
    err = (c.output.double() - out).abs()
    assert (err <= UNIT[c.dtype] * (out.abs() + area) + 2e-5 * area + 2.0 ** -24)[rows].all()
    assert ((c.lse.double() - lse).abs() <= 2e-5)[rows].all()
    return rows


@pytest.mark.parametrize("bad", [0, 1, 2])
@pytest.mark.parametrize("q", LONG)
@pytest.mark.parametrize("dim", [64, 128])
def test_bad_length(cuda_device, native_lib, q, bad, dim):
    from leanstream_b200 import _native as N

    c = Call(LONG[q], dim=dim, weights=True, seed=bad)
    expected = c.expected()
    pages = c.page_table[bad, :-(-LONG[q][bad][1] // c.page)].long()
    before = c.k_pages[pages].clone(), c.v_pages[pages].clone()
    engine = c.engine()
    for length in (c.page_table.shape[1] * c.page + 1, -1, -(1 << 31), (1 << 31) - 1):
        c.output.fill_(7)
        c.lse.fill_(7)
        c.weights.copy_(c.weights_before)
        c.kv_len[bad] = length
        engine.run(**c.kwargs())
        torch.cuda.synchronize()
        assert engine.error() == N.ATTN_LENGTH
        engine.clear_error()
        rows = compare(c, bad, expected)
        assert (c.output[~rows] == 7).all() and (c.lse[~rows] == 7).all()
        assert torch.equal(c.weights[bad], c.weights_before[bad])
        for now, was in zip((c.k_pages[pages], c.v_pages[pages]), before):
            assert torch.equal(now.view(torch.int16), was.view(torch.int16))


@pytest.mark.parametrize("bad", [0, 1, 2])
@pytest.mark.parametrize("q", LONG)
@pytest.mark.parametrize("index", [-1, -(1 << 31), (1 << 31) - 1, None])
def test_bad_page(cuda_device, native_lib, q, bad, index):
    """A page outside the pool, among the old slots or where the new tokens go."""
    from leanstream_b200 import _native as N

    for column in (2, (LONG[q][bad][1] - 1) // 16):
        c = Call(LONG[q], weights=True, seed=bad)
        expected = c.expected()
        c.page_table[bad, column] = c.k_pages.shape[0] if index is None else index
        engine = c.engine()
        engine.run(**c.kwargs())
        torch.cuda.synchronize()
        assert engine.error() == N.ATTN_PAGE
        compare(c, bad, expected)
