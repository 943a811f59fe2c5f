"""Exponents of a cache in 8 bits against the range of the attention's type: -24 to 9
for float16, -126 to 120 for bfloat16. A visible block outside is reported and reads
as NaN, whatever the number of rows; the range itself, and blocks that no row sees, are
not. Bounds as in test_gpu_attention_int8_small.py."""
import pytest
import torch

from test_gpu_attention_int8_small import Small

pytestmark = pytest.mark.gpu

ROWS = [1, 4, 6, 8, 60]
OUTSIDE = [(torch.float16, e) for e in (10, 127, -25, -126, -127)] + [(torch.bfloat16, e) for e in (121, 127, -127)]


def run(c):
    c.output.fill_(7), c.lse.fill_(7)
    engine = c.engine()
    engine.run(**c.kwargs())
    torch.cuda.synchronize()
    return engine.error()


@pytest.mark.parametrize("q", ROWS)
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("dtype,e", OUTSIDE)
def test_outside_the_range(cuda_device, native_lib, dtype, e, kv, q):
    from leanstream_b200 import _native as N

    for page in (16, 32):
        c = Small([(q, 200), (q, 150)], 0, dtype=dtype, page=page)
        assert run(c) == 0
        good = c.output.clone(), c.lse.clone()
        # slots 32 to 47 of the second sequence's second kv head
        c.exponents[int(c.page_table[1, 32 // page]), 1, 0, kv] = e
        assert run(c) == N.ATTN_EXPONENT
        assert c.output[q:, 4:].isnan().all()
        assert c.lse[q:, 4:].isnan().all() if kv == 0 else torch.equal(c.lse, good[1])
        rest = torch.ones_like(c.lse, dtype=torch.bool)
        rest[q:, 4:] = False
        assert torch.equal(c.output[rest], good[0][rest]) and torch.equal(c.lse[rest], good[1][rest])


@pytest.mark.parametrize("q", ROWS)
@pytest.mark.parametrize("dtype,e", [(torch.float16, 9), (torch.float16, -24), (torch.bfloat16, 100), (torch.bfloat16, -126)])
def test_the_ends_of_the_range(cuda_device, native_lib, dtype, e, q):
    for page in (16, 32):
        c = Small([(q, 200), (q, 150)], 0, dtype=dtype, page=page)
        where = int(c.page_table[1, 32 // page])
        c.exponents[where, 1, 0, 1] = e
        c.values[1][32:48, 1] = c.v_pages[where, :16, 1].double() * 2.0 ** e
        c.largest = max(c.largest, e)
        assert run(c) == 0
        if dtype is torch.float16 and e == 9:
            # codes are of [-127, 127], and Call8 draws some of -128: 128 * 2^9 = 65536, where float16 ends at
            # 65504 and 127 * 2^9 = 65024 still fits. Elements with such a code are not of the format.
            out = c.expected()[0]
            none = (c.v_pages[where, :16, 1] == -128).any(0)
            c.output[q:, 4:, none] = out[q:, 4:, none].to(dtype)
        c.check()
        if e < 0:  # keys of next to no size
            c.exponents[where, 0, 0, 0] = e
            c.keys[1][32:48, 0] = c.k_pages[where, :16, 0].double() * 2.0 ** e
            assert run(c) == 0
            c.check()


@pytest.mark.parametrize("q", ROWS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_blocks_that_no_row_sees(cuda_device, native_lib, dtype, q):
    for page in (16, 32, 128):
        for window, sinks in ((0, 0), (50, 0), (70, 5)):
            c = Small([(q, 500), (q, 200)], 0, dtype=dtype, page=page, window=window, sinks=sinks)
            c.exponents[c.exponents == -128] = 127
            assert run(c) == 0
            c.check()


@pytest.mark.parametrize("q", ROWS)
@pytest.mark.parametrize("filled,read,power", [(torch.bfloat16, torch.float16, -40), (torch.bfloat16, torch.float16, 30),
                                               (torch.bfloat16, torch.float16, 0), (torch.float16, torch.bfloat16, 0),
                                               (torch.float16, torch.bfloat16, -10)])
def test_a_cache_that_another_type_filled(cuda_device, native_lib, filled, read, power, q):
    """Few rows and chunks give the same answer: NaN and a report where the values do not fit, else their attention."""
    from leanstream_b200 import _native as N, append_cache

    c = Small([(q, 100)], 0, dtype=read, page=32)
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn(100, 2, 128, generator=g, device="cuda").to(filled) for _ in range(2))
    v *= 2.0 ** power
    starts = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    append_cache(k_new=k, v_new=v, k_pages=c.k_pages, v_pages=c.v_pages, exponents=c.exponents,
                 page_table=c.page_table, q_start=starts, kv_len=c.kv_len)
    if power in (-40, 30):
        assert run(c) == N.ATTN_EXPONENT and c.output.isnan().all()
        return
    i = torch.arange(100, device="cuda")
    where = c.page_table[0].long()[i // 32]
    size = c.exponents[where, :, i // 16 % 2].double()
    c.largest = float(size[..., 1].max())
    c.keys, c.values = ([p[where, i % 32].double() * (2.0 ** size[..., j])[..., None]]
                        for j, p in enumerate((c.k_pages, c.v_pages)))
    assert run(c) == 0
    c.check()
