"""Attention over a paged cache in 8 bits whose values are all small, or lie far
apart, against the formula in 64 bits on the values that the cache stands for.

Bounds, per element, all relative to what is computed (u: half a step of the output's
type; A = sum p |v|; E: the largest exponent of the sequence's visible values):
the output is rounded once, u |out|, or half the type's smallest step; a
probability is rounded once to 16 bits, r A (few rows: float16, r = 2^-11; chunks:
the queries' type, r = u), and where that is float16 it ends at half of its smallest
step, 2^-25, taken after a shift of 2^7: 2^-32 of the row's largest, times 2^(E - e),
times a code of at most 128 here, for each of the n slots: n 2^(E - 25); the
exponential and the logits (below 40) are good to 1e-5 of a probability, twice with
the normalisation: 2e-5 A. The output's rounding also meets the errors before it."""
import pytest
import torch

from test_gpu_attention import UNIT
from test_gpu_attention_int8 import Call8

pytestmark = pytest.mark.gpu

SMALLEST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
FEW = 32  # rows of a kv head on the kernel of few rows


class Small(Call8):
    """Call8 with its values, of exponents -8 to -5, times 2^shift; blocks that no row sees stay marked."""

    def __init__(self, lengths, shift, **kw):
        super().__init__(lengths, **kw)
        e = self.exponents[..., 1]
        e[e != -128] += shift
        self.values = [v * 2.0 ** shift for v in self.values]
        self.largest = -5 + shift

    def check(self):
        out, area, lse, _, _ = self.expected()
        u, few = UNIT[self.dtype], self.max_q * (self.heads // self.kv_heads) <= FEW
        r = 2.0 ** -11 if few else u
        end = 2.0 ** (self.largest - 25) if few or self.dtype is torch.float16 else 0.0
        slots = torch.cat([torch.full((q,), float(n)) for q, n in self.lengths]).cuda()[:, None, None]
        before = (r + 2e-5) * area + end * slots
        tol = u * (out.abs() + before) + before + SMALLEST[self.dtype] / 2
        assert torch.isfinite(self.output).all()
        off = ((self.output.double() - out).abs() / tol).amax((1, 2))
        assert (off <= 1).all(), f"output off by {off.max().item():.3g} of its bound"
        empty = torch.isinf(lse)
        assert torch.equal(empty, torch.isinf(self.lse)) and (self.output[empty] == 0).all()
        if (~empty).any():
            assert (self.lse.double() - lse)[~empty].abs().max().item() <= 2e-5

    def run(self):
        engine = self.engine()
        engine.run(**self.kwargs())
        torch.cuda.synchronize()
        assert engine.error() == 0
        self.check()


# float16 takes exponents from -24, bfloat16 from -126
SHIFTS = [(torch.float16, -12), (torch.float16, -16), (torch.bfloat16, -15), (torch.bfloat16, -35),
          (torch.bfloat16, -100)]
SHORT = [1, 15, 16, 17, 32, 33, 48, 49, 65, 300, 304]


@pytest.mark.parametrize("q", [1, 4, 6, 8, 40])
@pytest.mark.parametrize("dtype,shift", SHIFTS)
def test_lengths_that_end_in_a_first_block(cuda_device, native_lib, dtype, shift, q):
    for page in (16, 32, 128):
        lengths = [(min(q, n), n) for n in SHORT]
        Small(lengths, shift, dtype=dtype, page=page, seed=page).run()
        Small(lengths, shift, dtype=dtype, page=page, heads=16, kv_heads=4, dim=64, seed=page).run()


@pytest.mark.parametrize("q", [1, 4, 8, 40])
@pytest.mark.parametrize("dtype,shift", SHIFTS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 4), (90, 16), (200, 1), (500, 20)])
def test_windows_and_first_slots(cuda_device, native_lib, dtype, shift, window, sinks, q):
    """Windows that begin in a second block, and first slots of one block, which the window has left."""
    lengths = [(q, 600 + 11 * i) for i in range(3)] + [(1, 4000)]
    for page in (16, 64):
        Small(lengths, shift, dtype=dtype, page=page, window=window, sinks=sinks, seed=page).run()


@pytest.mark.parametrize("q", [1, 6, 40])
@pytest.mark.parametrize("dtype,shift", SHIFTS)
def test_pages_outside_the_pool(cuda_device, native_lib, dtype, shift, q):
    """They are reported, read as zeros, and leave the others' accuracy alone."""
    from leanstream_b200 import _native as N

    for page, at in ((16, 3), (16, 6), (32, 0)):
        c = Small([(q, 200), (q, 90)], shift, dtype=dtype, page=page)
        c.page_table[0, at] = c.k_pages.shape[0] if at else -1
        for t in (c.keys[0], c.values[0]):
            t[at * page:(at + 1) * page] = 0
        engine = c.engine()
        engine.run(**c.kwargs())
        torch.cuda.synchronize()
        assert engine.error() == N.ATTN_PAGE
        c.check()


@pytest.mark.parametrize("q", [1, 4, 6, 8, 40, 100])
@pytest.mark.parametrize("shift", [-111, -115, -117, -118])
def test_the_lowest_exponents(cuda_device, native_lib, shift, q):
    """bfloat16 down to -126."""
    for page in (16, 32):
        Small([(min(q, n), n) for n in SHORT], shift, dtype=torch.bfloat16, page=page).run()
        c = Small([(q, 500), (q, 2000)], shift, dtype=torch.bfloat16, page=page, heads=16, kv_heads=8, dim=64)
        for b, n in enumerate((500, 2000)):  # every block at the lowest one
            i = torch.arange(n, device="cuda")
            where = c.page_table[b].long()[i // page]
            c.exponents[where, :, i // 16 % (page // 16), 1] = -126
            c.values[b] = c.v_pages[where, i % page].double() * 2.0 ** -126
        c.largest = -126
        c.run()


@pytest.mark.parametrize("q", [1, 6])
def test_values_of_no_weight_and_a_large_exponent(cuda_device, native_lib, q):
    """A block 2^226 above the others whose probabilities are far below 2^-226: the others may count as 0,
    and for no more than themselves."""
    c = Small([(q, 600)], -118, dtype=torch.bfloat16, page=16, spread=1, marked=False)
    where = int(c.page_table[0, 16])  # slots 256 to 271, of a warp that has taken earlier ones
    # logits near -570, against the others' few tens
    c.k_pages[where] = -127
    c.q.abs_()
    c.exponents[where, :, 0, 0], c.exponents[where, :, 0, 1] = -1, 100
    c.keys[0][256:272] = -63.5
    c.values[0][256:272] = c.v_pages[where].double() * 2.0 ** 100
    engine = c.engine()
    engine.run(**c.kwargs())
    torch.cuda.synchronize()
    assert engine.error() == 0
    _, area, lse, _, _ = c.expected()
    # area + u (area + ..), with the probabilities' own rounding
    assert (c.output.double().abs() <= area * (1 + 2.0 ** -8) * (1 + 2.0 ** -10) + SMALLEST[torch.bfloat16] / 2).all()
    assert (c.lse.double() - lse).abs().max().item() <= 2e-5


@pytest.mark.parametrize("dtype,scale", [(torch.float16, 2.0 ** -13), (torch.bfloat16, 2.0 ** -40), (torch.bfloat16, 2.0 ** -112)])
def test_decoding_with_small_values(cuda_device, native_lib, dtype, scale):
    """Token after token through append_cache and the attention, past the ends of blocks and steps."""
    from leanstream_b200 import append_cache

    c = Small([(1, 70)], 0, dtype=dtype, page=32)
    g = torch.Generator(device="cuda").manual_seed(9)
    k, v = (torch.randn(70, 2, 128, generator=g, device="cuda") for _ in range(2))
    k, v = k.to(dtype), (v * scale).to(dtype)
    c.exponents.zero_()
    starts, engine, got = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), c.engine(), []
    for n in range(1, 71):
        c.kv_len.fill_(n)
        append_cache(k_new=k[n - 1:n], v_new=v[n - 1:n], k_pages=c.k_pages, v_pages=c.v_pages, exponents=c.exponents,
                     page_table=c.page_table, q_start=starts, kv_len=c.kv_len)
        engine.run(**c.kwargs())
        got.append([t.clone() for t in (c.output, c.lse, c.k_pages, c.v_pages, c.exponents)])
    torch.cuda.synchronize()
    assert engine.error() == 0
    for n, (output, lse, k_pages, v_pages, exponents) in enumerate(got, 1):
        i = torch.arange(n, device="cuda")
        where = c.page_table[0].long()[i // 32]
        size = exponents[where, :, i // 16 % 2].double()
        c.lengths, c.largest, c.output, c.lse = [(1, n)], float(size[..., 1].max()), output, lse
        c.keys, c.values = ([p[where, i % 32].double() * (2.0 ** size[..., j])[..., None]]
                            for j, p in enumerate((k_pages, v_pages)))
        c.check()
        assert (c.values[0] - v[:n].double()).abs().max() < 2.0 ** c.largest
