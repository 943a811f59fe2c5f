"""append_cache on the GPU against the formula in 64 bits.

Bounds, per element. Rotated values: two products and a sum in 32 bits, each off
by at most 2^-24 of itself, so 2^-23 (|a cos| + |b sin|), here `slack`; 16-bit
results add one rounding, u |x| (u = 2^-11 for float16, 2^-8 for bfloat16) or half
of float16's smallest step. Codes: half a step 2^e, plus slack. Values of a
cache in 8 bits and rows that are not rotated are exact: equal. An exponent e is
the smallest with max <= 127 * 2^e, where max is known to within the slack."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}
RANGE = {torch.float16: (-24, 9), torch.bfloat16: (-126, 120)}


def angles(rows, rotary, seed=0):
    """cos and sin of real angles, [rows][rotary] float32."""
    half = rotary // 2
    a = torch.arange(rows, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(half, device="cuda") / half)
    return torch.cat([a.cos(), a.sin()], -1).float()


class Case:
    """`lengths` = [(new tokens, slots)]; `rows` more rows of q lie behind the last sequence."""

    def __init__(self, lengths, heads=4, kv_heads=2, dim=128, page=16, dtype=torch.float16, int8=False, rotary=None,
                 interleaved=False, positions=False, layout="nhd", seed=0, rows=0, pages=None, scale=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lengths, self.dim, self.page, self.dtype, self.int8 = lengths, dim, page, dtype, int8
        self.rotary, self.interleaved, self.hk, self.hq = dim if rotary is None else rotary, interleaved, kv_heads, heads
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda") * scale  # noqa: E731
        batch, tokens = len(lengths), sum(q for q, _ in lengths)
        columns = max([-(-n // page) for _, n in lengths] + [1])
        pages = pages or batch * columns + 3
        shape = (pages, page, kv_heads, dim) if layout == "nhd" else (pages, kv_heads, page, dim)
        view = (lambda t: t) if layout == "nhd" else (lambda t: t.transpose(1, 2))
        cached = torch.int8 if int8 else dtype

        def pool():
            if not int8:
                return view(rand(*shape).to(dtype))
            return view(torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=cached))

        self.k_pages, self.v_pages = pool(), pool()
        self.exponents = torch.randint(-9, -2, (pages, kv_heads, page // 16, 2), generator=g, device="cuda",
                                       dtype=torch.int8) if int8 else None
        order = torch.randperm(pages, generator=g, device="cuda").int()
        self.page_table = order[:batch * columns].reshape(batch, columns).clone()
        qkv = rand(tokens + rows, heads + 2 * kv_heads, dim).to(dtype)
        self.q, self.k_new, self.v_new = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        self.q_out = torch.full((tokens + rows, heads, dim), 7.0, dtype=dtype, device="cuda")
        self.q_start = torch.tensor([0] + [q for q, _ in lengths], device="cuda").cumsum(0).int()
        self.kv_len = torch.tensor([n for _, n in lengths], dtype=torch.int32, device="cuda")
        longest = max([n for _, n in lengths] + [1])
        self.cos_sin = angles(longest + 50, self.rotary) if self.rotary else None
        self.positions = torch.randint(0, longest + 50, (tokens + rows,), generator=g, device="cuda",
                                       dtype=torch.int32) if positions and self.rotary else None
        self.error = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.keep()

    def keep(self):
        self.before = [t.clone() if t is not None else None for t in (self.k_pages, self.v_pages, self.exponents)]

    def kwargs(self):
        return dict(k_new=self.k_new, v_new=self.v_new, k_pages=self.k_pages, v_pages=self.v_pages,
                    page_table=self.page_table, q_start=self.q_start, kv_len=self.kv_len,
                    q=self.q if self.rotary else None, q_out=self.q_out if self.rotary else None, cos_sin=self.cos_sin,
                    positions=self.positions, interleaved=self.interleaved, exponents=self.exponents, error=self.error)

    def turned(self, x, position):
        """x [heads][dim] of one token, and the slack of each element."""
        y, slack = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
        if self.rotary:
            half = self.rotary // 2
            i = torch.arange(half, device="cuda")
            a, b = (2 * i, 2 * i + 1) if self.interleaved else (i, i + half)
            c, s = self.cos_sin[position, :half].double(), self.cos_sin[position, half:].double()
            y[:, a], y[:, b] = x[:, a].double() * c - x[:, b].double() * s, x[:, b].double() * c + x[:, a].double() * s
            slack[:, a] = 2.0 ** -23 * ((x[:, a].double() * c).abs() + (x[:, b].double() * s).abs())
            slack[:, b] = 2.0 ** -23 * ((x[:, b].double() * c).abs() + (x[:, a].double() * s).abs())
        return y, slack

    def near(self, got, want, slack):
        top = torch.finfo(self.dtype).max
        inside = want.abs() <= top
        tol = slack + UNIT[self.dtype] * (want.abs() + slack) + 2.0 ** -25
        assert ((got.double() - want).abs() <= tol)[inside].all()

    def check(self, skip=()):
        """Everything that the call writes, and that it writes nothing else. `skip`: sequences that it leaves out."""
        assert not skip or self.error.item()
        k_pages, v_pages, exponents = self.before
        written, at, q_rows = [], 0, torch.zeros(len(self.q), dtype=torch.bool, device="cuda")
        for b, (q, n) in enumerate(self.lengths):
            if b in skip:
                at += q
                continue
            for t in range(q):
                slot = n - q + t
                where = int(self.positions[at + t]) if self.positions is not None else slot
                if slot < 0 and self.positions is None:
                    continue
                if self.rotary:
                    q_rows[at + t] = True
                    self.near(self.q_out[at + t], *self.turned(self.q[at + t], where))
                if slot < 0:
                    continue
                page, row = int(self.page_table[b, slot // self.page]), slot % self.page
                if not self.int8:
                    if self.rotary:
                        self.near(self.k_pages[page, row], *self.turned(self.k_new[at + t], where))
                    else:
                        assert torch.equal(self.k_pages[page, row], self.k_new[at + t])
                    assert torch.equal(self.v_pages[page, row], self.v_new[at + t])
                    k_pages[page, row], v_pages[page, row] = self.k_pages[page, row], self.v_pages[page, row]
            if self.int8 and min(q, n):
                for block in range(max(0, n - q) // 16, (n - 1) // 16 + 1):
                    self.check_block(b, block, at, q, n)
            at += q
        assert torch.equal(self.k_pages, k_pages) and torch.equal(self.v_pages, v_pages)
        if self.int8:
            assert torch.equal(self.exponents, exponents)
        if self.rotary:
            assert (self.q_out[~q_rows] == 7).all()

    def check_block(self, b, block, at, q, n):
        """Checks a block of a cache in 8 bits, and marks it in `before` as it should be."""
        first, start, end = n - q, max(block * 16, n - q), min(block * 16 + 16, n)
        page, row = int(self.page_table[b, block * 16 // self.page]), block * 16 % self.page
        lowest, highest = RANGE[self.dtype]
        for kv, (pages, new) in enumerate(((self.k_pages, self.k_new), (self.v_pages, self.v_new))):
            was = self.before[kv]
            rows = [(new[at + s - first].double(), 0) if kv else
                    self.turned(new[at + s - first], s if self.positions is None else int(self.positions[at + s - first]))
                    for s in range(start, end)]
            x = torch.stack([r[0] for r in rows])
            slack = torch.stack([r[1] for r in rows]) if not kv else torch.zeros_like(x)
            for h in range(self.hk):
                e_was = int(self.before[2][page, h, row // 16, kv])
                e = int(self.exponents[page, h, row // 16, kv])
                older = start > block * 16
                top, give = float(x[:, h].abs().max()), float(slack[:, h].max())
                least = max(lowest, e_was if older else lowest)
                if e_was == -128 and older:
                    assert e == -128
                    self.before[kv][page, row:row + 16, h] = pages[page, row:row + 16, h]
                    continue
                assert least <= e <= max(highest, least)
                assert e == highest or top - give <= 127 * 2.0 ** e
                assert e == least or top + give > 127 * 2.0 ** (e - 1)
                at_row = row + start - block * 16
                got = pages[page, at_row:at_row + end - start, h].double()
                inside = x[:, h].abs() <= 127 * 2.0 ** e
                off = (got * 2.0 ** e - x[:, h]).abs() - 0.5 * 2.0 ** e - slack[:, h]
                assert (off[inside] <= 0).all() and (got.abs() <= 127).all()
                assert (got[~inside].abs() == 127).all()
                old = was[page, row:at_row, h].double()
                was[page, row:at_row, h] = torch.round(old * 2.0 ** (e_was - e)).to(torch.int8) if older else \
                    was[page, row:at_row, h]
                was[page, at_row:at_row + end - start, h] = pages[page, at_row:at_row + end - start, h]
                self.before[2][page, h, row // 16, kv] = e

    def run(self, **kw):
        from leanstream_b200 import append_cache

        append_cache(**self.kwargs(), **kw)
        torch.cuda.synchronize()
        assert self.error.item() == 0
        self.check()


LENGTHS = [[(1, 1)], [(1, 16), (1, 17), (1, 40), (0, 9), (1, 33)], [(5, 5), (20, 70), (1, 31), (16, 32)], [(70, 130), (33, 33)]]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,rotary,interleaved", [(64, 64, False), (64, 32, True), (64, 48, False), (128, 128, False),
                                                    (128, 128, True), (128, 16, False), (128, 80, False), (128, 0, False)])
def test_rows_and_queries(cuda_device, native_lib, dim, rotary, interleaved, dtype, int8):
    for i, lengths in enumerate(LENGTHS):
        Case(lengths, (4, 7, 2, 9)[i], (2, 1, 2, 3)[i], dim, 16 << i, dtype, int8, rotary, interleaved, positions=i % 2,
             seed=i).run()


@pytest.mark.parametrize("int8", [False, True])
def test_layouts_positions_and_rows_behind(cuda_device, native_lib, int8):
    for i, lengths in enumerate(LENGTHS):
        Case(lengths, layout="hnd", int8=int8, rows=5, positions=True, seed=i, page=32).run()
    Case([(2, 40)] * 300, 2, 1, 64, int8=int8).run()  # more sequences than threads
    Case([(9, 4), (20, 0), (30, 12)], int8=int8).run()  # more tokens than slots
    Case([(9, 4), (20, 0), (30, 12)], int8=int8, positions=True).run()


@pytest.mark.parametrize("int8", [False, True])
def test_keys_alone_large_pages_and_slices(cuda_device, native_lib, int8):
    """No queries; pages of 256 slots; pools that are one layer's part of all layers'; a key head for all."""
    from leanstream_b200 import append_cache

    for dim in (64, 128):
        c = Case(LENGTHS[2], dim=dim, page=256, int8=int8)
        for name in ("k_pages", "v_pages", "exponents")[:3 if int8 else 2]:
            t = getattr(c, name)
            layers = torch.zeros(t.shape[0], 3, *t.shape[1:], dtype=t.dtype, device="cuda")
            layers[:, 1] = t
            setattr(c, name, layers[:, 1])
        c.k_new = c.k_new[:, :1].expand(-1, 2, -1)
        c.keep()
        append_cache(**{**c.kwargs(), "q": None, "q_out": None})
        torch.cuda.synchronize()
        assert (c.q_out == 7).all()
        append_cache(**c.kwargs())
        torch.cuda.synchronize()
        assert c.error.item() == 0
        c.check()


@pytest.mark.parametrize("int8", [False, True])
def test_many_sequences_and_tokens(cuda_device, native_lib, int8):
    """Against the same rows appended sequence by sequence: more tasks than warps, and
    more sequences than a CTA counts at a time."""
    from leanstream_b200 import append_cache

    for lengths in ([(700 + 37 * i, 900 + 41 * i) for i in range(9)], [(1 + i % 5, 9 + i % 40) for i in range(700)]):
        c = Case(lengths, 12, 4, 128, 32, torch.bfloat16, int8, 48, positions=True)
        append_cache(**c.kwargs())
        torch.cuda.synchronize()
        assert c.error.item() == 0
        got = [t.clone() for t in (c.k_pages, c.v_pages, c.q_out)] + ([c.exponents.clone()] if int8 else [])
        for now, was in zip((c.k_pages, c.v_pages, c.exponents), c.before):
            if now is not None:
                now.copy_(was)
        c.q_out.fill_(7)
        at = 0
        for b, (q, n) in enumerate(lengths):
            part = slice(at, at + q)
            append_cache(**{**c.kwargs(), "k_new": c.k_new[part], "v_new": c.v_new[part], "q": c.q[part],
                            "q_out": c.q_out[part], "positions": c.positions[part], "kv_len": c.kv_len[b:b + 1],
                            "page_table": c.page_table[b:b + 1],
                            "q_start": torch.tensor([0, q], dtype=torch.int32, device="cuda")})
            at += q
        torch.cuda.synchronize()
        for a, b in zip(got, (c.k_pages, c.v_pages, c.q_out, c.exponents)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("int8", [False, True])
def test_queries_in_place_and_streams(cuda_device, native_lib, int8):
    c = Case(LENGTHS[2], int8=int8)
    same = c.q.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    from leanstream_b200 import append_cache

    append_cache(stream=stream, **{**c.kwargs(), "q": same, "q_out": same})
    with torch.cuda.stream(stream):
        append_cache(**{**c.kwargs(), "q": c.q, "q_out": c.q_out})
    stream.synchronize()
    assert torch.equal(same, c.q_out) and c.error.item() == 0
    c.check()


@pytest.mark.parametrize("int8", [False, True])
def test_graph(cuda_device, native_lib, int8):
    """Replayed with lengths that grew on the device since the capture."""
    from leanstream_b200 import append_cache

    c = Case([(1, 70), (1, 31)], int8=int8)
    c.kv_len -= 20
    append_cache(**c.kwargs())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append_cache(**c.kwargs())
    for _ in range(20):
        c.kv_len += 1
        c.q_out.fill_(7)
        c.keep()
        graph.replay()
        torch.cuda.synchronize()
        lengths = c.kv_len.tolist()
        c.lengths = [(1, n) for n in lengths]
        c.check()
    assert lengths == [70, 31]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_block_that_grows(cuda_device, native_lib, dtype):
    """Token by token, with larger and larger rows: every row ends within one
    step of its value (half a step, and half of each wider one after it)."""
    from leanstream_b200 import append_cache

    g = torch.Generator(device="cuda").manual_seed(3)
    c = Case([(1, 48)], kv_heads=2, int8=True, rotary=0, dtype=dtype)
    x = torch.randn(48, 2, 128, generator=g, device="cuda") * 2.0 ** torch.linspace(-7, 5, 48, device="cuda")[:, None, None]
    x = x.to(dtype)
    for n in range(1, 49):
        c.kv_len.fill_(n)
        append_cache(**{**c.kwargs(), "k_new": x[n - 1:n], "v_new": -x[n - 1:n]})
    torch.cuda.synchronize()
    for kv, (pages, sign) in enumerate(((c.k_pages, 1), (c.v_pages, -1))):
        for n in range(48):
            page = int(c.page_table[0, n // 16])
            step = 2.0 ** c.exponents[page, :, 0, kv].double()[:, None]
            off = (pages[page, n % 16].double() * step - sign * x[n].double()).abs()
            assert (off < step).all()


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite(cuda_device, native_lib, value):
    """A block that takes one is marked, stays so while it goes on, and begins anew with its first slot."""
    from leanstream_b200 import append_cache

    c = Case([(1, 40), (20, 40)], int8=True, rotary=0)
    c.k_new[0, 1, 5], c.v_new[3, 0, 9] = value, value
    append_cache(**c.kwargs())
    torch.cuda.synchronize()
    first, other = int(c.page_table[0, 2]), int(c.page_table[1, 1])  # slots 39, and 22 in the second one
    marked = (c.exponents == -128).nonzero().tolist()
    assert sorted(marked) == sorted([[first, 1, 0, 0], [other, 0, 0, 1]])
    c.k_new[0, 1, 5], c.v_new[3, 0, 9] = 0, 0
    c.keep()
    append_cache(**c.kwargs())
    torch.cuda.synchronize()
    # both blocks hold older slots, and stay marked
    assert int(c.exponents[first, 1, 0, 0]) == int(c.exponents[other, 0, 0, 1]) == -128
    c.check()
    begin = Case([(8, 40), (24, 40)], int8=True, rotary=0)
    begin.exponents.fill_(-128)
    begin.keep()
    begin.run()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_smallest_and_largest_values(cuda_device, native_lib, dtype):
    info = torch.finfo(dtype)
    for x in (0.0, info.smallest_normal / 4 if dtype is torch.float16 else info.smallest_normal, info.max,
              127 * 2.0 ** -5, 127.5 * 2.0 ** -5, -info.max):
        c = Case([(3, 19), (1, 1)], int8=True, rotary=0, dtype=dtype)
        c.k_new.fill_(x)
        c.v_new.mul_(0.001)
        c.v_new[0] = x
        c.run()
        if x == 0.0:
            assert (c.exponents[int(c.page_table[1, 0]), :, 0, 0] == RANGE[dtype][0]).all()
    c = Case([(3, 19), (20, 20)], dtype=dtype, scale=info.max / 8)  # rotated keys may pass the largest number
    c.run()
    c = Case([(3, 19), (20, 20)], dtype=dtype, scale=info.max / 8, int8=True)
    c.run()


@pytest.mark.parametrize("int8", [False, True])
def test_offsets_past_32_bits(cuda_device, native_lib, int8):
    c = Case([(20, 300), (1, 90)], 2, 8, 128, page=64, int8=int8, rotary=32)
    pages = 70000
    k, v = (torch.zeros(pages, 64, 8, 128, dtype=c.k_pages.dtype, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 32
    n = c.k_pages.shape[0]
    k[-n:], v[-n:] = c.k_pages, c.v_pages
    if int8:
        ex = torch.zeros(pages, 8, 4, 2, dtype=torch.int8, device="cuda")
        ex[-n:] = c.exponents
        c.exponents = ex
    c.k_pages, c.v_pages = k, v
    c.page_table += pages - n
    c.keep()
    c.run()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("bad", [0, 1, 2])
def test_what_does_not_fit_is_left_out(cuda_device, native_lib, bad, int8):
    """Lengths, pages and positions: reported, their neighbours are right, theirs is as it was."""
    from leanstream_b200 import _native as N, append_cache

    for length in (1 << 20, -1, -(1 << 31), (1 << 31) - 1):
        c = Case([(5, 60), (5, 33), (5, 20)], int8=int8)
        c.kv_len[bad] = length
        append_cache(**c.kwargs())
        torch.cuda.synchronize()
        assert c.error.item() == N.ATTN_LENGTH
        c.check(skip=(bad,))
    for index in (-1, -(1 << 31), (1 << 31) - 1, None):
        c = Case([(5, 60), (5, 31), (5, 20)], int8=int8)
        page = c.page_table[bad, (c.lengths[bad][1] - 1) // 16].clone()
        c.page_table[bad, (c.lengths[bad][1] - 1) // 16] = c.k_pages.shape[0] if index is None else index
        append_cache(**c.kwargs())
        torch.cuda.synchronize()
        assert c.error.item() == N.ATTN_PAGE
        assert torch.equal(c.k_pages[page.long()], c.before[0][page.long()])
        for b in range(3):  # its queries too
            for t in range(5):
                c.near(c.q_out[5 * b + t], *c.turned(c.q[5 * b + t], c.lengths[b][1] - 5 + t))
    for at in (-1, 1 << 20, -(1 << 31)):
        c = Case([(5, 60), (5, 31), (5, 20)], int8=int8, positions=True)
        c.positions[5 * bad:5 * bad + 5] = at
        append_cache(**c.kwargs())
        torch.cuda.synchronize()
        assert c.error.item() == N.ATTN_POSITION
        c.check(skip=(bad,))
