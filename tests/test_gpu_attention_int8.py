"""Attention over a paged cache in 8 bits on the GPU, against the formula in 64
bits on the values that the cache stands for (code * 2^exponent).

Bounds as in test_gpu_attention.py: codes and their powers of two are exact in
every operand, so nothing is added but, where the exponents of a sequence's
values lie far apart, what float16 probabilities lose below the largest: each is
off by at most 2^-40 of 2^E (E the sequence's largest exponent), times a code of
at most 127."""
import math

import pytest
import torch

from test_gpu_attention import DECODE, HEADS, UNIT, Call

pytestmark = pytest.mark.gpu


class Call8(Call):
    """Blocks without a visible slot are marked (exponent -128) and hold any codes; so do the slots behind."""

    def __init__(self, lengths, heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16, window=0, sinks=0, seed=0,
                 layout="nhd", q_scale=1.0, spread=4, extra_pages=3, marked=True):
        super().__init__(lengths, heads, kv_heads, dim, page, dtype, window, sinks, False, seed, "nhd", False, q_scale,
                         extra_pages)
        g = torch.Generator(device="cuda").manual_seed(1000 + seed)
        pages = self.k_pages.shape[0]
        shape = (pages, page, kv_heads, dim) if layout == "nhd" else (pages, kv_heads, page, dim)
        view = (lambda t: t) if layout == "nhd" else (lambda t: t.transpose(1, 2))
        self.k_pages, self.v_pages = (view(torch.randint(-128, 128, shape, generator=g, device="cuda",
                                                         dtype=torch.int8)) for _ in range(2))
        self.exponents = torch.randint(-4 - spread, -4, (pages, kv_heads, page // 16, 2), generator=g, device="cuda",
                                       dtype=torch.int8)
        kept = self.exponents.clone()
        if marked:
            self.exponents.fill_(-128)
        self.keys, self.values = [], []
        for b, (q, n) in enumerate(lengths):
            first, i = n - q, torch.arange(n, device="cuda")
            seen = (i > first - window) | (i < sinks) if window else i >= 0
            where = self.page_table[b].long()[i // page]
            held = (where >= 0) & (where < pages)
            where = where.clamp(0, pages - 1)
            blocks = i // 16 % (page // 16)
            self.exponents[where[seen], :, blocks[seen]] = kept[where[seen], :, blocks[seen]]
            step = 2.0 ** kept[where, :, blocks].double()
            for kv, (pool, got) in enumerate(((self.k_pages, self.keys), (self.v_pages, self.values))):
                got.append(torch.where(held[:, None, None], pool[where, i % page].double() * step[..., kv][..., None], 0))
        if heads * dim and dtype is torch.float16:
            self.q *= 0.5

    def engine(self, **kw):
        from leanstream_b200 import PagedAttention

        return PagedAttention(self.heads, self.kv_heads, self.dim, page_size=self.page, dtype=self.dtype,
                              cache_dtype="int8", max_sequences=len(self.lengths), max_tokens=max(1, self.q.shape[0]),
                              max_queries=max(1, self.max_q), **kw)

    def kwargs(self):
        return {**super().kwargs(), "exponents": self.exponents}

    def check(self):
        before = [t.clone() for t in (self.k_pages, self.v_pages, self.exponents)]
        super().check()
        assert all(torch.equal(a, b) for a, b in zip(before, (self.k_pages, self.v_pages, self.exponents)))


CHUNKS = [(2, 2), (5, 70), (1, 300)], [(33, 33), (0, 5), (64, 200), (1, 129)], [(150, 421)], [(257, 257), (3, 640)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
def test_one_token_each(cuda_device, native_lib, dtype, heads):
    for i, lengths in enumerate(DECODE):
        Call8(lengths, *heads, dtype=dtype, page=16 << i, seed=i, q_scale=2.0).run()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
def test_chunks(cuda_device, native_lib, dtype, heads):
    for i, lengths in enumerate(CHUNKS):
        Call8(lengths, *heads, dtype=dtype, page=16 << i, seed=10 + i, q_scale=2.0).run()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 0), (100, 17), (128, 130), (1000, 4)])
@pytest.mark.parametrize("lengths", [[(1, 1), (1, 90), (1, 700)], [(5, 5), (9, 400)], [(140, 140), (200, 611), (1, 350)]])
def test_window_and_first_slots(cuda_device, native_lib, lengths, window, sinks):
    Call8(lengths, 8, 2, 128, page=16, window=window, sinks=sinks, dtype=torch.bfloat16).run()
    Call8(lengths, 6, 2, 64, page=32, window=window, sinks=sinks).run()


@pytest.mark.parametrize("q", [1, 6, 90])
def test_rows_without_slots(cuda_device, native_lib, q):
    Call8([(q, max(0, q - 3)), (q, q // 2), (q, 0), (q, 200)]).run()


@pytest.mark.parametrize("q", [1, 8, 70])
def test_layouts_long_caches_and_reuse(cuda_device, native_lib, q):
    Call8([(q, 200), (1, 77)], layout="hnd", page=32).run()
    Call8([(q, 9000)], page=64, q_scale=2.0, dtype=torch.bfloat16).run()
    Call8([(1 + i % q, 40 + 37 * i) for i in range(40)], q_scale=2.0).run()
    Call8([(1 + i % q, 10 + i) for i in range(150)], 2, 2, 64, q_scale=2.0).run()
    c = Call8([(q, 3000), (q, 129)], q_scale=2.0)
    engine = c.engine()
    engine.run(**c.kwargs())
    torch.cuda.synchronize()
    again = c.output.clone(), c.lse.clone()
    c.output.fill_(7)
    engine.run(**c.kwargs())
    torch.cuda.synchronize()
    assert torch.equal(again[0], c.output) and torch.equal(again[1], c.lse)
    c.check()


@pytest.mark.parametrize("q", [1, 2, 3])
@pytest.mark.parametrize("heads", [(16, 16, 64), (12, 6, 64), (24, 3, 64), (16, 4, 128)])
def test_many_sequences(cuda_device, native_lib, heads, q):
    """Items of one, two and four kv heads, more than one list of pieces per CTA, windows among them."""
    lengths = [(1 + i % q, 5 + 13 * i % 700) for i in range(80)] + [(0, 3), (q, 1), (q, 0)]
    Call8(lengths, *heads, page=16, q_scale=2.0).run()
    Call8(lengths, *heads, page=64, dtype=torch.bfloat16, layout="hnd", window=100, sinks=3).run()
    Call8([(q, 7 + i % 60) for i in range(500)], heads[0] // heads[1], 1, heads[2], page=32).run()


@pytest.mark.parametrize("q", [1, 60])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_exponents_far_apart(cuda_device, native_lib, dtype, q):
    """Values from blocks 2^18 apart, in either order, and keys of little and much weight."""
    for seed in range(3):
        c = Call8([(q, 400), (q, 90)], dtype=dtype, spread=18, seed=seed, q_scale=2.0 ** 9 if seed else 1.0)
        if seed:  # keys small enough for logits of some tens
            c.exponents[..., 0].clamp_(max=-16)
            for b, (_, n) in enumerate(c.lengths):
                i = torch.arange(n, device="cuda")
                where = c.page_table[b].long()[i // 16]
                c.keys[b] = c.k_pages[where, i % 16].double() * 2.0 ** c.exponents[where, :, 0, 0].double()[..., None]
        engine = c.engine()
        engine.run(**c.kwargs())
        torch.cuda.synchronize()
        assert engine.error() == 0
        out, area, lse, _, _ = c.expected()
        scale = max(1.0, lse[torch.isfinite(lse)].abs().max().item())
        err = (c.output.double() - out).abs()
        # logits of size `scale`: their 32-bit rounding is that much larger than in test_gpu_attention.py's 40
        tol = UNIT[dtype] * (out.abs() + area) + 2e-5 * max(1.0, scale / 40) * area + 2.0 ** -24 + \
            127 * 400 * 2.0 ** (-5 - 40)
        assert (err <= tol).all(), (err / tol).max()
        assert ((c.lse.double() - lse).abs() <= 2e-5 * max(1.0, scale / 40)).all()


@pytest.mark.parametrize("q", [1, 60])
@pytest.mark.parametrize("kv", [0, 1])
def test_a_marked_block_reads_as_nan(cuda_device, native_lib, q, kv):
    c = Call8([(q, 200), (q, 150)])
    out, area, lse, _, _ = c.expected()
    c.exponents[c.page_table[1, 2].long(), 1, 0, kv] = -128
    engine = c.engine()
    engine.run(**c.kwargs())
    torch.cuda.synchronize()
    assert engine.error() == 0
    assert c.output[q:, 4:].isnan().all() and (kv or c.lse[q:, 4:].isnan().all())
    rest = torch.ones_like(c.lse, dtype=torch.bool)
    rest[q:, 4:] = False
    err, tol = (c.output.double() - out).abs(), UNIT[c.dtype] * (out.abs() + area) + 2e-5 * area + 2.0 ** -24
    assert (err <= tol)[rest].all()


@pytest.mark.parametrize("q", [1, 60])
def test_queries_that_are_not_finite(cuda_device, native_lib, q):
    for dtype in (torch.float16, torch.bfloat16):
        for value in (math.inf, math.nan):
            c = Call8([(q, 200), (q, 150)], dtype=dtype)
            out, area, _, _, _ = c.expected()
            c.q[q, 3, 7] = value
            engine = c.engine()
            engine.run(**c.kwargs())
            torch.cuda.synchronize()
            assert c.output[q, 3].isnan().all() and c.lse[q, 3].isnan()
            rest = torch.ones_like(c.lse, dtype=torch.bool)
            rest[q, 3] = False
            err, tol = (c.output.double() - out).abs(), UNIT[dtype] * (out.abs() + area) + 2e-5 * area + 2.0 ** -24
            assert (err <= tol)[rest].all()


@pytest.mark.parametrize("q", [1, 60])
def test_small_and_large_queries(cuda_device, native_lib, q):
    """Queries of bfloat16's range, against keys that bring the logits back."""
    for power in (-60, 60):
        c = Call8([(q, 200), (q, 150)], dtype=torch.bfloat16, marked=False)
        c.q *= 2.0 ** power
        c.exponents[..., 0] -= power
        for b in range(2):
            c.keys[b] = c.keys[b] * 2.0 ** -power
        c.run()


@pytest.mark.parametrize("q", [1, 60])
def test_other_stream_and_graph(cuda_device, native_lib, q):
    c = Call8([(q, 500), (q, 77)])
    engine, stream = c.engine(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        engine.run(**c.kwargs())
    engine2 = c.engine()
    stream.synchronize()
    c.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        engine2.run(**c.kwargs())
    # another call of the same shape, in the captured buffers
    other = Call8([(q, 480), (q, 60)], seed=5)
    n = other.k_pages.shape[0]
    for name in ("k_pages", "v_pages", "exponents"):
        getattr(c, name)[:n] = getattr(other, name)
    c.page_table.zero_()
    c.page_table[:, :other.page_table.shape[1]] = other.page_table
    c.q.copy_(other.q), c.kv_len.copy_(other.kv_len)
    for _ in range(2):
        c.output.fill_(7), c.lse.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        other.output, other.lse = c.output, c.lse
        other.check()


@pytest.mark.parametrize("q", [1, 60])
def test_offsets_past_32_bits(cuda_device, native_lib, q):
    c = Call8([(q, 300)], 8, 8, 128, page=64)
    pages, n = 70000, c.k_pages.shape[0]
    for name in ("k_pages", "v_pages", "exponents"):
        t = getattr(c, name)
        big = torch.zeros(pages, *t.shape[1:], dtype=torch.int8, device="cuda")
        big[-n:] = t
        setattr(c, name, big)
    c.page_table[:, :5] += pages - n
    c.run()


@pytest.mark.parametrize("q", [1, 5, 60])
@pytest.mark.parametrize("dim", [64, 128])
def test_pages_of_256_and_slices_of_a_pool(cuda_device, native_lib, q, dim):
    """The largest pages; pools and exponents that are one layer's part of all layers'."""
    c = Call8([(q, 900), (q, 256), (q, 257)], 8, 2, dim, page=256)
    c.run()
    for name in ("k_pages", "v_pages", "exponents"):
        t = getattr(c, name)
        layers = torch.randint(-128, 128, (t.shape[0], 3, *t.shape[1:]), device="cuda").to(torch.int8)
        layers[:, 1] = t
        setattr(c, name, layers[:, 1])
    c.run()


@pytest.mark.parametrize("q", [1, 60])
def test_two_engines_at_once(cuda_device, native_lib, q):
    calls = [Call8([(q, 5000), (q, 300)], seed=i, page=32) for i in range(2)]
    engines, streams = [c.engine() for c in calls], [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, engine, stream in zip(calls, engines, streams):
            engine.run(stream=stream, **c.kwargs())
    torch.cuda.synchronize()
    for c, engine in zip(calls, engines):
        assert engine.error() == 0
        c.check()


@pytest.mark.parametrize("bound", [3, 64, 1 << 16])
@pytest.mark.parametrize("batch", [3, 1 << 13])
def test_loose_bound(cuda_device, native_lib, batch, bound):
    """max_q far above the new tokens, most sequences without any."""
    from leanstream_b200 import PagedAttention

    lengths = [(0, 9), (3, 300), (1, 77)] + [(0, 0)] * (batch - 3)
    lengths[-1] = lengths[-1] if batch == 3 else (2, 50)
    c = Call8(lengths, 8, 2, 64, page=32)
    engine = PagedAttention(8, 2, 64, page_size=32, cache_dtype="int8", max_sequences=batch,
                            max_tokens=c.q.shape[0], max_queries=bound)
    engine.run(**{**c.kwargs(), "max_q": bound})
    torch.cuda.synchronize()
    assert engine.error() == 0
    c.check()


@pytest.mark.parametrize("q", [1, 50])
def test_bad_lengths_and_pages_are_reported(cuda_device, native_lib, q):
    from leanstream_b200 import _native as N

    for length in (1 << 20, -1, (1 << 31) - 1):
        c = Call8([(q, 200), (q, 150), (q, 333)])
        out, area, lse, _, _ = c.expected()
        engine = c.engine()
        c.kv_len[1] = length
        engine.run(**c.kwargs())
        torch.cuda.synchronize()
        assert engine.error() == N.ATTN_LENGTH
        assert (c.output[q:2 * q] == 7).all()
        good = torch.cat([torch.arange(q), torch.arange(2 * q, 3 * q)]).cuda()
        err, tol = (c.output.double() - out).abs(), UNIT[c.dtype] * (out.abs() + area) + 2e-5 * area + 2.0 ** -24
        assert (err <= tol)[good].all()
        engine.clear_error()
        c.kv_len[1] = 150
        for index in (-1, c.k_pages.shape[0], (1 << 31) - 1):
            c.page_table[1, 2] = index
            engine.run(**c.kwargs())
            torch.cuda.synchronize()
            assert engine.error() == N.ATTN_PAGE
            engine.clear_error()
            err = (c.output.double() - out).abs()
            assert (err <= tol)[good].all()


@pytest.mark.parametrize("q", [1, 40])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_and_attend(cuda_device, native_lib, dtype, q):
    """Both calls as a decoder makes them, step after step on one stream: the
    attention reads what the append wrote (values as the cache holds them)."""
    from leanstream_b200 import PagedAttention, append_cache
    from test_gpu_append import angles

    g = torch.Generator(device="cuda").manual_seed(1)
    heads, hk, dim, page, batch, steps = 8, 2, 128, 32, 3, 5
    table = torch.randperm(60, generator=g, device="cuda")[:batch * 10].int().reshape(batch, 10)
    k_pages, v_pages = (torch.zeros(60, page, hk, dim, dtype=torch.int8, device="cuda") for _ in range(2))
    exponents = torch.zeros(60, hk, page // 16, 2, dtype=torch.int8, device="cuda")
    kv_len = torch.zeros(batch, dtype=torch.int32, device="cuda")
    q_start = (torch.arange(batch + 1, device="cuda") * q).int()
    engine = PagedAttention(heads, hk, dim, page_size=page, dtype=dtype, cache_dtype="int8", max_sequences=batch,
                            max_tokens=batch * q, max_queries=q)
    cos_sin, done = angles(400, dim), []
    for _ in range(steps):
        x = torch.randn(batch * q, heads + 2 * hk, dim, generator=g, device="cuda").to(dtype)
        out = torch.empty(batch * q, heads, dim, dtype=dtype, device="cuda")
        lse = torch.empty(batch * q, heads, device="cuda")
        kv_len += q
        turned = torch.empty_like(x[:, :heads])
        append_cache(q=x[:, :heads], q_out=turned, k_new=x[:, heads:heads + hk], v_new=x[:, heads + hk:],
                     k_pages=k_pages, v_pages=v_pages, exponents=exponents, page_table=table, q_start=q_start,
                     kv_len=kv_len, cos_sin=cos_sin)
        engine.run(q=turned, output=out, k_pages=k_pages, v_pages=v_pages, exponents=exponents, page_table=table,
                   q_start=q_start, kv_len=kv_len, max_q=q, lse=lse)
        done.append((turned, out, lse, k_pages.clone(), v_pages.clone(), exponents.clone()))
    torch.cuda.synchronize()
    assert engine.error() == 0
    for step, (turned, out, lse, kp, vp, ex) in enumerate(done):
        n = (step + 1) * q
        c = Call8([(q, n)] * batch, heads, hk, dim, page, dtype)
        c.q, c.output, c.lse, c.k_pages, c.v_pages, c.exponents = turned, out, lse, kp, vp, ex
        i = torch.arange(n, device="cuda")
        for b in range(batch):
            where = table[b].long()[i // page]
            size = 2.0 ** ex[where, :, i // 16 % (page // 16)].double()
            c.keys[b] = kp[where, i % page].double() * size[..., 0][..., None]
            c.values[b] = vp[where, i % page].double() * size[..., 1][..., None]
        c.check()


@pytest.mark.parametrize("q", [1, 40])
def test_step_in_a_graph_between_other_work(cuda_device, native_lib, q):
    """Append and attention captured after copies, fills and another stream's work,
    before some; replayed step after step with lengths that grow on the device."""
    from leanstream_b200 import PagedAttention, append_cache
    from test_gpu_append import angles

    g = torch.Generator(device="cuda").manual_seed(2)
    heads, hk, dim, page, batch, steps = 8, 2, 64, 16, 2, 4
    int8, int32 = dict(dtype=torch.int8, device="cuda"), dict(dtype=torch.int32, device="cuda")
    half = dict(dtype=torch.float16, device="cuda")
    table = torch.randperm(40, generator=g, device="cuda")[:batch * 15].int().reshape(batch, 15)
    pages, exponents = [torch.zeros(40, page, hk, dim, **int8) for _ in range(2)], torch.zeros(40, hk, 1, 2, **int8)
    kv_len, more = torch.zeros(batch, **int32), torch.full((batch,), q, **int32)
    x, given = (torch.empty(batch * q, heads + 2 * hk, dim, **half) for _ in range(2))
    out, last = torch.empty(batch * q, heads, dim, **half), torch.empty(batch * q, heads, dim, **half)
    lse = torch.empty(batch * q, heads, device="cuda")
    starts, cos_sin = (torch.arange(batch + 1, device="cuda") * q).int(), angles(200, dim)
    engine = PagedAttention(heads, hk, dim, page_size=page, cache_dtype="int8", max_sequences=batch,
                            max_tokens=batch * q, max_queries=q)
    other = torch.cuda.Stream()

    def step():
        main = torch.cuda.current_stream()
        other.wait_stream(main)
        with torch.cuda.stream(other):
            kv_len.add_(more)
        x.copy_(given)
        main.wait_stream(other)
        append_cache(q=x[:, :heads], q_out=x[:, :heads], k_new=x[:, heads:heads + hk], v_new=x[:, heads + hk:],
                     k_pages=pages[0], v_pages=pages[1], exponents=exponents, page_table=table, q_start=starts,
                     kv_len=kv_len, cos_sin=cos_sin)
        out.zero_()
        engine.run(q=x[:, :heads], output=out, k_pages=pages[0], v_pages=pages[1], exponents=exponents,
                   page_table=table, q_start=starts, kv_len=kv_len, max_q=q, lse=lse)
        last.copy_(out)

    given.copy_(torch.randn(given.shape, generator=g, device="cuda"))
    step()  # (sets kernel attributes)
    torch.cuda.synchronize()
    kv_len.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(steps):
        given.copy_(torch.randn(given.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        n = (i + 1) * q
        assert engine.error() == 0 and kv_len.tolist() == [n] * batch
        c = Call8([(q, n)] * batch, heads, hk, dim, page)
        c.q, c.output, c.lse = x[:, :heads].clone(), last, lse
        c.k_pages, c.v_pages, c.exponents = pages[0], pages[1], exponents
        at = torch.arange(n, device="cuda")
        for b in range(batch):
            where = table[b].long()[at // page]
            size = 2.0 ** exponents[where, :, 0].double()
            c.keys[b] = pages[0][where, at % page].double() * size[..., 0][..., None]
            c.values[b] = pages[1][where, at % page].double() * size[..., 1][..., None]
        c.check()
