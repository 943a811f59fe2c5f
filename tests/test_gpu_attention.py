"""Attention over a paged cache (leanstream_b200/attention.py) on the GPU,
against the formula in 64 bits.

Bounds, per element. Output: the result is rounded once to 16 bits (unit
roundoff u = 2^-11 for float16, 2^-8 for bfloat16), and each probability may
be rounded to 16 bits before it meets its value, which moves the sum by at most
u * A, A = sum p |v|; the logits (up to about 40 here, a 128-term sum in 32
bits times scale * log2 e, one rounding each) and the exponential are good to
1e-5 of a probability, twice with the normalisation: u (|out| + A) + 2e-5 A,
plus float16's smallest step. lse: 2e-5 absolute. Weights: 2e-5 of the summed
probabilities, plus the 32-bit sum's rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}


class Call:
    """Inputs of one call. `lengths` = [(new tokens, slots)]; the pool is
    filled with NaN except for the slots that some row may see."""

    def __init__(self, lengths, heads=8, kv_heads=2, dim=128, page=16, dtype=torch.float16, window=0, sinks=0,
                 weights=False, seed=0, layout="nhd", append=True, q_scale=1.0, extra_pages=3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lengths, self.heads, self.kv_heads, self.dim, self.page = lengths, heads, kv_heads, dim, page
        self.dtype, self.window, self.sinks, self.append = dtype, window, sinks, append
        batch, tokens = len(lengths), sum(q for q, _ in lengths)
        self.max_q = max((q for q, _ in lengths), default=0)
        columns = max([-(-n // page) for _, n in lengths] + [1])
        pages = batch * columns + extra_pages
        shape = {"nhd": (pages, page, kv_heads, dim), "hnd": (pages, kv_heads, page, dim)}[layout]
        view = (lambda t: t) if layout == "nhd" else (lambda t: t.transpose(1, 2))
        self.k_pages = view(torch.full(shape, math.nan, dtype=dtype, device="cuda"))
        self.v_pages = view(torch.full(shape, math.nan, dtype=dtype, device="cuda"))
        order = torch.randperm(pages, generator=g, device="cuda").int()
        self.page_table = order[:batch * columns].reshape(batch, columns).clone()
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        qkv = rand(tokens, heads + 2 * kv_heads, dim).to(dtype)
        qkv[:, :heads] *= q_scale
        self.q, self.k_new, self.v_new = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        self.keys, self.values = [], []  # of each sequence, all slots
        at = 0
        starts = [0]
        for b, (q, n) in enumerate(lengths):
            k, v = rand(n, kv_heads, dim).to(dtype), rand(n, kv_heads, dim).to(dtype)
            fresh = min(q, n)
            if fresh:
                k[n - fresh:] = self.k_new[at + q - fresh:at + q]
                v[n - fresh:] = self.v_new[at + q - fresh:at + q]
            self.keys.append(k)
            self.values.append(v)
            first = n - q
            for i in range(n):  # what no row sees stays NaN in the pool
                seen = not window or i > first - window or i < sinks
                if seen and not (append and i >= first):
                    where = int(self.page_table[b, i // page])
                    self.k_pages[where, i % page] = k[i]
                    self.v_pages[where, i % page] = v[i]
            used = -(-n // page)
            self.page_table[b, used:] = 0x7fffffff if b % 2 else -7  # never to be looked up
            if window and first - window + 1 >= page:  # pages the window left behind
                gone = (first - window + 1) // page
                keep = -(-sinks // page)
                self.page_table[b, keep:gone] = -1
            at += q
            starts.append(at)
        self.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.kv_len = torch.tensor([n for _, n in lengths], dtype=torch.int32, device="cuda")
        self.output = torch.full((tokens, heads, dim), 7.0, dtype=dtype, device="cuda")
        self.lse = torch.full((tokens, heads), 7.0, device="cuda")
        self.weights = torch.rand(batch, kv_heads, columns * page + 5, generator=g, device="cuda") if weights else None
        self.weights_before = self.weights.clone() if weights else None

    def engine(self, **kw):
        from leanstream_b200 import PagedAttention

        return PagedAttention(self.heads, self.kv_heads, self.dim, page_size=self.page, dtype=self.dtype,
                              max_sequences=len(self.lengths), max_tokens=max(1, self.q.shape[0]),
                              max_queries=max(1, self.max_q),
                              max_weights_length=0 if self.weights is None else self.weights.shape[2], **kw)

    def kwargs(self):
        return dict(q=self.q, output=self.output, k_pages=self.k_pages, v_pages=self.v_pages,
                    page_table=self.page_table, q_start=self.q_start, kv_len=self.kv_len, max_q=self.max_q,
                    k_new=self.k_new if self.append else None, v_new=self.v_new if self.append else None,
                    window=self.window, sinks=self.sinks, lse=self.lse, weights=self.weights)

    def expected(self):
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        lse = torch.full(self.lse.shape, -math.inf, dtype=torch.float64, device="cuda")
        weights = None if self.weights is None else self.weights_before.double()
        mass = None if weights is None else torch.zeros_like(weights)
        group, at = self.heads // self.kv_heads, 0
        for b, (q, n) in enumerate(self.lengths):
            slot = torch.arange(n, device="cuda")[None]
            p = torch.arange(n - q, n, device="cuda")[:, None]
            seen = slot <= p
            if self.window:
                seen = seen & ((slot > p - self.window) | (slot < self.sinks))
            if weights is not None:
                weights[b, :, max(0, n - q):n] = 0
            for h in range(self.heads if q and n else 0):
                k, v = self.keys[b][:, h // group].double(), self.values[b][:, h // group].double()
                s = (self.q[at:at + q, h].double() @ k.T) * self.dim ** -0.5
                s = torch.where(seen, s, -math.inf)
                top = s.amax(-1, keepdim=True)
                e = torch.where(seen, torch.exp(s - torch.where(top > -math.inf, top, 0)), 0)
                total = e.sum(-1, keepdim=True)
                pr = torch.where(total > 0, e / total.clamp_min(1e-300), 0)
                out[at:at + q, h] = pr @ v
                bound[at:at + q, h] = pr @ v.abs()
                lse[at:at + q, h] = (top + torch.log(total))[:, 0]
                if weights is not None:
                    weights[b, h // group, :n] += pr.sum(0)
                    mass[b, h // group, :n] += pr.sum(0)
            at += q
        return out, bound, lse, weights, mass

    def check(self):
        out, area, lse, weights, mass = self.expected()
        u = UNIT[self.dtype]
        err = (self.output.double() - out).abs()
        tol = u * (out.abs() + area) + 2e-5 * area + 2.0 ** -24
        assert torch.isfinite(self.output).all()
        assert (err <= tol).all(), f"output off by {(err / tol).max().item():.3g} of its bound"
        empty = torch.isinf(lse)
        assert torch.equal(empty, self.lse == -math.inf)
        assert (self.output[empty] == 0).all()
        if (~empty).any():
            assert (self.lse.double() - lse)[~empty].abs().max().item() <= 2e-5
        if weights is not None:
            err = (self.weights.double() - weights).abs()
            tol = 2e-5 * mass + 2.0 ** -22 * weights.abs() + 1e-30
            assert (err <= tol).all(), f"weights off by {(err / tol).max().item():.3g} of their bound"
        if self.append:
            at = 0
            for b, (q, n) in enumerate(self.lengths):
                for i in range(max(0, n - q), n):
                    page = int(self.page_table[b, i // self.page])
                    assert torch.equal(self.k_pages[page, i % self.page], self.k_new[at + i - (n - q)])
                    assert torch.equal(self.v_pages[page, i % self.page], self.v_new[at + i - (n - q)])
                at += q

    def run(self, **kw):
        engine = self.engine()
        engine.run(**self.kwargs(), **kw)
        torch.cuda.synchronize()
        assert engine.error() == 0
        self.check()


DECODE = [(1, 1)], [(1, 2), (1, 15), (1, 16), (1, 17)], [(1, 63), (1, 64), (1, 65), (1, 1000)], [(1, 0), (0, 9), (1, 33)]
HEADS = [(8, 8, 64), (8, 2, 128), (7, 1, 128), (48, 3, 64), (16, 1, 128), (32, 1, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
def test_one_token_each(cuda_device, native_lib, dtype, heads):
    for i, lengths in enumerate(DECODE):
        Call(lengths, *heads, dtype=dtype, page=16 << i, seed=i, q_scale=2.0).run()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
def test_chunks(cuda_device, native_lib, dtype, heads):
    for i, lengths in enumerate(([(2, 2), (5, 70), (1, 300)], [(33, 33), (0, 5), (64, 200), (1, 129)],
                                 [(150, 421)], [(257, 257), (3, 640)])):
        Call(lengths, *heads, dtype=dtype, page=16 << i, seed=10 + i, q_scale=2.0).run()


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 0), (100, 17), (128, 130), (1000, 4)])
def test_window_and_first_slots(cuda_device, native_lib, window, sinks, weights):
    for i, lengths in enumerate(([(1, 1), (1, 90), (1, 700)], [(5, 5), (9, 400)], [(140, 140), (200, 611), (1, 350)])):
        Call(lengths, 8, 2, 128, page=16, window=window, sinks=sinks, weights=weights, seed=i,
             dtype=torch.bfloat16 if i else torch.float16).run()
        Call(lengths, 6, 2, 64, page=32, window=window, sinks=sinks, weights=weights, seed=i).run()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
def test_weights(cuda_device, native_lib, dtype, heads):
    for i, lengths in enumerate((DECODE[3], [(1, 500), (1, 66)], [(4, 4), (3, 333)], [(130, 260), (40, 40), (0, 7)])):
        Call(lengths, *heads, dtype=dtype, page=16 << i, weights=True, seed=20 + i, q_scale=2.0).run()


@pytest.mark.parametrize("q", [1, 6, 90])
def test_rows_without_slots(cuda_device, native_lib, q):
    """More new tokens than slots: the first rows see nothing."""
    Call([(q, max(0, q - 3)), (q, q // 2), (q, 0), (q, 200)], weights=True, append=False).run()


@pytest.mark.parametrize("lengths", [[(1, 70)], [(40, 200), (1, 3)]])
def test_layouts_and_reuse(cuda_device, native_lib, lengths):
    """Head-major pages, tokens already in the cache, and one engine for several calls in turn."""
    Call(lengths, layout="hnd").run()
    Call(lengths, append=False, dim=64).run()
    first, second = Call(lengths, seed=1), Call(lengths, seed=2)
    engine = first.engine()
    for c in (first, second, first):
        engine.run(**c.kwargs())
    torch.cuda.synchronize()
    first.check()
    second.check()
    again = first.output.clone(), first.lse.clone()
    engine.run(**first.kwargs())
    torch.cuda.synchronize()
    assert torch.equal(again[0], first.output) and torch.equal(again[1], first.lse)


@pytest.mark.parametrize("q", [1, 8, 70])
def test_long_cache_splits(cuda_device, native_lib, q):
    """One sequence over many CTAs, and many short ones."""
    Call([(q, 9000)], page=64, weights=True, q_scale=2.0).run()
    Call([(1 + i % q, 40 + 37 * i) for i in range(40)], page=16, q_scale=2.0).run()


def test_large_logits(cuda_device, native_lib):
    """Maxima that grow along the cache, and probabilities near one."""
    for lengths in ([(1, 600)], [(70, 600)]):
        c = Call(lengths, q_scale=6.0, seed=5)
        ramp = torch.linspace(0.05, 1.0, 600, device="cuda")[:, None, None]
        for b, (q, n) in enumerate(lengths):
            c.keys[b] = (c.keys[b].float() * ramp).to(c.dtype)
            c.keys[b][n - q:] = c.k_new
            for i in range(n - q):
                c.k_pages[int(c.page_table[b, i // 16]), i % 16] = c.keys[b][i]
        c.run()


def test_other_stream(cuda_device, native_lib):
    c = Call([(1, 500), (1, 77)], weights=True)
    engine, stream = c.engine(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        c.q *= 1
        engine.run(**c.kwargs())
        engine.run(stream=stream, **{**c.kwargs(), "weights": None})
    stream.synchronize()
    c.check()


def test_graph_capture(cuda_device, native_lib):
    c = Call([(1, 500), (1, 77)])
    engine = c.engine()
    engine.run(**c.kwargs())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        engine.run(**c.kwargs())
    c.output.zero_()
    graph.replay()
    torch.cuda.synchronize()
    c.check()


@pytest.mark.parametrize("q", [1, 60])
def test_offsets_past_32_bits(cuda_device, native_lib, q):
    """A pool of more than 2^32 elements, read and written at its end."""
    c = Call([(q, 300)], 8, 8, 128, page=64)
    pages = 70000
    k, v = (torch.empty(pages, 64, 8, 128, dtype=c.dtype, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 32
    for old in range(c.k_pages.shape[0]):
        k[pages - 1 - old], v[pages - 1 - old] = c.k_pages[old], c.v_pages[old]
    used = -(-300 // 64)
    c.page_table[:, :used] = pages - 1 - c.page_table[:, :used]
    c.k_pages, c.v_pages = k, v
    c.run()


def test_bad_lengths_and_pages_are_reported(cuda_device, native_lib):
    """What does not fit is skipped and reported; the other sequences are right."""
    from leanstream_b200 import _native as N

    for q in (1, 50):
        c = Call([(q, 200), (q, 150)])
        engine = c.engine()
        c.kv_len[1] = c.page_table.shape[1] * c.page + 1
        engine.run(**c.kwargs())
        torch.cuda.synchronize()
        assert engine.error() == N.ATTN_LENGTH
        engine.clear_error()
        good = Call([(q, 200)])
        assert torch.isfinite(c.output[:q]).all() and (c.output[q:] == 7).all()
        c.kv_len[1] = 150
        c.page_table[1, 2] = c.k_pages.shape[0]
        engine.run(**c.kwargs())
        torch.cuda.synchronize()
        assert engine.error() == N.ATTN_PAGE
        engine.clear_error()
        good.run()
