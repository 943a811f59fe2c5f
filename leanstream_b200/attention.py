"""Attention over a paged key/value cache, and eviction from it, over the C ABI
(ls_b200_paged_attention, ls_b200_evict_cache).

The cache is a pool of pages, `k_pages` and `v_pages` [pages][page_size]
[kv_heads][head_dim]; row b of `page_table` lists the pages of sequence b in
the order of its slots. `PagedAttention` appends the new tokens of every
sequence and attends from them: one token each while decoding, a few drafted
ones, or a chunk of a prompt, mixed as they come. With a `window` the last
`window` slots and the first `sinks` are visible. With `weights` the softmax
weight that each slot received is summed per kv head, and `evict_cache` keeps
the slots of a budget by those sums.

The caller owns every buffer until the stream has run; nothing synchronises.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _native as N
from .backend import _check


def _dtype_code(dtype) -> int:
    name = str(dtype).replace("torch.", "")
    if name not in ("float16", "bfloat16"):
        raise ValueError(f"float16 or bfloat16, got {name}")
    return N.FP16 if name == "float16" else N.BF16


def _handle(stream) -> int:
    if stream is None:
        import torch

        stream = torch.cuda.current_stream()
    return stream if isinstance(stream, int) else stream.cuda_stream


def _want(name, t, dtype, shape):
    """Shape and type of a tensor; -1 in `shape` takes any size."""
    if str(t.dtype) != dtype or t.dim() != len(shape) or any(w not in (-1, s) for w, s in zip(shape, t.shape)):
        raise ValueError(f"{name}: {dtype} {list(shape)} expected, got {t.dtype} {list(t.shape)}")
    if t.numel() and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension has to be contiguous")


class PagedAttention:
    """Attention of new tokens over a paged cache at fixed head sizes. Scratch
    is allocated here, for calls of at most `max_sequences` sequences and
    `max_tokens` new tokens in all, `max_queries` of one sequence, and with
    weights of at most `max_weights_length` slots; calls on one PagedAttention
    must not overlap. `scratch` = (pointer, bytes) supplies caller-owned, zeroed
    device memory instead; `error` is then the device address of a
    caller-owned, zeroed 32-bit error word (or None)."""

    def __init__(self, q_heads: int, kv_heads: int, head_dim: int, *, page_size: int, dtype="float16",
                 max_sequences: int, max_tokens: int, max_queries: int = 1, max_weights_length: int = 0, device=None,
                 scratch: Optional[tuple] = None, error: Optional[int] = None):
        self.lib = N.load()
        self.q_heads, self.kv_heads, self.head_dim, self.page_size = q_heads, kv_heads, head_dim, page_size
        self.dtype = _dtype_code(dtype)
        self.element = "torch.float16" if self.dtype == N.FP16 else "torch.bfloat16"
        self.max_sequences, self.max_tokens = max_sequences, max_tokens
        self.max_queries, self.max_weights_length = max_queries, max_weights_length
        shape = N.AttentionArgs(dtype=self.dtype, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                                page_size=page_size, batch=max_sequences, tokens=max_tokens, max_q=max_queries,
                                weights_length=max_weights_length, scale=1.0)
        self.scratch_bytes = int(self.lib.ls_b200_attention_scratch_bytes(C.byref(shape)))
        if not self.scratch_bytes:
            raise ValueError(f"unsupported shape: {q_heads} query heads, {kv_heads} kv heads of {head_dim}, pages of "
                             f"{page_size} slots")
        self._scratch = self._error = None
        if scratch is not None:
            self.scratch_ptr, have = int(scratch[0]), int(scratch[1])
            if have < self.scratch_bytes:
                raise ValueError(f"scratch of {have} B, {self.scratch_bytes} B needed")
            self.error_ptr = int(error or 0)
        else:
            import torch

            self._scratch = torch.zeros(self.scratch_bytes, dtype=torch.uint8, device=device or "cuda")
            self.scratch_ptr = self._scratch.data_ptr()
            self._error = torch.zeros(1, dtype=torch.int32, device=device or "cuda")
            self.error_ptr = self._error.data_ptr()

    def args(self, *, q, output, k_pages, v_pages, page_table, q_start, kv_len, max_q: int, k_new=None, v_new=None,
             scale: Optional[float] = None, window: int = 0, sinks: int = 0, lse=None, weights=None,
             timeout_ns: int = 0) -> N.AttentionArgs:
        """q, output [tokens][q_heads][head_dim]; k_new, v_new [tokens]
        [kv_heads][head_dim], written to their slots first (without them the
        cache holds the new tokens already); page_table [sequences][columns],
        q_start [sequences + 1], kv_len [sequences] int32 on the device, kv_len
        with the new tokens; max_q: the most new tokens of one sequence. scale:
        1 / sqrt(head_dim) unless given. lse [tokens][q_heads] and weights
        [sequences][kv_heads][slots] float32, optional."""
        tokens, batch = q.shape[0] if q.dim() else 0, kv_len.shape[0] if kv_len.dim() else 0
        hq, hk, dim = self.q_heads, self.kv_heads, self.head_dim
        _want("q", q, self.element, (-1, hq, dim))
        _want("output", output, self.element, (tokens, hq, dim))
        _want("k_pages", k_pages, self.element, (-1, self.page_size, hk, dim))
        _want("v_pages", v_pages, self.element, (k_pages.shape[0], self.page_size, hk, dim))
        _want("kv_len", kv_len, "torch.int32", (-1,))
        _want("page_table", page_table, "torch.int32", (batch, -1))
        _want("q_start", q_start, "torch.int32", (batch + 1,))
        if (k_new is None) != (v_new is None):
            raise ValueError("k_new and v_new come together")
        if k_new is not None:
            _want("k_new", k_new, self.element, (tokens, hk, dim))
            _want("v_new", v_new, self.element, (tokens, hk, dim))
        if lse is not None:
            _want("lse", lse, "torch.float32", (tokens, hq))
            if not lse.is_contiguous():
                raise ValueError("lse has to be contiguous")
        length = 0
        if weights is not None:
            _want("weights", weights, "torch.float32", (batch, hk, -1))
            length = weights.shape[2]
        if batch > self.max_sequences or tokens > self.max_tokens or max_q > self.max_queries or \
                length > self.max_weights_length:
            raise ValueError(f"{batch} sequences, {tokens} tokens, {max_q} of one sequence, weights of {length} slots: "
                             f"sized for {self.max_sequences}, {self.max_tokens}, {self.max_queries}, "
                             f"{self.max_weights_length}")
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks are not negative")
        for name, t in (("q", q), ("output", output), ("k_pages", k_pages), ("v_pages", v_pages),
                        ("page_table", page_table), ("q_start", q_start), ("kv_len", kv_len), ("k_new", k_new),
                        ("v_new", v_new), ("lse", lse), ("weights", weights)):
            if t is not None and not t.is_cuda:
                raise ValueError(f"{name}: a tensor on the GPU is expected")
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        two = lambda t: (t.stride(0), t.stride(1)) if t is not None else (0, 0)  # noqa: E731
        return N.AttentionArgs(
            self.dtype, hq, hk, dim, self.page_size, k_pages.shape[0], batch, tokens, max_q, page_table.shape[1],
            window, sinks, dim ** -0.5 if scale is None else scale, length, ptr(q), ptr(k_new), ptr(v_new),
            ptr(k_pages), ptr(v_pages), ptr(page_table), ptr(q_start), ptr(kv_len), ptr(output), ptr(lse),
            ptr(weights), *two(q), *two(k_new), *two(v_new), *k_pages.stride()[:3], *v_pages.stride()[:3],
            *two(output), page_table.stride(0), *two(weights), self.scratch_ptr, self.scratch_bytes, self.error_ptr,
            int(timeout_ns))

    def run(self, stream=None, **kw) -> None:
        """Enqueues one call on `stream` (a torch stream, a raw cudaStream_t as
        int, or None for torch's current stream). Keyword arguments as `args`."""
        a = self.args(**kw)
        _check(self.lib.ls_b200_paged_attention(C.byref(a), _handle(stream)), "ls_b200_paged_attention")

    def error(self) -> int:
        """The sticky N.ATTN_* bits of the calls so far; reads a device word."""
        if self._error is None:
            raise RuntimeError("the error word is caller-owned (PagedAttention(error=...)): read it there")
        return int(self._error.item())

    def clear_error(self) -> None:
        """Zeroes the owned error word and the scratch (stream-ordered on
        torch's current stream)."""
        if self._error is None:
            raise RuntimeError("the error word is caller-owned (PagedAttention(error=...)): clear it there")
        self._error.zero_()
        self._scratch.zero_()


def evict_cache(*, k_pages, v_pages, page_table, kv_len, weights, budget: int, new_table, new_len, kept,
                sinks: int = 0, recent: int = 0, new_weights=None, error=None, stream=None) -> None:
    """Keeps `budget` slots of each sequence and kv head by their weights
    [sequences][kv_heads][slots]: the first `sinks`, the last `recent`, and the
    heaviest between. The kept rows go, in order, to the pages of `new_table`,
    none of which may be a page of `page_table`; new_len [sequences], kept
    [sequences][kv_heads][budget] (each new slot's old one, -1 past new_len) and
    new_weights (the same shape, float32, optional) are written. error: an
    optional int32 device tensor, N.ATTN_* bits are ORed in."""
    batch, hk = kv_len.shape[0] if kv_len.dim() else 0, k_pages.shape[2] if k_pages.dim() == 4 else 0
    element = str(k_pages.dtype)
    _dtype_code(element)
    _want("k_pages", k_pages, element, (-1, -1, -1, -1))
    _want("v_pages", v_pages, element, tuple(k_pages.shape))
    _want("kv_len", kv_len, "torch.int32", (-1,))
    _want("page_table", page_table, "torch.int32", (batch, -1))
    _want("new_table", new_table, "torch.int32", (batch, -1))
    _want("weights", weights, "torch.float32", (batch, hk, -1))
    _want("new_len", new_len, "torch.int32", (batch,))
    _want("kept", kept, "torch.int32", (batch, hk, budget))
    if new_weights is not None:
        _want("new_weights", new_weights, "torch.float32", (batch, hk, budget))
    if error is not None:
        _want("error", error, "torch.int32", (1,))
    if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"a budget of {budget} slots holds {sinks} first and {recent} last ones?")
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages), ("page_table", page_table), ("new_table", new_table),
                    ("kv_len", kv_len), ("weights", weights), ("new_len", new_len), ("kept", kept),
                    ("new_weights", new_weights), ("error", error)):
        if t is not None and not t.is_cuda:
            raise ValueError(f"{name}: a tensor on the GPU is expected")
    if not kept.is_contiguous() or (new_weights is not None and not new_weights.is_contiguous()):
        raise ValueError("kept and new_weights have to be contiguous")
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    a = N.EvictArgs(hk, k_pages.shape[3], k_pages.shape[1], k_pages.shape[0], batch, page_table.shape[1],
                    new_table.shape[1], weights.shape[2], budget, sinks, recent, 0, ptr(k_pages), ptr(v_pages),
                    ptr(page_table), ptr(new_table), ptr(kv_len), ptr(weights), ptr(new_len), ptr(kept),
                    ptr(new_weights), *k_pages.stride()[:3], *v_pages.stride()[:3], page_table.stride(0),
                    new_table.stride(0), weights.stride(0), weights.stride(1), ptr(error))
    _check(N.load().ls_b200_evict_cache(C.byref(a), _handle(stream)), "ls_b200_evict_cache")
