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
import struct
from typing import Optional

import torch

from . import _native as N
from .backend import _check

# The argument structures as one pack each: a call a decode step is worth the
# few microseconds that filling ctypes fields one by one would take.
_ATTENTION = struct.Struct("=12IfI11Q17qQQQQ")
_EVICT = struct.Struct("=12I9Q10qQ")
assert _ATTENTION.size == C.sizeof(N.AttentionArgs) and _EVICT.size == C.sizeof(N.EvictArgs)

_INT, _FLOAT = torch.int32, torch.float32
_CODES = {torch.float16: N.FP16, torch.bfloat16: N.BF16}


def _element(dtype) -> torch.dtype:
    got = dtype if isinstance(dtype, torch.dtype) else getattr(torch, str(dtype), None)
    if got not in _CODES:
        raise ValueError(f"float16 or bfloat16, got {dtype}")
    return got


# torch's current stream as an integer, without the stream object around it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _handle(stream, device: int) -> int:
    if stream is None:
        return _raw_stream(device)
    if isinstance(stream, int):
        return stream
    if stream.device_index != device:
        raise ValueError(f"stream: on cuda:{stream.device_index}, the tensors are on cuda:{device}")
    return stream.cuda_stream


def _run_on(device: int, call, *args):
    """`call` with `device` current: a launch goes to the current device, and
    every device's default stream has the same handle."""
    if device == _current_device():
        return call(*args)
    with torch.cuda.device(device):
        return call(*args)


def _want(name, t, dtype, shape, device: int, contiguous=False):
    """Refuses a tensor of another type or shape (-1 in `shape` takes any
    size), with a strided last dimension, or that is not on the GPU `device`."""
    if t.dtype is not dtype or t.dim() != len(shape) or any(w not in (-1, s) for w, s in zip(shape, t.shape)):
        raise ValueError(f"{name}: {dtype} {list(shape)} expected, got {t.dtype} {list(t.shape)}")
    if t.numel() and (t.stride(-1) != 1 or (contiguous and not t.is_contiguous())):
        raise ValueError(f"{name}: {'a contiguous tensor' if contiguous else 'a contiguous last dimension'} expected")
    if t.get_device() != device or device < 0:
        where = t.get_device()
        raise ValueError(f"{name}: a tensor on {f'cuda:{device}' if device >= 0 else 'the GPU'} is expected, got one "
                         f"on {f'cuda:{where}' if where >= 0 else t.device}")


class PagedAttention:
    """Attention of new tokens over a paged cache at fixed head sizes. Scratch
    is allocated here, for calls of at most `max_sequences` sequences and
    `max_tokens` new tokens in all, `max_queries` of one sequence, and with
    weights of at most `max_weights_length` slots (those cost scratch:
    max_sequences * q_heads * max_weights_length * 4 B for each of up to 16 /
    group new tokens of a sequence); calls on one PagedAttention must not
    overlap. `scratch` = (pointer, bytes) supplies caller-owned, zeroed device
    memory instead; `error` is then the device address of a caller-owned, zeroed
    32-bit error word (or None)."""

    def __init__(self, q_heads: int, kv_heads: int, head_dim: int, *, page_size: int, dtype="float16",
                 max_sequences: int, max_tokens: int, max_queries: int = 1, max_weights_length: int = 0, device=None,
                 scratch: Optional[tuple] = None, error: Optional[int] = None):
        self.lib = N.load()
        self.q_heads, self.kv_heads, self.head_dim, self.page_size = q_heads, kv_heads, head_dim, page_size
        self.dtype = _element(dtype)
        self.max_sequences, self.max_tokens = max_sequences, max_tokens
        self.max_queries, self.max_weights_length = max_queries, max_weights_length
        self._code, self._scale = _CODES[self.dtype], head_dim ** -0.5 if head_dim > 0 else 1.0
        self._row, self._page, self._new = (q_heads, head_dim), (page_size, kv_heads, head_dim), (kv_heads, head_dim)
        self._call = self.lib.ls_b200_paged_attention
        shape = N.AttentionArgs(dtype=self._code, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                                page_size=page_size, batch=max_sequences, tokens=max_tokens, max_q=max_queries,
                                weights_length=max_weights_length, scale=1.0)
        self._device = None  # of the scratch, where that is known
        if device is not None:
            if torch.device(device).type != "cuda":
                raise ValueError(f"a GPU expected, got device {device}")
            self._device = torch.device(device).index
            if self._device is None:
                self._device = _current_device()
        size = self.lib.ls_b200_attention_scratch_bytes
        self.scratch_bytes = int(size(C.byref(shape)) if self._device is None else
                                 _run_on(self._device, size, C.byref(shape)))
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
            where = "cuda" if device is None else device
            self._scratch = torch.zeros(self.scratch_bytes, dtype=torch.uint8, device=where)
            self._device = self._scratch.get_device()
            self.scratch_ptr = self._scratch.data_ptr()
            self._error = torch.zeros(1, dtype=torch.int32, device=where)
            self.error_ptr = self._error.data_ptr()

    def _refuse(self, q, output, k_pages, v_pages, page_table, q_start, kv_len, max_q, k_new, v_new, lse, weights,
                window, sinks):
        """Names what is wrong with the arguments of a call."""
        hq, hk, dim, size, e = self.q_heads, self.kv_heads, self.head_dim, self.page_size, self.dtype
        on = q.get_device() if self._device is None else self._device
        _want("q", q, e, (-1, hq, dim), on)
        _want("output", output, e, (q.shape[0], hq, dim), on)
        _want("k_pages", k_pages, e, (-1, size, hk, dim), on)
        _want("v_pages", v_pages, e, (k_pages.shape[0], size, hk, dim), on)
        _want("kv_len", kv_len, _INT, (-1,), on)
        _want("page_table", page_table, _INT, (kv_len.shape[0], -1), on)
        _want("q_start", q_start, _INT, (kv_len.shape[0] + 1,), on)
        if (k_new is None) != (v_new is None):
            raise ValueError("k_new and v_new come together")
        if k_new is not None:
            _want("k_new", k_new, e, (q.shape[0], hk, dim), on)
            _want("v_new", v_new, e, (q.shape[0], hk, dim), on)
        if lse is not None:
            _want("lse", lse, _FLOAT, (q.shape[0], hq), on, contiguous=True)
        if weights is not None:
            _want("weights", weights, _FLOAT, (kv_len.shape[0], hk, -1), on)
        raise ValueError(f"{kv_len.shape[0]} sequences, {q.shape[0]} tokens, {max_q} of one sequence, weights of "
                         f"{0 if weights is None else weights.shape[2]} slots, window {window}, {sinks} first slots: "
                         f"sized for {self.max_sequences}, {self.max_tokens}, {self.max_queries}, "
                         f"{self.max_weights_length}, and none is negative")

    def run(self, stream=None, *, q, output, k_pages, v_pages, page_table, q_start, kv_len, max_q: int, k_new=None,
            v_new=None, scale: Optional[float] = None, window: int = 0, sinks: int = 0, lse=None, weights=None,
            timeout_ns: int = 0) -> None:
        """Enqueues one call on `stream` (a torch stream, a raw cudaStream_t as
        int, or None for torch's current stream) of the tensors' device, which
        is the engine's and need not be the current one. q, output [tokens][q_heads]
        [head_dim]; k_new, v_new [tokens][kv_heads][head_dim], written to their
        slots by the call (without them the cache holds the new tokens
        already); page_table [sequences][columns], q_start [sequences + 1],
        kv_len [sequences] int32 on the device, kv_len with the new tokens;
        max_q: the most new tokens of one sequence. scale: 1 / sqrt(head_dim)
        unless given. lse [tokens][q_heads] and weights [sequences][kv_heads]
        [slots] float32, optional."""
        # one pass over the tensors: each attribute of a tensor costs about 0.1 us
        e, rows, pool = self.dtype, q.shape, k_pages.shape
        table, lengths, dev = page_table.shape, kv_len.shape, q.get_device()
        kn = vn = ls = ws = slots = kn0 = kn1 = vn0 = vn1 = ws0 = ws1 = q0 = q1 = o0 = o1 = t0 = 0
        k0 = k1 = k2 = v0 = v1 = v2 = batch = tokens = 0
        good = (len(rows) == 3 and rows[1:] == self._row and len(pool) == 4 and pool[1:] == self._page and
                len(table) == 2 and len(lengths) == 1 and output.shape == rows and v_pages.shape == pool and
                q.dtype is e and output.dtype is e and k_pages.dtype is e and v_pages.dtype is e and
                page_table.dtype is _INT and kv_len.dtype is _INT and q_start.dtype is _INT and
                dev >= 0 and (self._device is None or self._device == dev) and dev == output.get_device() and
                dev == k_pages.get_device() and dev == v_pages.get_device() and dev == page_table.get_device() and
                dev == kv_len.get_device() and dev == q_start.get_device() and window >= 0 and sinks >= 0 and
                0 <= max_q <= self.max_queries)
        if good:
            tokens, batch = rows[0], lengths[0]
            q0, q1, a = q.stride()
            o0, o1, b = output.stride()
            k0, k1, k2, c = k_pages.stride()
            v0, v1, v2, d = v_pages.stride()
            t0, f = page_table.stride()
            good = (table[0] == batch <= self.max_sequences and tokens <= self.max_tokens and
                    (a == b == 1 or not tokens) and (c == d == 1 or not pool[0]) and (f == 1 or not table[1]) and
                    q_start.shape == (batch + 1,) and kv_len.is_contiguous() and q_start.is_contiguous() and
                    (k_new is None) == (v_new is None))
        if good and k_new is not None:
            kn, vn = k_new.data_ptr(), v_new.data_ptr()
            kn0, kn1, a = k_new.stride()
            vn0, vn1, b = v_new.stride()
            good = (k_new.shape == v_new.shape == (tokens, *self._new) and k_new.dtype is e and v_new.dtype is e and
                    k_new.get_device() == v_new.get_device() == dev and (a == b == 1 or not tokens))
        if good and lse is not None:
            ls = lse.data_ptr()
            good = lse.shape == rows[:2] and lse.dtype is _FLOAT and lse.is_contiguous() and \
                lse.get_device() == dev
        if good and weights is not None:
            ws, wide = weights.data_ptr(), weights.shape
            good = weights.dtype is _FLOAT and wide[:2] == (batch, self.kv_heads) and len(wide) == 3 and \
                wide[2] <= self.max_weights_length and weights.get_device() == dev
            if good:
                slots = wide[2]
                ws0, ws1, a = weights.stride()
                good = a == 1 or not weights.numel()
        if not good:
            self._refuse(q, output, k_pages, v_pages, page_table, q_start, kv_len, max_q, k_new, v_new, lse, weights,
                         window, sinks)
        try:
            args = _ATTENTION.pack(
                self._code, self.q_heads, self.kv_heads, self.head_dim, self.page_size, pool[0], batch, tokens, max_q,
                table[1], window, sinks, self._scale if scale is None else scale, slots, q.data_ptr(), kn, vn,
                k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(),
                output.data_ptr(), ls, ws, q0, q1, kn0, kn1, vn0, vn1, k0, k1, k2, v0, v1, v2, o0, o1, t0, ws0, ws1,
                self.scratch_ptr, self.scratch_bytes, self.error_ptr, timeout_ns)
        except (struct.error, OverflowError) as e:
            raise ValueError(f"window {window}, sinks {sinks}, scale {scale}, timeout_ns {timeout_ns}: {e}") from None
        if stream is None and dev == _current_device():
            rc = self._call(args, _raw_stream(dev))
        else:
            rc = _run_on(dev, self._call, args, _handle(stream, dev))
        if rc:
            _check(rc, "ls_b200_paged_attention")

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


def _refuse_evict(k_pages, v_pages, page_table, kv_len, weights, budget, new_table, new_len, kept, sinks, recent,
                  new_weights, error):
    e, on = _element(k_pages.dtype), kv_len.get_device()
    _want("k_pages", k_pages, e, (-1, -1, -1, -1), on)
    _want("v_pages", v_pages, e, tuple(k_pages.shape), on)
    _want("kv_len", kv_len, _INT, (-1,), on)
    batch, hk = kv_len.shape[0], k_pages.shape[2]
    _want("page_table", page_table, _INT, (batch, -1), on)
    _want("new_table", new_table, _INT, (batch, -1), on)
    _want("weights", weights, _FLOAT, (batch, hk, -1), on)
    _want("new_len", new_len, _INT, (batch,), on, contiguous=True)
    _want("kept", kept, _INT, (batch, hk, budget), on, contiguous=True)
    if new_weights is not None:
        _want("new_weights", new_weights, _FLOAT, (batch, hk, budget), on, contiguous=True)
    if error is not None:
        _want("error", error, _INT, (1,), on)
    raise ValueError(f"a budget of {budget} slots does not hold {sinks} first and {recent} last ones")


def evict_cache(*, k_pages, v_pages, page_table, kv_len, weights, budget: int, new_table, new_len, kept,
                sinks: int = 0, recent: int = 0, new_weights=None, error=None, stream=None) -> None:
    """Keeps `budget` slots of each sequence and kv head by their weights
    [sequences][kv_heads][slots]: the first `sinks`, the last `recent`, and the
    heaviest between. The kept rows go, in order, to the pages of `new_table`,
    none of which may be a page of `page_table`; new_len [sequences], kept
    [sequences][kv_heads][budget] (each new slot's old one, -1 past new_len) and
    new_weights (the same shape, float32, optional) are written. error: an
    optional int32 device tensor, N.ATTN_* bits are ORed in. `stream` as in
    PagedAttention.run."""
    pool, table, new, wide = k_pages.shape, page_table.shape, new_table.shape, weights.shape
    lengths = kv_len.shape
    batch, dev = lengths[0] if lengths else 0, kv_len.get_device()
    good = (len(pool) == 4 and len(table) == len(new) == 2 and len(wide) == 3 and k_pages.dtype in _CODES and
            v_pages.dtype is k_pages.dtype and v_pages.shape == pool and len(lengths) == 1 and
            kv_len.dtype is _INT and page_table.dtype is _INT and new_table.dtype is _INT and
            weights.dtype is _FLOAT and new_len.dtype is _INT and kept.dtype is _INT and table[0] == batch and
            new[0] == batch and wide[0] == batch and wide[1] == pool[2] and new_len.shape == (batch,) and
            kept.shape == (batch, pool[2], budget) and budget >= 1 and sinks >= 0 and recent >= 0 and
            sinks + recent <= budget and dev >= 0 and k_pages.get_device() == v_pages.get_device() == dev and
            page_table.get_device() == new_table.get_device() == dev and weights.get_device() == dev and
            new_len.get_device() == kept.get_device() == dev and kept.is_contiguous() and
            new_len.is_contiguous() and kv_len.is_contiguous())
    nw = er = 0
    if good and new_weights is not None:
        nw = new_weights.data_ptr()
        good = new_weights.dtype is _FLOAT and new_weights.shape == kept.shape and new_weights.is_contiguous() and \
            new_weights.get_device() == dev
    if good and error is not None:
        er = error.data_ptr()
        good = error.dtype is _INT and error.shape == (1,) and error.get_device() == dev
    if good:
        k0, k1, k2, a = k_pages.stride()
        v0, v1, v2, b = v_pages.stride()
        t0, c = page_table.stride()
        n0, d = new_table.stride()
        w0, w1, f = weights.stride()
        good = (a == b == 1 or not k_pages.numel()) and (c == 1 or not page_table.numel()) and \
            (d == 1 or not new_table.numel()) and (f == 1 or not weights.numel())
    if not good:
        _refuse_evict(k_pages, v_pages, page_table, kv_len, weights, budget, new_table, new_len, kept, sinks, recent,
                      new_weights, error)
    args = _EVICT.pack(pool[2], pool[3], pool[1], pool[0], batch, table[1], new[1], wide[2], budget, sinks, recent, 0,
                       k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), new_table.data_ptr(),
                       kv_len.data_ptr(), weights.data_ptr(), new_len.data_ptr(), kept.data_ptr(), nw, k0, k1, k2, v0,
                       v1, v2, t0, n0, w0, w1, er)
    rc = _run_on(dev, N.load().ls_b200_evict_cache, args, _handle(stream, dev))
    if rc:
        _check(rc, "ls_b200_evict_cache")
