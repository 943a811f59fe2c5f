"""Appending to a paged key/value cache, attention over it, and eviction from it,
over the C ABI (ls_b200_append_cache, ls_b200_paged_attention,
ls_b200_evict_cache).

The cache is a pool of pages, `k_pages` and `v_pages` [pages][page_size]
[kv_heads][head_dim]; row b of `page_table` lists the pages of sequence b in
the order of its slots. `PagedAttention` appends the new tokens of every
sequence and attends from them: one token each while decoding, a few drafted
ones, or a chunk of a prompt, mixed as they come. With a `window` the last
`window` slots and the first `sinks` are visible. With `weights` the softmax
weight that each slot received is summed per kv head, and `evict_cache` keeps
the slots of a budget by those sums.

`append_cache` writes new keys and values by itself, with the position rotation
of keys and queries on the way, into 16-bit pages or into a cache of 8-bit
integers with an exponent for each block of 16 slots and kv head.

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
_APPEND = struct.Struct("=14I12Q18qQ")
_EXPONENTS = struct.Struct("=Q2q")
assert _APPEND.size == C.sizeof(N.AppendArgs)
assert _ATTENTION.size == C.sizeof(N.AttentionArgs) and _EVICT.size == C.sizeof(N.EvictArgs)

_INT, _FLOAT, _BYTE = torch.int32, torch.float32, torch.int8
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
    32-bit error word (or None). cache_dtype "int8": the cache is in 8 bits, as
    append_cache fills it (no weights; the call does not append). Its exponents
    then lie in the range of `dtype`, -24 to 9 for float16 and -126 to 120 for
    bfloat16, as they do where it was filled from that type: a visible block
    outside reads as NaN and sets N.ATTN_EXPONENT."""

    def __init__(self, q_heads: int, kv_heads: int, head_dim: int, *, page_size: int, dtype="float16",
                 max_sequences: int, max_tokens: int, max_queries: int = 1, max_weights_length: int = 0, device=None,
                 scratch: Optional[tuple] = None, error: Optional[int] = None, cache_dtype=None):
        self.lib = N.load()
        self.q_heads, self.kv_heads, self.head_dim, self.page_size = q_heads, kv_heads, head_dim, page_size
        self.dtype = _element(dtype)
        self._int8 = cache_dtype in (_BYTE, "int8")
        self.cache_dtype = _BYTE if self._int8 else self.dtype
        if cache_dtype is not None and not self._int8 and _element(cache_dtype) is not self.dtype:
            raise ValueError(f"cache_dtype: {self.dtype} or int8, got {cache_dtype}")
        if self._int8 and max_weights_length:
            raise ValueError("weights are of 16-bit caches")
        self.max_sequences, self.max_tokens = max_sequences, max_tokens
        self.max_queries, self.max_weights_length = max_queries, max_weights_length
        self._code, self._scale = _CODES[self.dtype], head_dim ** -0.5 if head_dim > 0 else 1.0
        self._row, self._page, self._new = (q_heads, head_dim), (page_size, kv_heads, head_dim), (kv_heads, head_dim)
        self._call = self.lib.ls_b200_paged_attention_int8 if self._int8 else self.lib.ls_b200_paged_attention
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
                window, sinks, exponents):
        """Names what is wrong with the arguments of a call."""
        hq, hk, dim, size, e = self.q_heads, self.kv_heads, self.head_dim, self.page_size, self.dtype
        on = q.get_device() if self._device is None else self._device
        _want("q", q, e, (-1, hq, dim), on)
        _want("output", output, e, (q.shape[0], hq, dim), on)
        _want("k_pages", k_pages, self.cache_dtype, (-1, size, hk, dim), on)
        _want("v_pages", v_pages, self.cache_dtype, (k_pages.shape[0], size, hk, dim), on)
        if (exponents is not None) != self._int8:
            raise ValueError("exponents come with a cache in 8 bits")
        if self._int8:
            if k_new is not None or weights is not None:
                raise ValueError("a cache in 8 bits is filled by append_cache, and keeps no weights")
            _want("exponents", exponents, _BYTE, (k_pages.shape[0], hk, size // N.CACHE_BLOCK, 2), on)
            if exponents.stride(2) != 2 and exponents.shape[2] != 1:
                raise ValueError("exponents: contiguous last dimensions expected")
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
            timeout_ns: int = 0, exponents=None) -> None:
        """Enqueues one call on `stream` (a torch stream, a raw cudaStream_t as
        int, or None for torch's current stream) of the tensors' device, which
        is the engine's and need not be the current one. q, output [tokens][q_heads]
        [head_dim]; k_new, v_new [tokens][kv_heads][head_dim], written to their
        slots by the call (without them the cache holds the new tokens
        already); page_table [sequences][columns], q_start [sequences + 1],
        kv_len [sequences] int32 on the device, kv_len with the new tokens;
        max_q: the most new tokens of one sequence. scale: 1 / sqrt(head_dim)
        unless given. lse [tokens][q_heads] and weights [sequences][kv_heads]
        [slots] float32, optional. exponents [pages][kv_heads][page_size / 16][2]
        int8: of a cache in 8 bits."""
        # one pass over the tensors: each attribute of a tensor costs about 0.1 us
        e, rows, pool = self.dtype, q.shape, k_pages.shape
        table, lengths, dev = page_table.shape, kv_len.shape, q.get_device()
        kn = vn = ls = ws = slots = kn0 = kn1 = vn0 = vn1 = ws0 = ws1 = q0 = q1 = o0 = o1 = t0 = 0
        k0 = k1 = k2 = v0 = v1 = v2 = batch = tokens = 0
        good = (len(rows) == 3 and rows[1:] == self._row and len(pool) == 4 and pool[1:] == self._page and
                len(table) == 2 and len(lengths) == 1 and output.shape == rows and v_pages.shape == pool and
                q.dtype is e and output.dtype is e and k_pages.dtype is v_pages.dtype is self.cache_dtype and
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
        if good and exponents is not None:
            good = self._int8 and k_new is None and weights is None and exponents.dtype is _BYTE and \
                exponents.shape == (pool[0], self.kv_heads, self.page_size // 16, 2) and \
                exponents.get_device() == dev
            if good:
                ex0, ex1, a, b = exponents.stride()
                good = (a == 2 or self.page_size == 16) and b == 1 or not pool[0]
        elif good:
            good = not self._int8
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
                         window, sinks, exponents)
        try:
            args = _ATTENTION.pack(
                self._code, self.q_heads, self.kv_heads, self.head_dim, self.page_size, pool[0], batch, tokens, max_q,
                table[1], window, sinks, self._scale if scale is None else scale, slots, q.data_ptr(), kn, vn,
                k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(),
                output.data_ptr(), ls, ws, q0, q1, kn0, kn1, vn0, vn1, k0, k1, k2, v0, v1, v2, o0, o1, t0, ws0, ws1,
                self.scratch_ptr, self.scratch_bytes, self.error_ptr, timeout_ns)
        except (struct.error, OverflowError) as e:
            raise ValueError(f"window {window}, sinks {sinks}, scale {scale}, timeout_ns {timeout_ns}: {e}") from None
        more = (_EXPONENTS.pack(exponents.data_ptr(), ex0, ex1),) if self._int8 else ()
        if stream is None and dev == _current_device():
            rc = self._call(args, *more, _raw_stream(dev))
        else:
            rc = _run_on(dev, self._call, args, *more, _handle(stream, dev))
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


def _refuse_append(k_new, v_new, k_pages, v_pages, page_table, q_start, kv_len, q, q_out, cos_sin, positions,
                   exponents, error):
    e, on = _element(k_new.dtype), kv_len.get_device()
    _want("kv_len", kv_len, _INT, (-1,), on, contiguous=True)
    _want("k_new", k_new, e, (-1, -1, -1), on)
    _want("v_new", v_new, e, tuple(k_new.shape), on)
    tokens, hk, dim = k_new.shape
    cached = e if exponents is None else _BYTE
    _want("k_pages", k_pages, cached, (-1, -1, hk, dim), on)
    _want("v_pages", v_pages, cached, tuple(k_pages.shape), on)
    _want("page_table", page_table, _INT, (kv_len.shape[0], -1), on)
    _want("q_start", q_start, _INT, (kv_len.shape[0] + 1,), on, contiguous=True)
    if exponents is not None:
        _want("exponents", exponents, _BYTE, (k_pages.shape[0], hk, k_pages.shape[1] // N.CACHE_BLOCK, 2), on)
        if exponents.stride(2) != 2 and exponents.shape[2] != 1:
            raise ValueError("exponents: contiguous last dimensions expected")
    if (q is None) != (q_out is None):
        raise ValueError("q and q_out come together")
    if cos_sin is None and (q is not None or positions is not None):
        raise ValueError("q and positions come with cos_sin")
    if q is not None:
        _want("q", q, e, (tokens, -1, dim), on)
        _want("q_out", q_out, e, tuple(q.shape), on)
    if cos_sin is not None:
        _want("cos_sin", cos_sin, _FLOAT, (-1, -1), on)
    if positions is not None:
        _want("positions", positions, _INT, (tokens,), on, contiguous=True)
    if error is not None:
        _want("error", error, _INT, (1,), on)
    raise ValueError("the arguments do not fit together")


def append_cache(*, k_new, v_new, k_pages, v_pages, page_table, q_start, kv_len, q=None, q_out=None, cos_sin=None,
                 positions=None, interleaved: bool = False, exponents=None, error=None, stream=None) -> None:
    """Writes the new tokens' k_new and v_new [tokens][kv_heads][head_dim] to their
    cache slots (page_table, q_start and kv_len as in PagedAttention.run, which is
    then called without k_new and v_new).

    With cos_sin [positions][rotary] float32, the cosines of the rotary / 2 pairs
    and then their sines, the first `rotary` elements of each key, and of q
    [tokens][q_heads][head_dim] into q_out (which may be q), are rotated by the
    angles of the token's position: positions [tokens] int32, or its cache slot.
    Pairs are (i, i + rotary / 2), or neighbours where `interleaved`.

    A cache in 8 bits has int8 pages and `exponents` [pages][kv_heads]
    [page_size / 16][2] int8 (keys', values'): the values are code * 2^exponent.
    A block's exponent is the smallest that reaches its largest value; it grows
    with later tokens, and the block's older codes are rounded to the new step
    then. A block with a value that is not finite reads as NaN (exponent -128).

    error: an optional int32 device tensor, N.ATTN_* bits are ORed in (lengths,
    pages and positions that do not fit: what they would have touched is left as
    it was, in 8 bits the codes, which read with the exponent of their block's
    other new rows). `stream` as in PagedAttention.run."""
    new, pool, table, lengths = k_new.shape, k_pages.shape, page_table.shape, kv_len.shape
    e, cached, dev = k_new.dtype, k_pages.dtype, kv_len.get_device()
    qp = op = hq = q0 = q1 = o0 = o1 = ps = cs = rotary = angles = cs0 = ex = ex0 = ex1 = er = 0
    good = (len(new) == 3 and len(pool) == 4 and len(table) == 2 and len(lengths) == 1 and e in _CODES and
            v_new.shape == new and v_new.dtype is e and v_pages.shape == pool and v_pages.dtype is cached and
            pool[2:] == new[1:] and page_table.dtype is _INT and kv_len.dtype is _INT and q_start.dtype is _INT and
            table[0] == lengths[0] and q_start.shape == (lengths[0] + 1,) and kv_len.is_contiguous() and
            q_start.is_contiguous() and dev >= 0 and k_new.get_device() == v_new.get_device() == dev and
            k_pages.get_device() == v_pages.get_device() == dev and
            page_table.get_device() == q_start.get_device() == dev)
    if good and exponents is None:
        good = cached is e
    elif good:
        good = cached is _BYTE and exponents.dtype is _BYTE and exponents.get_device() == dev and \
            exponents.shape == (pool[0], pool[2], pool[1] // 16, 2)
        if good:
            ex = exponents.data_ptr()
            ex0, ex1, a, b = exponents.stride()
            good = ((a == 2 or pool[1] == 16) and b == 1) or not exponents.numel()
    if good and q is not None:
        wide = q.shape
        good = q_out is not None and len(wide) == 3 and q_out.shape == wide and wide[0] == new[0] and \
            wide[2] == new[2] and q.dtype is e and q_out.dtype is e and q.get_device() == q_out.get_device() == dev \
            and cos_sin is not None
        if good:
            qp, op, hq = q.data_ptr(), q_out.data_ptr(), wide[1]
            q0, q1, a = q.stride()
            o0, o1, b = q_out.stride()
            good = a == b == 1 or not q.numel()
    elif good:
        good = q_out is None
    if good and cos_sin is not None:
        good = cos_sin.dtype is _FLOAT and len(cos_sin.shape) == 2 and cos_sin.get_device() == dev
        if good:
            angles, rotary = cos_sin.shape
            cs = cos_sin.data_ptr()
            cs0, a = cos_sin.stride()
            good = a == 1 or not cos_sin.numel()
    if good and positions is not None:
        ps = positions.data_ptr()
        good = cos_sin is not None and positions.dtype is _INT and positions.shape == new[:1] and \
            positions.is_contiguous() and positions.get_device() == dev
    if good and error is not None:
        er = error.data_ptr()
        good = error.dtype is _INT and error.shape == (1,) and error.get_device() == dev
    if good:
        kn0, kn1, a = k_new.stride()
        vn0, vn1, b = v_new.stride()
        k0, k1, k2, c = k_pages.stride()
        v0, v1, v2, d = v_pages.stride()
        t0, f = page_table.stride()
        good = (a == b == 1 or not new[0]) and (c == d == 1 or not pool[0]) and (f == 1 or not table[1])
    if not good:
        _refuse_append(k_new, v_new, k_pages, v_pages, page_table, q_start, kv_len, q, q_out, cos_sin, positions,
                       exponents, error)
    code = _CODES[e]
    args = _APPEND.pack(code, code if exponents is None else N.INT8, hq, new[1], new[2], pool[1], pool[0], lengths[0],
                        new[0], table[1], rotary, angles, bool(interleaved), 0, qp, op, k_new.data_ptr(),
                        v_new.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), ex, page_table.data_ptr(),
                        q_start.data_ptr(), kv_len.data_ptr(), ps, cs, q0, q1, o0, o1, kn0, kn1, vn0, vn1, k0, k1, k2,
                        v0, v1, v2, ex0, ex1, t0, cs0, er)
    call = N.load().ls_b200_append_cache
    if stream is None and dev == _current_device():
        rc = call(args, _raw_stream(dev))
    else:
        rc = _run_on(dev, call, args, _handle(stream, dev))
    if rc:
        _check(rc, "ls_b200_append_cache")


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
