"""Host side of attention over a cache in 8 bits on CPU: refusals of the C ABI
before any CUDA call, and the argument checks of the Python entry point."""
import ctypes as C
import errno

import pytest
import torch

from test_attention_devices import OnGpu, calls, on  # noqa: F401
from test_attention_host import _args


def _exponents(**change):
    from leanstream_b200 import _native as N

    return N.CacheExponents(**{**dict(exponents=1 << 27, page_stride=4, head_stride=2), **change})


@pytest.mark.parametrize("change", [
    dict(k_new=1 << 27, v_new=1 << 27), dict(weights=1 << 27), dict(weights=1 << 27, weights_length=100),
    dict(k_slot_stride=264), dict(v_page_stride=4104), dict(k_head_stride=136), dict(dtype=2), dict(head_dim=96),
    dict(k_pages=(1 << 21) + 8), dict(scratch=None)], ids=str)
def test_refusals(native_lib, change):
    call = native_lib.ls_b200_paged_attention_int8
    assert call(C.byref(_args(**change)), C.byref(_exponents()), None) == errno.EINVAL


@pytest.mark.parametrize("change", [dict(exponents=None), dict(exponents=(1 << 27) + 1), dict(page_stride=3),
                                    dict(head_stride=-2)], ids=str)
def test_refused_exponents(native_lib, change):
    call = native_lib.ls_b200_paged_attention_int8
    assert call(C.byref(_args()), C.byref(_exponents(**change)), None) == errno.EINVAL
    assert call(C.byref(_args()), None, None) == errno.EINVAL
    assert call(None, C.byref(_exponents()), None) == errno.EINVAL


def test_scratch_and_nothing_to_do(native_lib):
    call = native_lib.ls_b200_paged_attention_int8
    need = native_lib.ls_b200_attention_scratch_bytes(C.byref(_args()))
    assert call(C.byref(_args(scratch_bytes=need - 1)), C.byref(_exponents()), None) == errno.ENOSPC
    for change in (dict(batch=0), dict(tokens=0), dict(max_q=0)):
        assert call(C.byref(_args(**change)), C.byref(_exponents()), None) == 0


def engine(**kw):
    from leanstream_b200 import PagedAttention

    return PagedAttention(8, 2, 128, page_size=32, max_sequences=3, max_tokens=12, max_queries=4,
                          scratch=(1 << 28, 1 << 40), **{**dict(cache_dtype="int8"), **kw})


def good(index=0, **change):
    i32, i8 = dict(dtype=torch.int32), dict(dtype=torch.int8)
    return {**dict(q=on(index, 6, 8, 128), output=on(index, 6, 8, 128), k_pages=on(index, 9, 32, 2, 128, **i8),
                   v_pages=on(index, 9, 32, 2, 128, **i8), exponents=on(index, 9, 2, 2, 2, **i8),
                   page_table=on(index, 2, 4, **i32), q_start=on(index, 3, **i32), kv_len=on(index, 2, **i32), max_q=4,
                   lse=on(index, 6, 8, dtype=torch.float32)), **change}


@pytest.fixture
def eight(calls, monkeypatch):  # noqa: F811
    from leanstream_b200 import _native as N

    seen = []
    record = N.load().__class__.ls_b200_evict_cache

    def attend(self, args, exponents, stream):
        seen.append(exponents)
        return record(self, args, stream)

    N.load().__class__.ls_b200_paged_attention_int8 = attend
    return calls


def test_calls_run_on_their_tensors_device(eight):
    for index in (0, 1):
        engine().run(**good(index))
        engine(device=f"cuda:{index}", dtype="float16", cache_dtype=torch.int8).run(stream=7, **good(index))
        assert eight == [(index, 100 + index), (index, 7)]
        eight.clear()
    for name, t in good(0).items():
        if isinstance(t, OnGpu):
            with pytest.raises(ValueError, match=name if name != "q" else None):
                engine().run(**good(0, **{name: on(1, *t.shape, dtype=t.dtype)}))
    assert not eight


def test_arguments_are_checked(eight):
    def of(*shape, dtype=torch.float16):
        return on(0, *shape, dtype=dtype)

    strided = of(9, 2, 2, 4, dtype=torch.int8)[..., :2]
    strided.index = 0
    new = of(6, 2, 128)
    for change in (dict(exponents=None), dict(exponents=of(9, 2, 1, 2, dtype=torch.int8)), dict(exponents=strided),
                   dict(exponents=of(9, 2, 2, 2)), dict(k_pages=of(9, 32, 2, 128), v_pages=of(9, 32, 2, 128)),
                   dict(v_pages=of(9, 32, 2, 128)), dict(k_new=new, v_new=new),
                   dict(weights=of(2, 2, 64, dtype=torch.float32)), dict(max_q=5)):
        with pytest.raises(ValueError):
            engine().run(**good(0, **change))
    sixteen = dict(k_pages=of(9, 32, 2, 128), v_pages=of(9, 32, 2, 128))
    for change in (dict(), sixteen):  # a 16-bit engine takes no exponents
        with pytest.raises(ValueError):
            engine(cache_dtype=None).run(**good(0, **change))
    engine(cache_dtype="float16").run(**good(0, exponents=None, **sixteen))
    for kw in (dict(cache_dtype="bfloat16"), dict(cache_dtype="int4"), dict(max_weights_length=64)):
        with pytest.raises(ValueError):
            engine(**kw)
