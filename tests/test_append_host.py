"""Host side of append_cache on CPU: the refusals of the C ABI, which come before
any CUDA call, the argument checks of the Python entry point, and its device."""
import ctypes as C
import errno

import pytest
import torch

from test_attention_devices import OnGpu, calls, on  # noqa: F401


def _args(**change):
    from leanstream_b200 import _native as N

    a = N.AppendArgs(dtype=N.FP16, cache_dtype=N.FP16, q_heads=8, kv_heads=2, head_dim=128, page_size=16, pages=40,
                     batch=3, tokens=12, table_pages=10, rotary_dim=128, angles=200, q=1 << 20, q_out=1 << 21,
                     k_new=1 << 22, v_new=1 << 23, k_pages=1 << 24, v_pages=1 << 25, page_table=1 << 26,
                     q_start=1 << 27, kv_len=1 << 28, cos_sin=1 << 29, q_token_stride=1024, q_head_stride=128,
                     q_out_token_stride=1024, q_out_head_stride=128, k_new_token_stride=256, k_new_head_stride=128,
                     v_new_token_stride=256, v_new_head_stride=128, k_page_stride=4096, k_slot_stride=256,
                     k_head_stride=128, v_page_stride=4096, v_slot_stride=256, v_head_stride=128, table_stride=10,
                     cos_sin_stride=128)
    for k, v in change.items():
        setattr(a, k, v)
    return a


INT8 = dict(cache_dtype=2, exponents=1 << 30, exponents_page_stride=4, exponents_head_stride=2)


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(cache_dtype=1), dict(cache_dtype=3), dict(kv_heads=0), dict(q_heads=0), dict(head_dim=96),
    dict(page_size=8), dict(page_size=24), dict(page_size=512), dict(table_pages=1 << 28), dict(pages=0),
    dict(table_pages=0), dict(tokens=(1 << 27) + 1), dict(rotary_dim=0), dict(rotary_dim=24), dict(rotary_dim=144),
    dict(angles=0), dict(interleaved=2), dict(reserved=1), dict(q=None), dict(q_out=None), dict(q=(1 << 20) + 2),
    dict(k_new=None), dict(v_new=(1 << 23) + 8), dict(k_pages=None), dict(v_pages=(1 << 25) + 8),
    dict(page_table=None), dict(q_start=None), dict(kv_len=None), dict(cos_sin=None), dict(cos_sin=(1 << 29) + 4),
    dict(exponents=1 << 30), dict(cache_dtype=2), dict(q_token_stride=1020), dict(q_out_head_stride=-128),
    dict(k_slot_stride=260), dict(cos_sin_stride=130), dict(table_stride=-1),
    dict(cos_sin=None, rotary_dim=0, angles=0),
    dict(cos_sin=None, rotary_dim=0, angles=0, q=None, q_out=None, q_heads=0, positions=1 << 31),
    {**INT8, "exponents": (1 << 30) + 1}, {**INT8, "exponents_page_stride": 3}, {**INT8, "exponents_head_stride": -2},
    {**INT8, "k_slot_stride": 264}], ids=str)
def test_refusals(native_lib, change):
    assert native_lib.ls_b200_append_cache(C.byref(_args(**change)), None) == errno.EINVAL
    assert native_lib.ls_b200_append_cache(None, None) == errno.EINVAL


def test_nothing_to_do(native_lib):
    for change in (dict(batch=0), dict(tokens=0)):
        assert native_lib.ls_b200_append_cache(C.byref(_args(**change)), None) == 0


def good(index=0, int8=False, make=on, **change):
    i32, f32 = dict(dtype=torch.int32), dict(dtype=torch.float32)
    pages = dict(dtype=torch.int8) if int8 else {}
    got = dict(k_new=make(index, 6, 2, 128), v_new=make(index, 6, 2, 128), k_pages=make(index, 9, 32, 2, 128, **pages),
               v_pages=make(index, 9, 32, 2, 128, **pages), page_table=make(index, 2, 4, **i32),
               q_start=make(index, 3, **i32), kv_len=make(index, 2, **i32), q=make(index, 6, 8, 128),
               q_out=make(index, 6, 8, 128), cos_sin=make(index, 50, 64, **f32), positions=make(index, 6, **i32),
               error=make(index, 1, **i32))
    if int8:
        got["exponents"] = make(index, 9, 2, 2, 2, **pages)
    return {**got, **change}


def test_calls_run_on_their_tensors_device(calls, monkeypatch):  # noqa: F811
    from leanstream_b200 import _native as N, append_cache

    N.load().__class__.ls_b200_append_cache = N.load().__class__.ls_b200_evict_cache
    for index in (0, 1):
        for int8 in (False, True):
            append_cache(**good(index, int8))
            append_cache(stream=7, **good(index, int8))
            append_cache(**good(index, int8, q=None, q_out=None, cos_sin=None, positions=None, error=None))
            assert calls == [(index, 100 + index), (index, 7), (index, 100 + index)]
            calls.clear()
    for int8 in (False, True):
        for name, t in good(0, int8).items():
            with pytest.raises(ValueError, match=name if name != "kv_len" else None):
                append_cache(**good(0, int8, **{name: on(1, *t.shape, dtype=t.dtype)}))
    with pytest.raises(ValueError):
        append_cache(stream=type("Stream", (), dict(cuda_stream=5, device_index=1))(), **good(0))
    assert not calls


def test_tensors_are_checked(calls):  # noqa: F811
    from leanstream_b200 import append_cache

    def of(*shape, dtype=torch.float16):
        return on(0, *shape, dtype=dtype)

    for change in (dict(k_new=of(6, 2, 64)), dict(v_new=of(5, 2, 128)), dict(v_new=of(6, 2, 128, dtype=torch.bfloat16)),
                   dict(k_new=of(6, 2, 128, dtype=torch.float32)), dict(k_pages=of(9, 32, 2, 128, dtype=torch.int8)),
                   dict(v_pages=of(9, 16, 2, 128)), dict(page_table=of(3, 4, dtype=torch.int32)),
                   dict(kv_len=of(2, dtype=torch.int64)), dict(q_start=of(2, dtype=torch.int32)), dict(q=None),
                   dict(q_out=None), dict(q=of(6, 8, 64), q_out=of(6, 8, 64)), dict(q_out=of(6, 4, 128)),
                   dict(cos_sin=None), dict(cos_sin=None, q=None, q_out=None), dict(cos_sin=of(50, 64)),
                   dict(positions=of(5, dtype=torch.int32)), dict(positions=of(6, dtype=torch.int64)),
                   dict(error=of(2, dtype=torch.int32)), dict(exponents=of(9, 2, 2, 2, dtype=torch.int8))):
        with pytest.raises(ValueError):
            append_cache(**good(0, **change))
    for change in (dict(exponents=None), dict(exponents=of(9, 2, 1, 2, dtype=torch.int8)),
                   dict(exponents=of(9, 2, 2, 2)), dict(k_pages=of(9, 32, 2, 128), v_pages=of(9, 32, 2, 128))):
        with pytest.raises(ValueError):
            append_cache(**good(0, True, **change))
    for name, t in good(0, True).items():  # a strided last dimension
        if t.dim() > 1:
            twice = on(0, *t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype)
            twice = twice[..., ::2]
            twice.index = 0
            with pytest.raises(ValueError, match=name):
                append_cache(**good(0, True, **{name: twice}))
    assert not calls


@pytest.mark.parametrize("change", [
    dict(), dict(q=None, q_out=None), dict(q=None, q_out=None, k_new=None, v_new=None, positions=None),
    dict(q=None, q_out=None, k_new=None, v_new=None, cos_sin=None, angles=0),
    {**INT8, "q": None, "q_out": None, "k_new": None, "v_new": None}], ids=str)
def test_no_new_tokens(native_lib, change):
    """Tensors without elements have no address."""
    for empty in (dict(tokens=0), dict(tokens=0, batch=0)):
        assert native_lib.ls_b200_append_cache(C.byref(_args(**{**change, **empty})), None) == 0
    for wrong in (dict(rotary_dim=24), dict(rotary_dim=144), dict(head_dim=96), dict(interleaved=2)):
        assert native_lib.ls_b200_append_cache(C.byref(_args(**{**change, **wrong, "tokens": 0})), None) == errno.EINVAL


def test_no_new_tokens_by_the_entry_point(native_lib, monkeypatch):
    from leanstream_b200 import append_cache, attention

    monkeypatch.setattr(attention, "_current_device", lambda: 0)
    monkeypatch.setattr(attention, "_raw_stream", lambda index: 0)
    i32 = dict(dtype=torch.int32)
    empty = dict(k_new=on(0, 0, 2, 128), v_new=on(0, 0, 2, 128), q=on(0, 0, 8, 128), q_out=on(0, 0, 8, 128),
                 positions=on(0, 0, **i32))
    assert empty["q"].data_ptr() == 0
    for int8 in (False, True):
        append_cache(**good(0, int8, **empty))
        append_cache(**good(0, int8, **{**empty, "q": None, "q_out": None}))
        append_cache(**good(0, int8, **empty, kv_len=on(0, 0, **i32), q_start=on(0, 1, **i32),
                            page_table=on(0, 0, 4, **i32)))
