"""Host side of the paged cache operators on CPU: refusals, which the C ABI
answers before any CUDA call, and the argument checks of the Python entry
points (no compute is launched here)."""
import ctypes as C
import errno

import pytest
import torch


def _args(**change):
    from leanstream_b200 import _native as N

    a = N.AttentionArgs(dtype=N.FP16, q_heads=8, kv_heads=2, head_dim=128, page_size=16, pages=40, batch=3, tokens=12,
                        max_q=4, table_pages=10, scale=0.1, q=1 << 20, k_pages=1 << 21, v_pages=1 << 22,
                        page_table=1 << 23, q_start=1 << 24, kv_len=1 << 25, output=1 << 26, q_token_stride=1024,
                        q_head_stride=128, k_page_stride=4096, k_slot_stride=256, k_head_stride=128,
                        v_page_stride=4096, v_slot_stride=256, v_head_stride=128, output_token_stride=1024,
                        output_head_stride=128, table_stride=10, scratch=1 << 28, scratch_bytes=1 << 40)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(kv_heads=0), dict(q_heads=0), dict(q_heads=7), dict(head_dim=96), dict(head_dim=0),
    dict(page_size=8), dict(page_size=24), dict(page_size=512), dict(table_pages=1 << 28), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=1 << 31), dict(sinks=1 << 31),
    dict(q=None), dict(q=(1 << 20) + 2), dict(output=None), dict(k_pages=None), dict(v_pages=(1 << 22) + 8),
    dict(page_table=None), dict(q_start=None), dict(kv_len=None), dict(scratch=None), dict(pages=0),
    dict(table_pages=0), dict(k_new=1 << 27), dict(v_new=1 << 27), dict(weights=1 << 27), dict(q_token_stride=1020),
    dict(k_slot_stride=-256), dict(output_head_stride=4), dict(timeout_ns=61 * 10 ** 9)], ids=str)
def test_attention_refusals(native_lib, change):
    assert native_lib.ls_b200_paged_attention(C.byref(_args(**change)), None) == errno.EINVAL


def test_attention_scratch(native_lib):
    need = native_lib.ls_b200_attention_scratch_bytes(C.byref(_args()))
    assert need > 0
    assert native_lib.ls_b200_paged_attention(C.byref(_args(scratch_bytes=need - 1)), None) == errno.ENOSPC
    assert native_lib.ls_b200_attention_scratch_bytes(C.byref(_args(head_dim=80))) == 0
    assert native_lib.ls_b200_attention_scratch_bytes(C.byref(_args(weights_length=1000))) > need
    assert native_lib.ls_b200_attention_scratch_bytes(None) == 0
    assert native_lib.ls_b200_paged_attention(None, None) == errno.EINVAL


def test_nothing_to_do(native_lib):
    for change in (dict(batch=0), dict(tokens=0), dict(max_q=0)):
        assert native_lib.ls_b200_paged_attention(C.byref(_args(**change)), None) == 0


@pytest.mark.parametrize("change", [
    dict(kv_heads=0), dict(head_dim=32), dict(page_size=48), dict(budget=0), dict(sinks=5, recent=4), dict(budget=33),
    dict(k_pages=None), dict(v_pages=(1 << 21) + 2), dict(page_table=None), dict(new_table=None), dict(kv_len=None),
    dict(weights=None), dict(kept=None), dict(new_len=None), dict(pages=0), dict(k_page_stride=12)], ids=str)
def test_evict_refusals(native_lib, change):
    from leanstream_b200 import _native as N

    a = N.EvictArgs(kv_heads=2, head_dim=128, page_size=16, pages=40, batch=3, table_pages=10, new_table_pages=2,
                    weights_length=160, budget=8, k_pages=1 << 20, v_pages=1 << 21, page_table=1 << 22,
                    new_table=1 << 23, kv_len=1 << 24, weights=1 << 25, new_len=1 << 26, kept=1 << 27,
                    k_page_stride=4096, k_slot_stride=256, k_head_stride=128, v_page_stride=4096, v_slot_stride=256,
                    v_head_stride=128, table_stride=10, new_table_stride=2)
    for k, v in change.items():
        setattr(a, k, v)
    assert native_lib.ls_b200_evict_cache(C.byref(a), None) == errno.EINVAL
    assert native_lib.ls_b200_evict_cache(None, None) == errno.EINVAL


def _engine(**kw):
    from leanstream_b200 import PagedAttention

    return PagedAttention(**{**dict(q_heads=8, kv_heads=2, head_dim=128, page_size=16, max_sequences=3, max_tokens=12,
                                    max_queries=4, scratch=(1 << 28, 1 << 40)), **kw})


def test_engine_refuses_shapes(native_lib):
    for kw in (dict(head_dim=80), dict(q_heads=9), dict(page_size=20), dict(dtype=torch.float32),
               dict(scratch=(1 << 28, 64))):
        with pytest.raises(ValueError):
            _engine(**kw)
    with pytest.raises(RuntimeError):
        _engine().error()
    with pytest.raises(RuntimeError):
        _engine().clear_error()


def test_engine_refuses_tensors(native_lib):
    half, i32 = dict(dtype=torch.float16), dict(dtype=torch.int32)
    good = dict(q=torch.zeros(6, 8, 128, **half), output=torch.zeros(6, 8, 128, **half),
                k_pages=torch.zeros(9, 16, 2, 128, **half), v_pages=torch.zeros(9, 16, 2, 128, **half),
                page_table=torch.zeros(2, 4, **i32), q_start=torch.zeros(3, **i32), kv_len=torch.zeros(2, **i32),
                max_q=4)
    for change in (dict(q=torch.zeros(6, 8, 128)), dict(q=torch.zeros(6, 4, 128, **half)),
                   dict(output=torch.zeros(5, 8, 128, **half)), dict(k_pages=torch.zeros(9, 32, 2, 128, **half)),
                   dict(v_pages=torch.zeros(8, 16, 2, 128, **half)), dict(q_start=torch.zeros(2, **i32)),
                   dict(kv_len=torch.zeros(2, dtype=torch.int64)), dict(k_new=torch.zeros(6, 2, 128, **half)),
                   dict(lse=torch.zeros(8, 6)), dict(weights=torch.zeros(2, 2, 64)), dict(max_q=5),
                   dict(q=torch.zeros(6, 8, 256, **half)[..., ::2]), dict(window=-1), dict(sinks=-2),
                   dict(page_table=torch.zeros(3, 4, **i32)), {}):  # the last: not on the GPU
        with pytest.raises(ValueError):
            _engine().run(stream=0, **{**good, **change})


def test_evict_refuses_tensors(native_lib):
    from leanstream_b200 import evict_cache

    half, i32 = dict(dtype=torch.float16), dict(dtype=torch.int32)
    good = dict(k_pages=torch.zeros(9, 16, 2, 128, **half), v_pages=torch.zeros(9, 16, 2, 128, **half),
                page_table=torch.zeros(2, 4, **i32), new_table=torch.zeros(2, 1, **i32),
                kv_len=torch.zeros(2, **i32), weights=torch.zeros(2, 2, 64), budget=8,
                new_len=torch.zeros(2, **i32), kept=torch.zeros(2, 2, 8, **i32))
    for change in (dict(weights=torch.zeros(2, 1, 64)), dict(kept=torch.zeros(2, 2, 9, **i32)),
                   dict(budget=0), dict(sinks=5, recent=4), dict(k_pages=torch.zeros(9, 16, 2, 128)),
                   dict(new_weights=torch.zeros(2, 2, 7)), {}):
        with pytest.raises(ValueError):
            evict_cache(stream=0, **{**good, **change})
