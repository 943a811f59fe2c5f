"""The device of the paged cache calls, on CPU: tensors that say they are on some
GPU, and a recorded native call. A call runs with its tensors' device current,
whichever was, and refuses tensors of two devices."""
import contextlib

import pytest
import torch


class OnGpu(torch.Tensor):
    """A CPU tensor that gives `index` as its CUDA device."""
    __torch_function__ = torch._C._disabled_torch_function_impl
    is_cuda = True

    def get_device(self):
        return self.index


def on(index, *shape, dtype=torch.float16):
    t = torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)
    t.index = index
    return t


@pytest.fixture
def calls(native_lib, monkeypatch):
    """(device current in the call, stream handle) of each native call; device 0 is current outside."""
    from leanstream_b200 import _native as N, attention

    current, got = [0], []

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], torch.device("cuda", index).index
        yield
        current[0] = before

    class Library:
        def ls_b200_evict_cache(self, args, stream):
            got.append((current[0], stream))
            return 0

        ls_b200_paged_attention = ls_b200_evict_cache

        def ls_b200_attention_scratch_bytes(self, args):
            return 256

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(attention, "_raw_stream", lambda index: 100 + index)
    if hasattr(attention, "_current_device"):
        monkeypatch.setattr(attention, "_current_device", lambda: current[0])
    monkeypatch.setattr(N, "load", lambda: Library())
    return got


def attend(index, **change):
    i32 = dict(dtype=torch.int32)
    return {**dict(q=on(index, 6, 8, 128), output=on(index, 6, 8, 128), k_pages=on(index, 9, 16, 2, 128),
                   v_pages=on(index, 9, 16, 2, 128), page_table=on(index, 2, 4, **i32), q_start=on(index, 3, **i32),
                   kv_len=on(index, 2, **i32), max_q=4, k_new=on(index, 6, 2, 128), v_new=on(index, 6, 2, 128),
                   lse=on(index, 6, 8, dtype=torch.float32), weights=on(index, 2, 2, 64, dtype=torch.float32)),
            **change}


def cut(index, **change):
    i32 = dict(dtype=torch.int32)
    return {**dict(k_pages=on(index, 9, 16, 2, 128), v_pages=on(index, 9, 16, 2, 128),
                   page_table=on(index, 2, 4, **i32), new_table=on(index, 2, 1, **i32), kv_len=on(index, 2, **i32),
                   weights=on(index, 2, 2, 64, dtype=torch.float32), budget=8, new_len=on(index, 2, **i32),
                   kept=on(index, 2, 2, 8, **i32), new_weights=on(index, 2, 2, 8, dtype=torch.float32),
                   error=on(index, 1, **i32)), **change}


def engine(**kw):
    from leanstream_b200 import PagedAttention

    return PagedAttention(8, 2, 128, page_size=16, max_sequences=3, max_tokens=12, max_queries=4,
                          max_weights_length=64, scratch=(1 << 28, 1 << 40), **kw)


def test_calls_run_on_their_tensors_device(calls):
    from leanstream_b200 import evict_cache

    for index in (0, 1):
        engine().run(**attend(index))
        engine(device=f"cuda:{index}").run(stream=7, **attend(index))
        evict_cache(**cut(index))
        evict_cache(stream=7, **cut(index))
        assert calls == [(index, 100 + index), (index, 7)] * 2
        calls.clear()


def test_two_devices_are_refused(calls):
    from leanstream_b200 import evict_cache

    for name in [k for k, v in attend(0).items() if isinstance(v, OnGpu)]:
        with pytest.raises(ValueError, match=name if name != "q" else None):
            engine().run(**attend(0, **{name: on(1, *attend(0)[name].shape, dtype=attend(0)[name].dtype)}))
    with pytest.raises(ValueError):
        engine(device="cuda:1").run(**attend(0))
    with pytest.raises(ValueError):
        engine(device="cpu")
    for name in [k for k, v in cut(0).items() if isinstance(v, OnGpu)]:
        with pytest.raises(ValueError, match=name if name != "kv_len" else None):
            evict_cache(**cut(0, **{name: on(1, *cut(0)[name].shape, dtype=cut(0)[name].dtype)}))
    stream = type("Stream", (), dict(cuda_stream=5, device_index=1))()
    with pytest.raises(ValueError):
        engine().run(stream=stream, **attend(0))
    with pytest.raises(ValueError):
        evict_cache(stream=stream, **cut(0))
    assert not calls


@pytest.mark.parametrize("change", [dict(window=1 << 32), dict(sinks=1 << 40), dict(timeout_ns=-1),
                                    dict(timeout_ns=1 << 64), dict(scale=1e39)], ids=str)
def test_numbers_that_do_not_fit_are_refused(calls, change):
    with pytest.raises(ValueError):
        engine().run(**attend(0, **change))
    assert not calls
