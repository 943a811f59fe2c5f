"""Exponents of pages of 16 slots: their dimension of one block may have any stride (as
tensors from other libraries do), on CPU."""
import pytest
import torch

from test_append_host import good as append_args
from test_attention_devices import OnGpu, calls, on  # noqa: F401
from test_attention_int8_host import eight, good as attend_args  # noqa: F401


def exponents(stride, blocks=1):
    t = torch.zeros(200, dtype=torch.int8).as_strided((9, 2, blocks, 2), (8, 4, stride, 1)).as_subclass(OnGpu)
    t.index = 0
    return t


def pools(page):
    return {name: on(0, 9, page, 2, 128, dtype=torch.int8) for name in ("k_pages", "v_pages")}


def test_one_block(eight):  # noqa: F811
    from leanstream_b200 import PagedAttention, _native as N, append_cache

    N.load().__class__.ls_b200_append_cache = N.load().__class__.ls_b200_evict_cache
    engine = PagedAttention(8, 2, 128, page_size=16, max_sequences=3, max_tokens=12, max_queries=4,
                            scratch=(1 << 28, 1 << 40), cache_dtype="int8")
    for stride in (1, 2, 7):
        engine.run(**attend_args(0, **pools(16), exponents=exponents(stride)))
        append_cache(**append_args(0, True, **pools(16), exponents=exponents(stride)))
    assert len(eight) == 6
    engine = PagedAttention(8, 2, 128, page_size=32, max_sequences=3, max_tokens=12, max_queries=4,
                            scratch=(1 << 28, 1 << 40), cache_dtype="int8")
    for stride in (1, 4):
        with pytest.raises(ValueError, match="exponents"):
            engine.run(**attend_args(0, exponents=exponents(stride, 2)))
        with pytest.raises(ValueError, match="exponents"):
            append_cache(**append_args(0, True, exponents=exponents(stride, 2)))
