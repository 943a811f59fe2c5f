"""Scratch of the paged attention: what an engine asks for holds every call
within its limits, whichever kernels the call goes to. The sizes on CPU; one
engine from a prompt's chunk to single tokens on the GPU (bounds of the results
as in test_gpu_attention.py)."""
import ctypes as C
import itertools

import pytest


def scratch(lib, heads, dim, batch, tokens, max_q, slots):
    from leanstream_b200 import _native as N

    return lib.ls_b200_attention_scratch_bytes(C.byref(N.AttentionArgs(
        q_heads=heads[0], kv_heads=heads[1], head_dim=dim, page_size=16, batch=batch, tokens=tokens, max_q=max_q,
        weights_length=slots, scale=1.0)))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [(32, 8), (16, 16), (28, 4), (12, 2), (48, 3), (32, 1), (128, 1)])
def test_covers_every_smaller_call(native_lib, heads, dim):
    sizes = dict(batch=(1, 32), tokens=(1, 4096), max_q=(1, 4, 16, 17, 300), slots=(0, 1, 131072))
    known = {s: scratch(native_lib, heads, dim, *s) for s in itertools.product(*sizes.values())}
    assert all(known.values())
    for large, small in itertools.product(known, known):
        if all(s <= b for s, b in zip(small, large)):
            assert known[small] <= known[large], (large, small)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(32, 2, 64), (16, 4, 64)])
def test_decode_with_weights_on_an_engine_for_chunks(cuda_device, native_lib, heads):
    import torch
    from leanstream_b200 import PagedAttention
    from test_gpu_attention import Call

    wide = 1 << 18
    engine = PagedAttention(*heads, page_size=16, max_sequences=2, max_tokens=512, max_queries=400,
                            max_weights_length=wide)
    most = 16 * heads[1] // heads[0]  # new tokens that the decode kernel takes
    for seed, lengths in enumerate(([(300, 500), (1, 33)], [(1, 501), (1, 34)], [(most, 300), (1, 270)],
                                    [(most + 1, 300), (2, 2)])):
        call = Call(lengths, *heads, page=16, weights=True, seed=seed)
        call.weights = torch.rand(2, heads[1], wide, device="cuda")
        call.weights_before = call.weights.clone()
        engine.run(**call.kwargs())
        torch.cuda.synchronize()
        assert engine.error() == 0
        call.check()
