"""NativeDecodeSession(kv_cache="int4"): the prefix is held in 4 bits alone and survives its passes."""
import pytest
import torch

from marlin_style_fluxbin_amd.cached_attention import Int4KVCache
from marlin_style_fluxbin_amd.native_decode import NativeDecodeSession
from tests.test_native_decode_cache_gpu import setup

pytestmark = pytest.mark.gpu


def tensors(x, seen):
    """Every tensor that an object holds, its lists' and dicts' ones included."""
    if isinstance(x, torch.Tensor):
        yield x
    elif isinstance(x, (list, tuple)):
        for y in x:
            yield from tensors(y, seen)
    elif isinstance(x, dict):
        for y in x.values():
            yield from tensors(y, seen)
    elif hasattr(x, "__dict__") and not isinstance(x, torch.nn.Module) and id(x) not in seen:
        seen.add(id(x))
        for y in vars(x).values():
            yield from tensors(y, seen)


@pytest.mark.parametrize("kw", [dict(), dict(window=40, sinks=3)])
def test_no_16_bit_prefix_stays(gpu, kw):
    model, ids, forced = setup(gpu, True)
    plain = NativeDecodeSession(model, ids, forced)
    session = NativeDecodeSession(model, ids, forced, kv_cache="int4", **kw)
    length = ids.shape[1]
    for t in tensors(session, set()):  # cos and sin have a row for each position, and no heads
        assert not (t.dtype in (torch.bfloat16, torch.float16, torch.float32) and t.ndim >= 3 and length in t.shape), t.shape
    # what it holds is the prefill's keys and values, before and after passes
    want = []
    for k, v in zip(plain.prefix_k, plain.prefix_v):
        cache = Int4KVCache(1, k.shape[0], length, k.shape[2], device=gpu)
        cache.append(k[None], v[None], 0)
        want.append(cache)
    first = session.audit()
    session.capture()
    for _ in range(2):
        _, again = session.measure("sequence_graph")
        assert torch.equal(again["logits"], first["logits"])
    assert torch.equal(session.audit()["logits"], first["logits"])
    for cache, same in zip(session.int4_cache, want):
        assert all(torch.equal(x[:, :, :length], y) for x, y in zip(cache._parts(), same._parts()))
