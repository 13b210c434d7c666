"""window_attention, kv4_attention and Int4KVCache on the GPU against their definitions in 64 bits."""
import math

import pytest
import torch

from marlin_style_fluxbin_amd import Int4KVCache, kv4_attention, window_attention
from tests.attention_reference import bound16, bound4, packed, quantize, reference

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def normal(shape, seed, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def make(dtype, b, hk, g, t, length, d, token_major=False, seed=0):
    q = normal((b, t, hk * g, d), seed, dtype).transpose(1, 2)
    shape = (b, length, hk, d) if token_major else (b, hk, length, d)
    k, v = normal(shape, seed + 1, dtype, 1.5), normal(shape, seed + 2, dtype)
    return (q, k.transpose(1, 2), v.transpose(1, 2)) if token_major else (q, k, v)


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# name: dtype, batch, kv heads, group, tokens, max_len, head_dim, window, sinks, spans (keys, queries)
CASES = {
    # one token
    "decode": (BF, 1, 8, 4, 1, 700, 128, None, 0, [(700, 1)]),
    "decode_first_token": (BF, 2, 2, 4, 1, 64, 128, None, 0, [(1, 1), (2, 1)]),
    "decode_ragged_window": (HF, 3, 2, 7, 1, 1100, 128, 300, 5, [(1100, 1), (33, 1), (301, 1)]),
    "decode_window_1": (BF, 1, 1, 1, 1, 200, 64, 1, 0, [(200, 1)]),
    "decode_window_1_sink": (HF, 1, 1, 16, 1, 200, 64, 1, 1, [(199, 1)]),
    "decode_d256": (BF, 2, 2, 5, 1, 500, 256, None, 0, [(500, 1), (97, 1)]),
    "decode_d256_window": (HF, 1, 1, 8, 1, 900, 256, 130, 40, [(900, 1)]),
    "decode_long": (BF, 1, 1, 4, 1, 9000, 128, None, 0, [(8999, 1)]),
    # several tiles for each wave, the first one cut by the window
    "decode_many_tiles": (BF, 16, 16, 1, 1, 1500, 64, 1100, 3, [(1500 - 37 * i, 1) for i in range(16)]),
    "decode_many_tiles_d128": (HF, 16, 8, 2, 1, 3000, 128, 2011, 0, [(3000 - 91 * i, 1) for i in range(16)]),
    # several tokens in the few-rows kernel
    "verify": (BF, 2, 2, 3, 5, 333, 128, 100, 4, [(333, 5), (97, 3)]),
    "verify_d64": (HF, 2, 2, 1, 16, 130, 64, 33, 2, [(130, 16), (16, 16)]),
    "verify_more_queries_than_keys": (BF, 2, 1, 4, 4, 40, 128, None, 0, [(2, 4), (0, 4)]),
    "verify_groups": (BF, 2, 2, 7, 5, 700, 128, 200, 4, [(700, 5), (150, 3)]),
    # the rows kernel; fp16 over a 4-bit cache: row groups
    "rows_8_groups": (HF, 1, 1, 8, 40, 300, 128, 90, 3, [(299, 40)]),
    "rows_8_groups_d256": (HF, 2, 1, 4, 50, 190, 256, None, 0, [(190, 50), (40, 33)]),
    "rows_17": (BF, 1, 1, 1, 17, 90, 128, None, 0, [(90, 17)]),
    "rows_group_7": (HF, 2, 2, 7, 20, 260, 128, 64, 3, [(260, 20), (131, 13)]),
    "prompt": (BF, 1, 2, 4, 130, 130, 128, None, 0, [(130, 130)]),
    "prompt_window": (HF, 1, 2, 2, 200, 200, 128, 33, 4, [(200, 200)]),
    "prompt_window_1": (BF, 1, 1, 2, 70, 70, 64, 1, 0, [(70, 70)]),
    "prompt_padded": (BF, 3, 1, 4, 65, 65, 128, 20, 70, [(65, 65), (1, 1), (0, 0)]),
    "prompt_d64": (HF, 1, 3, 5, 67, 150, 64, 40, 9, [(149, 67)]),
    "prompt_d256": (BF, 1, 1, 3, 80, 190, 256, None, 0, [(187, 80)]),
    "prompt_d256_window": (HF, 2, 1, 2, 50, 140, 256, 48, 33, [(140, 50), (64, 49)]),
    "chunk_split": (BF, 1, 1, 4, 40, 3000, 128, None, 0, [(2999, 40)]),
    "chunk_split_window": (HF, 2, 1, 4, 9, 2500, 64, 2000, 70, [(2500, 9), (1700, 8)]),
    "rows_more_queries_than_keys": (BF, 2, 1, 2, 30, 40, 128, 8, 2, [(7, 30), (0, 25)]),
}


def spread(case):
    dtype, b, hk, g, t, length, d, window, sinks, spans = CASES[case]
    kw = dict(lengths=int32([n for n, _ in spans]), query_lengths=int32([m for _, m in spans]), window=window,
              sinks=sinks)
    return dtype, b, hk, g, t, length, d, window, sinks, spans, kw


def check(got, want, bound, spans, untouched):
    got = got.double()
    for i, (_, m) in enumerate(spans):
        error = (got[i, :, :m] - want[i, :, :m]).abs()
        assert not torch.isnan(error).any()
        assert (error <= bound[i, :, :m]).all(), f"sequence {i}: {(error / bound[i, :, :m]).max().item():.3g} of the bound"
        assert (got[i, :, m:] == untouched).all(), f"sequence {i}: rows behind its queries changed"


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_window_attention(case, token_major):
    dtype, b, hk, g, t, length, d, window, sinks, spans, kw = spread(case)
    q, k, v = make(dtype, b, hk, g, t, length, d, token_major)
    want, mass, score = reference(q, k, v, spans, window, sinks, 1 / math.sqrt(d))
    bound = bound16(want, mass, score, dtype, length)
    # what no query of a sequence sees is poison
    for i, (n, m) in enumerate(spans):
        k[i, :, n:], v[i, :, n:] = float("nan"), float("inf")
        if window:
            first = max(0, n - m - window + 1)
            k[i, :, min(sinks, first):first], v[i, :, min(sinks, first):first] = float("inf"), float("nan")
    out = torch.full((b, hk * g, t, d), 7.0, dtype=dtype, device="cuda")
    got = window_attention(q, k, v, out=out, **kw)
    assert got is out
    check(got, want, bound, spans, 7.0)


@pytest.mark.parametrize("case", CASES)
def test_kv4_attention(case):
    dtype, b, hk, g, t, length, d, window, sinks, spans, kw = spread(case)
    q, k, v = make(dtype, b, hk, g, t, length, d)
    cache = Int4KVCache(b, hk, length, d)
    cache.append(k, v, 0)
    (_, _, _, kv), (_, _, v_min, vv) = quantize(k), quantize(v)
    kv, vv = kv.cuda(), vv.cuda()
    want, _, score = reference(q, kv, vv, spans, window, sinks, 1 / math.sqrt(d))
    bound = bound4(want, score, dtype, length, vv.abs().max().item(), v_min.double().abs().max().item())
    for i, (n, m) in enumerate(spans):  # poison
        first = max(0, n - m - window + 1) if window else 0
        for a, e in ((n, length), (min(sinks, first), first)):
            for x in (cache.k_scales, cache.v_scales):
                x[i, :, a:e] = float("nan")
            for x in (cache.k_codes, cache.v_codes):
                x[i, :, a:e] = 255
    out = torch.full((b, hk * g, t, d), 7.0, dtype=dtype, device="cuda")
    check(kv4_attention(q, cache, out=out, **kw), want, bound, spans, 7.0)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("b,hk,t,start,counts", [
    (1, 1, 1, 0, None), (2, 3, 37, 5, None), (3, 2, 70, [0, 63, 90], [70, 1, 0]),
    (2, 1, 9, [96, -3], None)])  # past the end, before the beginning: dropped
def test_kv4_append_writes_the_format(dtype, d, b, hk, t, start, counts):
    length = 100
    k, v = normal((b, t, hk, d), 3, dtype, 2.0).transpose(1, 2), normal((b, hk, t, d), 4, dtype)
    k[0, 0, 0, :64] = 0.0                    # a group without range
    v[-1, -1, -1, :64] = -3.5
    if t > 3:
        k[-1, 0, 2, 5], v[0, 0, 1, 63], v[0, -1, 3, 0] = float("nan"), float("inf"), -33000.0
        k[0, 0, 3, 1] = 32768.0              # the largest that a group holds
    cache = Int4KVCache(b, hk, length, d)
    before = [x.fill_(3).clone() for x in cache._parts()]
    starts = [start] * b if isinstance(start, int) else start
    cache.append(k, v, start if isinstance(start, int) else int32(start), counts=None if counts is None else int32(counts))
    for x, codes, scales, was_c, was_s in ((k, cache.k_codes, cache.k_scales, *before[:2]),
                                           (v, cache.v_codes, cache.v_scales, *before[2:])):
        want_codes, scale, minimum, _ = quantize(x)
        want_c, want_s = was_c.cpu(), was_s.cpu()
        for i in range(b):
            for tok in range(t if counts is None else counts[i]):
                pos = starts[i] + tok
                if 0 <= pos < length:
                    want_c[i, :, pos] = packed(want_codes)[i, :, tok]
                    want_s[i, :, pos] = torch.stack((scale, minimum), -1)[i, :, tok]
        live = ~torch.isnan(want_s.float()).any(-1)  # a NaN group's codes stand for nothing
        assert torch.equal(torch.nan_to_num(scales.cpu(), 9.0), torch.nan_to_num(want_s, 9.0))
        keep = live[..., None, :, None].expand(*live.shape[:3], 16, d // 64, 2).reshape(want_c.shape)
        assert torch.equal(codes.cpu()[keep], want_c[keep])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,b,hk,length,rows", [(64, 2, 3, 77, 77), (128, 1, 2, 300, 131), (256, 2, 1, 33, 1),
                                                (128, 1, 1, 5, 0)])
def test_kv4_restore(dtype, d, b, hk, length, rows):
    k, v = normal((b, hk, length, d), 5, BF, 3.0), normal((b, hk, length, d), 6, BF)
    cache = Int4KVCache(b, hk, length, d)
    cache.append(k, v, 0)
    for got, x in zip(cache.restore(length=rows, dtype=dtype), (k, v)):
        assert got.shape == (b, hk, rows, d)
        # code * scale + minimum is one fp32 rounding (exact products), then one to dtype
        want = quantize(x)[3][:, :, :rows].float().to(dtype)
        assert torch.equal(got.cpu(), want)


def test_new_cache_stands_for_zeros():
    cache = Int4KVCache(1, 2, 50, 128)
    assert cache.nbytes == 2 * 2 * 50 * (64 + 8)
    for x in cache.restore(dtype=HF):
        assert (x == 0).all()
