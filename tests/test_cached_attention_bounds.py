"""The cached attention against 64 bits under bounds that a lost tile, a wrong mask or a lost
rounding would exceed; that they do is asserted here too, on the CPU, by planting each mistake
in the 64-bit result."""
import math

import pytest
import torch

from tests.attention_bounds import Cache, attend, reference_and_bound, visible
from tests.test_cached_attention_gpu import BF, CASES, HF, JOINS, check, int32

SHAPES = CASES | JOINS


def inputs(dtype, b, hk, g, t, length, d, device, seed=0):
    def normal(shape, seed, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        return (torch.randn(shape, generator=g) * scale).to(dtype).to(device)

    q = normal((b, t, hk * g, d), seed).transpose(1, 2)
    return q, normal((b, hk, length, d), seed + 1, 1.5), normal((b, hk, length, d), seed + 2)


def mutants(q, cache, spans, window, sinks, scale):
    """Name -> the 64-bit result with one mistake: nothing at all, 32 neighbouring keys lost,
    the sinks ignored, the window one key wider or narrower."""
    changes = {"zeros": None}
    # the tile: 32 keys in the middle of what the longest sequence's last query sees
    seq = max(range(len(spans)), key=lambda i: spans[i][0] if spans[i][1] else -1)
    n, m = spans[seq]
    seen = visible(n, m, window, sinks, "cpu")[-1].nonzero()[:, 0]
    if len(seen) > 1:
        middle = len(seen) // 2
        lost = seen[max(0, middle - 16):middle + 16]
        lost = lost[lost != n - 1]
        changes["a tile lost"] = lambda see, i: see.index_fill(1, lost, False) if i == seq else see
    for name, w, s in (("no sinks", window, 0), ("window + 1", (window or 0) + 1, sinks), ("window - 1", (window or 0) - 1, sinks)):
        if window and w and any(mm and (visible(nn, mm, w, s, "cpu") != visible(nn, mm, window, sinks, "cpu")).any()
                                for nn, mm in spans):
            changes[name] = lambda see, i, w=w, s=s: visible(*spans[i], w, s, "cpu")
    b, hq, t, d = q.shape
    hk = cache.k.shape[1]
    g = hq // hk
    for name, change in changes.items():
        out = torch.zeros(b, hq, t, d, dtype=torch.float64)
        for i, (n, m) in enumerate(spans):
            if change is None or n == 0 or m == 0:
                continue
            see = change(visible(n, m, window, sinks, "cpu"), i)
            for h in range(hk):
                out[i, h * g:h * g + g, :m] = attend(q[i, h * g:h * g + g, :m], cache.k[i, h, :n], cache.v[i, h, :n],
                                                     see, scale)[0]
        yield name, out


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("case", SHAPES)
def test_the_bounds_see_mistakes(case, bits):
    dtype, b, hk, g, t, length, d, window, sinks, spans = SHAPES[case]
    q, k, v = inputs(dtype, b, hk, g, t, length, d, "cpu")
    cache, scale = Cache(k, v, bits), 1 / math.sqrt(d)
    want, bound = reference_and_bound(q, cache, spans, window, sinks, scale)
    for name, wrong in mutants(q, cache, spans, window, sinks, scale):
        over = ((wrong - want).abs() / bound.clamp_min(1e-300)).amax().item()
        assert over > 2, f"{name}: at most {over:.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("case", SHAPES)
def test_attention_within_the_bounds(gpu, case, bits):
    from marlin_style_fluxbin_amd import Int4KVCache, kv4_attention, window_attention

    dtype, b, hk, g, t, length, d, window, sinks, spans = SHAPES[case]
    q, k, v = inputs(dtype, b, hk, g, t, length, d, gpu)
    want, bound = reference_and_bound(q, Cache(k, v, bits), spans, window, sinks, 1 / math.sqrt(d))
    out = torch.full((b, hk * g, t, d), 7.0, dtype=dtype, device=gpu)
    kw = dict(lengths=int32([n for n, _ in spans]), query_lengths=int32([m for _, m in spans]), window=window,
              sinks=sinks, out=out)
    if bits == 16:
        window_attention(q, k, v, **kw)
    else:
        cache = Int4KVCache(b, hk, length, d)
        cache.append(k, v, 0)
        kv4_attention(q, cache, **kw)
    check(out, want, bound, spans, 7.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits,limit", [(BF, 16, 2.0**-8), (BF, 4, 2.0**-8), (HF, 16, 2.0**-11), (HF, 4, 2.0**-11)])
@pytest.mark.parametrize("t", [1, 8, 150])
def test_error_relative_to_the_output(gpu, dtype, bits, limit, t):
    """Root mean square of the error over that of the output: a rounding of the output is at
    most `limit` of it and 1 / sqrt(3) of that in the mean, p's rounding the same again where p
    has the output's type, a widened cache's three of fp16 (8 times finer than bf16): all
    below sqrt(2 / 3) limit; the scores' part is 2^-11 |terms| of a widened key at most."""
    from marlin_style_fluxbin_amd import Int4KVCache, kv4_attention, window_attention

    b, hk, g, length, d = 2, 2, 4, 1200, 128
    q, k, v = inputs(dtype, b, hk, g, t, length, d, gpu)
    spans = [(length, t)] * b
    want, _ = reference_and_bound(q, Cache(k, v, bits), spans, None, 0, 1 / math.sqrt(d))
    if bits == 16:
        got = window_attention(q, k, v)
    else:
        cache = Int4KVCache(b, hk, length, d)
        cache.append(k, v, 0)
        got = kv4_attention(q, cache)
    error = ((got.double() - want).square().mean() / want.square().mean()).sqrt().item()
    assert error <= limit, error
