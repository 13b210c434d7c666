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


# ------------------------------------------------------------------ what a row does not see
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", [5, 150])  # the few-rows and the rows kernel
def test_infinities_stay_with_the_rows_that_see_them(dtype, d, t):
    """One key's value holds +inf, another's -inf, a third's NaN, a fourth key is NaN: rows in
    front of them are as if they were not there, rows that see a value's infinity have it."""
    n, window, sinks = t + 60, 40, 2
    q, k, v = make(dtype, 1, 1, 2, t, n, d)
    spans = [(n, t)]
    clean, mass, score = reference(q, k, v, spans, window, sinks, 1 / math.sqrt(d))
    bound = bound16(clean, mass, score, dtype, n)
    first = n - t
    plus, minus, nan, key = first + 1, first + 2, first + 3, first + 4
    v[0, 0, plus, 3], v[0, 0, minus, 3], v[0, 0, minus, 7], v[0, 0, nan, 9] = (
        float("inf"), float("-inf"), float("-inf"), float("nan"))
    k[0, 0, key, 11] = float("nan")
    got = window_attention(q, k, v, window=window, sinks=sinks).double()
    p = torch.arange(first, n, device="cuda")

    def seen(j):
        return ((j <= p) & (j > p - window))[None, :].expand(2, -1)

    want = clean[0].clone()
    inf = float("inf")
    want[..., 3] = torch.where(seen(plus), inf, want[..., 3])
    want[..., 3] = torch.where(seen(minus), want[..., 3] - inf, want[..., 3])  # both: NaN
    want[..., 7] = torch.where(seen(minus), -inf, want[..., 7])
    want[..., 9] = torch.where(seen(nan), float("nan"), want[..., 9])
    want[seen(key)] = float("nan")
    plain = torch.isfinite(want)
    assert torch.equal(torch.isnan(got[0]), torch.isnan(want))
    assert torch.equal(got[0][torch.isinf(want)], want[torch.isinf(want)])
    assert ((got[0] - want).abs()[plain] <= bound[0][plain]).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t", [4, 90])
def test_kv4_nan_groups_stay_with_the_rows_that_see_them(dtype, t):
    n, d = t + 40, 128
    q, k, v = make(dtype, 1, 1, 2, t, n, d)
    cache = Int4KVCache(1, 1, n, d)
    cache.append(k, v, 0)
    kv, (_, _, v_min, vv) = quantize(k)[3].cuda(), quantize(v)
    want, _, score = reference(q, kv, vv.cuda(), [(n, t)], None, 0, 1 / math.sqrt(d))
    bound = bound4(want, score, dtype, n, vv.abs().max().item(), v_min.double().abs().max().item())
    at = n - t + 2
    v[0, 0, at, 70] = float("inf")  # columns 64 .. 127 of that position stand for NaN
    cache.append(k, v, 0)
    got = kv4_attention(q, cache).double()
    see = torch.arange(t, device="cuda") >= 2
    assert torch.isnan(got[:, :, see, 64:]).all()
    got[:, :, see, 64:] = want[:, :, see, 64:]
    assert ((got - want).abs() <= bound).all()


def test_a_row_of_minus_infinity_has_no_softmax():
    """Every visible score -inf: NaN, as the formula; a row that sees no key: zeros."""
    q, k, v = make(BF, 1, 1, 1, 2, 8, 64)
    q.fill_(1.0)
    k.fill_(float("-inf"))
    got = window_attention(q, k, v, lengths=int32([1]))
    assert (got[0, 0, 0] == 0).all() and torch.isnan(got[0, 0, 1]).all()


# ------------------------------------------------------------------ how calls are made
def test_lengths_are_clamped():
    q, k, v = make(BF, 3, 2, 2, 6, 50, 64)
    whole = window_attention(q, k, v, window=9)
    out = torch.full_like(whole, 5.0)
    window_attention(q, k, v, window=9, lengths=int32([1000, -4, 50]), query_lengths=int32([99, 6, -1]), out=out)
    assert torch.equal(out[0], whole[0])
    assert (out[1] == 0).all()
    assert (out[2] == 5).all()


def test_new_output_has_zeros_behind_the_queries():
    q, k, v = make(HF, 2, 1, 2, 7, 30, 128)
    got = window_attention(q, k, v, query_lengths=int32([7, 3]))
    assert (got[1, :, 3:] == 0).all() and (got[1, :, :3] != 0).any()


@pytest.mark.parametrize("layout", ["odd_start", "odd_stride", "column_step", "expanded", "negated"])
def test_layouts(layout):
    b, hk, g, t, n, d = 2, 2, 3, 20, 70, 64
    q, k, v = make(HF, b, hk, g, t, n, d)
    want = window_attention(q, k, v, window=30, sinks=3)

    def odd(x):
        if layout == "odd_start":
            base = torch.empty(x.numel() + 3, dtype=x.dtype, device="cuda")
            return base[3:].view(x.shape).copy_(x)
        if layout == "odd_stride":
            base = torch.empty(*x.shape[:-1], d + 5, dtype=x.dtype, device="cuda")
            return base[..., :d].copy_(x)
        base = torch.empty(*x.shape[:-1], 2 * d, dtype=x.dtype, device="cuda")
        return base[..., ::2].copy_(x)

    if layout == "expanded":  # one sequence's cache for the whole batch
        k1, v1 = (x[:1].expand(b, -1, -1, -1) for x in (k, v))
        want = window_attention(q, k1.contiguous(), v1.contiguous(), window=30, sinks=3)
        assert torch.equal(window_attention(q, k1, v1, window=30, sinks=3), want)
        return
    if layout == "negated":
        lazy = torch.complex(torch.zeros_like(q).contiguous(), -q.contiguous()).conj().imag
        assert lazy.is_neg() and torch.equal(window_attention(lazy, k, v, window=30, sinks=3), want)
        return
    assert torch.equal(window_attention(odd(q), odd(k), odd(v), window=30, sinks=3), want)
    cache, same = Int4KVCache(b, hk, n, d), Int4KVCache(b, hk, n, d)
    cache.append(k, v, 0)
    same.append(odd(k), odd(v), 0)
    assert all(torch.equal(x, y) for x, y in zip(cache._parts(), same._parts()))


def test_output_layouts():
    q, k, v = make(BF, 2, 2, 2, 9, 40, 128)
    want = window_attention(q, k, v)
    heads_major = torch.empty(2, 4, 9, 128, dtype=BF, device="cuda")
    assert torch.equal(window_attention(q, k, v, out=heads_major), want)
    wide = torch.zeros(2, 4, 9, 160, dtype=BF, device="cuda")
    assert torch.equal(window_attention(q, k, v, out=wide[..., :128]), want)
    assert (wide[..., 128:] == 0).all()
    for bad in (torch.empty(2, 4, 9, 130, dtype=BF, device="cuda")[..., 1:129],
                torch.empty(1, 4, 9, 128, dtype=BF, device="cuda").expand(2, -1, -1, -1), heads_major.half(),
                heads_major[:1], torch.empty(2, 4, 9, 128, dtype=BF)):
        with pytest.raises(ValueError, match="out must have"):
            window_attention(q, k, v, out=bad)


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(1, 2, 64)), "shape"), (dict(window=0), "window"), (dict(window=2.0), "window"),
    (dict(window=True), "window"), (dict(sinks=-1), "sinks"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(lengths=[3]), "lengths"), (dict(query_lengths=[1, 1]), "query_lengths"), (dict(heads=3), "multiple"),
    (dict(dim=96), "head_dim"), (dict(v_len=9), "one shape"), (dict(k_dtype=HF), "share dtype"),
    (dict(dtype=torch.float32), "fp16 or bf16"), (dict(batch=2), "batch"), (dict(grad=True), "no backward")])
def test_refusals(change, message):
    b, dt, d = 1, change.get("dtype", BF), change.get("dim", 64)
    heads = change.get("heads", 4)
    q = torch.zeros(change.get("batch", b), heads, 1, d, dtype=dt, device="cuda")
    k = torch.zeros(b, 2, 10, d, dtype=change.get("k_dtype", dt), device="cuda")
    v = torch.zeros(b, 2, change.get("v_len", 10), d, dtype=dt, device="cuda")
    if "q" in change:
        q = change["q"].to(dt).cuda()
    kw = {n: change[n] for n in ("window", "sinks", "scale") if n in change}
    for n in ("lengths", "query_lengths"):
        if n in change:
            kw[n] = torch.tensor(change[n], device="cuda")  # int64
    if "grad" in change:
        q.requires_grad_()
    with pytest.raises((ValueError, TypeError), match=message):
        window_attention(q, k, v, **kw)
    if "grad" in change:
        with torch.no_grad():
            window_attention(q, k, v)


@pytest.mark.parametrize("change,message", [
    (dict(start=-1), "start"), (dict(start=1.5), "start"), (dict(start=[0, 0]), "start"), (dict(counts=[1.0]), "counts"),
    (dict(heads=3), "of the cache"), (dict(batch=2), "of the cache"), (dict(v_len=3), "share their shape"),
    (dict(dtype=torch.float32), "fp16 or bf16"), (dict(v_dtype=HF), "share dtype"), (dict(device="cpu"), "GPU"),
    (dict(grad=True), "no backward")])
def test_append_refusals(change, message):
    cache = Int4KVCache(1, 2, 20, 64)
    kw = dict(device=change.get("device", "cuda"), dtype=change.get("dtype", BF))
    k = torch.zeros(change.get("batch", 1), change.get("heads", 2), 4, 64, **kw)
    v = torch.zeros(k.shape[0], k.shape[1], change.get("v_len", 4), 64, **kw).to(change.get("v_dtype", kw["dtype"]))
    if "grad" in change:
        k.requires_grad_()
    start = change.get("start", 0)
    start = torch.tensor(start, device="cuda") if isinstance(start, list) else start
    counts = torch.tensor(change["counts"], device="cuda") if "counts" in change else None
    with pytest.raises(ValueError, match=message):
        cache.append(k, v, start, counts=counts)
    assert all((x == 0).all() for x in cache._parts())


def test_cache_refusals():
    cache = Int4KVCache(1, 2, 20, 64)
    for bad in (dict(length=21), dict(length=-1), dict(length=True), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            cache.restore(**bad)
    q = torch.zeros(1, 4, 1, 128, dtype=BF, device="cuda")
    with pytest.raises(ValueError, match="head_dim"):
        kv4_attention(q, cache)
    with pytest.raises(ValueError, match="multiple"):
        kv4_attention(q[:, :3, :, :64], cache)
    with pytest.raises(ValueError, match="GPU"):
        kv4_attention(q.cpu(), cache)


def test_empty_batches_and_calls():
    q, k, v = make(BF, 2, 1, 2, 3, 8, 64)
    assert window_attention(q[:, :, :0], k, v).shape == (2, 2, 0, 64)
    assert window_attention(q[:0], k[:0], v[:0]).shape == (0, 2, 3, 64)
    assert (window_attention(q, k[:, :, :0], v[:, :, :0]) == 0).all()


# ------------------------------------------------------------------ large addresses
def test_offsets_past_four_gib():
    """A 16-bit cache of 5 GiB and a 4-bit one of 4.7 GB: the last sequence lies past 2^32 bytes."""
    b, hk, n, d = 10, 8, 131072, 128
    k = torch.zeros(b, hk, n, d, dtype=BF, device="cuda")
    v = torch.zeros(b, hk, n, d, dtype=BF, device="cuda")
    assert k.numel() * 2 > 2**31
    q, kk, vv = make(BF, 1, hk, 4, 1, 200, d)
    k[-1:, :, -200:], v[-1:, :, -200:] = kk, vv
    lengths = torch.full((b,), n, dtype=torch.int32, device="cuda")
    got = window_attention(q.expand(b, -1, -1, -1), k, v, lengths=lengths, window=200)
    want, mass, score = reference(q, kk, vv, [(200, 1)], None, 0, 1 / math.sqrt(d))
    assert ((got[-1:].double() - want).abs() <= bound16(want, mass, score, BF, 200)).all()
    assert (got[:-1] == 0).all()
    del k, v
    b = 30
    cache = Int4KVCache(b, hk, n, d)
    assert cache.k_codes.numel() > 2**30 and cache.k_codes[-1].data_ptr() - cache.k_codes.data_ptr() > 1.9e9
    start = torch.full((b,), n, dtype=torch.int32, device="cuda")
    start[-1] = n - 200
    cache.append(kk.expand(b, -1, -1, -1), vv.expand(b, -1, -1, -1), start)  # only the last one's positions exist
    got = kv4_attention(q.expand(b, -1, -1, -1), cache, window=200)
    small = Int4KVCache(1, hk, 200, d)
    small.append(kk, vv, 0)
    assert all(torch.equal(x[-1:, :, -200:], y) for x, y in zip(cache._parts(), small._parts()))
    kv, vm = quantize(kk)[3].cuda(), quantize(vv)
    want, _, score = reference(q, kv, vm[3].cuda(), [(200, 1)], None, 0, 1 / math.sqrt(d))
    bound = bound4(want, score, BF, 200, vm[3].abs().max().item(), vm[2].double().abs().max().item())
    assert ((got[-1:].double() - want).abs() <= bound).all()
    assert (got[:-1] == 0).all()


# ------------------------------------------------------------------ streams, graphs, a run of them together
def test_results_do_not_depend_on_the_stream_or_the_time():
    q, k, v = make(BF, 4, 2, 4, 1, 3000, 128)
    want = window_attention(q, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [window_attention(q, k, v) for _ in range(20)]
    here = [window_attention(q, k, v) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in outs + here)


def _decode(cache, q, k, v, lengths, out, window, sinks):
    """One step: the new token into the cache at its position, then its attention."""
    cache.append(k, v, lengths - 1)
    return kv4_attention(q, cache, lengths=lengths, window=window, sinks=sinks, out=out)


@pytest.mark.parametrize("window,sinks", [(None, 0), (64, 4)])
def test_prompt_then_decode_on_the_cache(window, sinks):
    """As they are used: a padded batch's prompts are attended in 16 bits and appended, then
    decode steps append a token and attend to the 4-bit cache; each step eagerly, and as one
    captured graph that is replayed with other lengths and tokens."""
    b, hk, g, d, prompt, steps, length = 2, 2, 4, 128, 70, 6, 100
    q, k, v = make(BF, b, hk, g, prompt, prompt, d)
    counts = int32([70, 41])
    first = window_attention(q, k, v, lengths=counts, query_lengths=counts, window=window, sinks=sinks)
    assert (first[1, :, 41:] == 0).all()
    cache, replayed = Int4KVCache(b, hk, length, d), Int4KVCache(b, hk, length, d)
    for c in (cache, replayed):
        c.append(k, v, 0, counts=counts)
    tokens = [make(BF, b, hk, g, 1, 1, d, seed=100 + i) for i in range(steps)]
    values = [[quantize(k)[3][i, :, :n], quantize(v)[3][i, :, :n]] for i, n in enumerate((70, 41))]

    at = counts.clone()
    sq, sk, sv = (torch.empty_like(x) for x in tokens[0])
    out = torch.empty(b, hk * g, 1, d, dtype=BF, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        spare = Int4KVCache(b, hk, length, d)
        _decode(spare, tokens[0][0], tokens[0][1], tokens[0][2], at + 1, out, window, sinks)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _decode(replayed, sq, sk, sv, at, out, window, sinks)

    for i, (nq, nk, nv) in enumerate(tokens):
        at.add_(1)
        eager = _decode(cache, nq, nk, nv, at.clone(), None, window, sinks)
        for dst, src in ((sq, nq), (sk, nk), (sv, nv)):
            dst.copy_(src)
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert all(torch.equal(x, y) for x, y in zip(cache._parts(), replayed._parts()))
        for s in range(b):
            values[s] = [torch.cat((old, quantize(x)[3][s]), 1) for old, x in zip(values[s], (nk, nv))]
            n = values[s][0].shape[1]
            kk, vv = (x[None].cuda() for x in values[s])
            want, _, score = reference(nq[s:s + 1], kk, vv, [(n, 1)], window, sinks, 1 / math.sqrt(d))
            low = torch.cat([quantize(v)[2][s].flatten()] + [quantize(t[2])[2][s].flatten() for t in tokens])
            bound = bound4(want, score, BF, n, vv.abs().max().item(), low.double().abs().max().item())
            assert ((eager[s:s + 1].double() - want).abs() <= bound).all(), (i, s)


@pytest.mark.parametrize("t", [1, 40])
def test_two_captured_calls_share_nothing(t):
    """Two graphs of split calls, replayed in turn and interleaved with eager work."""
    ins = [make(BF, 1, 2, 4, t, 2000, 128, seed=s) for s in (0, 50)]
    want = [window_attention(*x) for x in ins]
    outs = [torch.empty_like(w) for w in want]
    graphs = []
    for x, out in zip(ins, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            window_attention(*x, out=out)
        graphs.append(graph)
    for order in ((0, 1), (1, 0), (0, 0, 1, 1), (1, 1, 0)):
        for out in outs:
            out.zero_()
        for i in order:
            graphs[i].replay()
        other = window_attention(*ins[order[0]])
        torch.cuda.synchronize()
        assert torch.equal(other, want[order[0]])
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


# Joined key splits: few rows (one to 64 splits), the rows kernel (4 to 64), fp16 rows in
# groups over a 4-bit cache (12 to 48), each with a window that cuts splits short and lengths
# that leave splits without a key.
JOINS = {
    "few_window": (HF, 2, 2, 4, 1, 1500, 128, 700, 5, [(1500, 1), (3, 1)]),
    "few_window_d64": (BF, 1, 1, 7, 2, 3000, 64, 1400, 3, [(2950, 2)]),
    "few_most": (BF, 1, 1, 4, 1, 9000, 128, 8000, 0, [(8999, 1)]),
    "few_heads": (HF, 6, 4, 2, 2, 900, 64, None, 0, [(900, 2), (0, 2), (31, 2), (33, 1), (1, 1), (600, 2)]),
    "few_d256": (HF, 1, 2, 3, 1, 3000, 256, 1400, 9, [(2999, 1)]),
    "rows_4": (BF, 2, 8, 5, 70, 900, 128, None, 0, [(900, 70), (71, 64)]),
    "rows_d256": (BF, 2, 5, 2, 70, 700, 256, None, 0, [(699, 70), (5, 3)]),
    "rows_d64_window": (HF, 2, 6, 3, 70, 900, 64, 600, 3, [(900, 70), (500, 1)]),
    "rows_window": (BF, 1, 1, 4, 40, 2500, 64, 1200, 5, [(2400, 40)]),
    "rows_most": (BF, 1, 1, 4, 33, 6000, 128, None, 0, [(5999, 33)]),
    "rows_most_window": (HF, 1, 1, 2, 66, 6000, 128, 3000, 7, [(6000, 66)]),
    "groups_most_window": (HF, 1, 1, 7, 5, 5000, 128, 3000, 3, [(4990, 5)]),
    "groups_d64": (HF, 1, 2, 9, 12, 1000, 64, None, 0, [(1000, 12)]),
}


@pytest.mark.parametrize("case", JOINS)
@pytest.mark.parametrize("bits", [16, 4])
def test_joined_splits(case, bits):
    dtype, b, hk, g, t, length, d, window, sinks, spans = JOINS[case]
    kw = dict(lengths=int32([n for n, _ in spans]), query_lengths=int32([m for _, m in spans]), window=window,
              sinks=sinks)
    q, k, v = make(dtype, b, hk, g, t, length, d)
    out = torch.full((b, hk * g, t, d), 7.0, dtype=dtype, device="cuda")
    if bits == 16:
        want, mass, score = reference(q, k, v, spans, window, sinks, 1 / math.sqrt(d))
        bound = bound16(want, mass, score, dtype, length)
        got = window_attention(q, k, v, out=out, **kw)
    else:
        cache = Int4KVCache(b, hk, length, d)
        cache.append(k, v, 0)
        (_, _, _, kv), (_, _, v_min, vv) = quantize(k), quantize(v)
        kv, vv = kv.cuda(), vv.cuda()
        want, _, score = reference(q, kv, vv, spans, window, sinks, 1 / math.sqrt(d))
        bound = bound4(want, score, dtype, length, vv.abs().max().item(), v_min.double().abs().max().item())
        got = kv4_attention(q, cache, out=out, **kw)
    check(got, want, bound, spans, 7.0)
    again = torch.full_like(out, 7.0)
    if bits == 16:
        window_attention(q, k, v, out=again, **kw)
    else:
        kv4_attention(q, cache, out=again, **kw)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype,power", [(HF, -24), (HF, -22), (HF, -16), (HF, 12), (BF, -120), (BF, -60), (BF, 60)])
@pytest.mark.parametrize("t", [1, 9, 40])
@pytest.mark.parametrize("bits", [16, 4])
def test_queries_of_any_size(dtype, power, t, bits):
    """Queries times 2^power under a scale times 2^-power (as far as a float holds it); fp16
    ones at 2^-22 and below are subnormals."""
    b, hk, g, length, d = 2, 2, 4, 150, 128
    q, k, v = make(dtype, b, hk, g, t, length, d)
    q = (q.float() * 2.0**power).to(dtype)
    scale = 2.0 ** -power / math.sqrt(d)
    spans = [(150, t), (100, t)]
    kw = dict(lengths=int32([150, 100]), scale=scale)
    if bits == 16:
        want, mass, score = reference(q, k, v, spans, None, 0, scale)
        check(window_attention(q, k, v, **kw), want, bound16(want, mass, score, dtype, length), spans, 7.0)
        return
    cache = Int4KVCache(b, hk, length, d)
    cache.append(k, v, 0)
    (_, _, _, kv), (_, _, v_min, vv) = quantize(k), quantize(v)
    kv, vv = kv.cuda(), vv.cuda()
    want, _, score = reference(q, kv, vv, spans, None, 0, scale)
    bound = bound4(want, score, dtype, length, vv.abs().max().item(), v_min.double().abs().max().item())
    check(kv4_attention(q, cache, **kw), want, bound, spans, 7.0)


@pytest.mark.parametrize("case", [
    (BF, 5, 8, 4, 200, 600, 128, None, 0, [(600, 200), (200, 200), (31, 40), (0, 200), (599, 1)]),
    (BF, 3, 14, 3, 270, 700, 64, 600, 5, [(700, 270), (270, 270), (423, 111)])])
def test_kv4_wide_row_tiles(case):
    """Enough row tiles of a 4-bit cache for workgroups of 256 rows."""
    dtype, b, hk, g, t, length, d, window, sinks, spans = case
    q, k, v = make(dtype, b, hk, g, t, length, d)
    cache = Int4KVCache(b, hk, length, d)
    cache.append(k, v, 0)
    (_, _, _, kv), (_, _, v_min, vv) = quantize(k), quantize(v)
    kv, vv = kv.cuda(), vv.cuda()
    scale = 1 / math.sqrt(d)
    want, _, score = reference(q, kv, vv, spans, window, sinks, scale)
    bound = bound4(want, score, dtype, length, vv.abs().max().item(), v_min.double().abs().max().item())
    for i, (n, m) in enumerate(spans):  # poison
        for x in (cache.k_scales, cache.v_scales):
            x[i, :, n:] = float("nan")
    out = torch.full((b, hk * g, t, d), 7.0, dtype=dtype, device="cuda")
    kw = dict(lengths=int32([n for n, _ in spans]), query_lengths=int32([m for _, m in spans]), window=window,
              sinks=sinks)
    check(kv4_attention(q, cache, out=out, **kw), want, bound, spans, 7.0)


def test_kv4_wide_row_tiles_nan_groups():
    """A NaN group reaches the rows that see it and no other, there too."""
    b, hk, g, t, length, d = 5, 8, 4, 200, 600, 128
    q, k, v = make(BF, b, hk, g, t, length, d)
    bad = 450  # queries sit at 400 .. 599
    v[1, 3, bad, 70] = float("inf")
    cache = Int4KVCache(b, hk, length, d)
    cache.append(k, v, 0)
    out = kv4_attention(q, cache)
    nan = torch.isnan(out)
    assert nan[1, 12:16, 50:, 64:].all()
    nan[1, 12:16, 50:, 64:] = False
    assert not nan.any()


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 128), (BF, 128), (BF, 256)])
@pytest.mark.parametrize("sinks", [1, 4, 8, 9, 24, 33, 64, 65])
@pytest.mark.parametrize("window,t,length", [(64, 150, 701), (100, 150, 690), (257, 33, 683), (5, 300, 640), (130, 257, 663)])
def test_sinks_and_window_in_every_place(dtype, d, sinks, window, t, length):
    """Sinks in tiles of their own and joining the window's."""
    b, hk, g = 2, 1, 2
    spans = [(length, t), (length - 61, t - 7)]
    q, k, v = make(dtype, b, hk, g, t, length, d)
    want, mass, score = reference(q, k, v, spans, window, sinks, 1 / math.sqrt(d))
    bound = bound16(want, mass, score, dtype, length)
    for i, (n, m) in enumerate(spans):  # what no query of a sequence sees is poison
        k[i, :, n:], v[i, :, n:] = float("nan"), float("inf")
        first = max(0, n - m - window + 1)
        k[i, :, min(sinks, first):first], v[i, :, min(sinks, first):first] = float("inf"), float("nan")
    kw = dict(lengths=int32([n for n, _ in spans]), query_lengths=int32([m for _, m in spans]), window=window,
              sinks=sinks)
    out = torch.full((b, hk * g, t, d), 7.0, dtype=dtype, device="cuda")
    check(window_attention(q, k, v, out=out, **kw), want, bound, spans, 7.0)


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 128), (BF, 256)])
@pytest.mark.parametrize("sinks", [3, 8])
def test_infinities_among_sinks_and_window(dtype, d, sinks):
    """An infinite sink reaches every row, a NaN of the window the rows that see it alone."""
    b, hk, g, t, length, window = 1, 1, 2, 70, 400, 40
    spans = [(length, t)]
    q, k, v = make(dtype, b, hk, g, t, length, d)
    want, mass, score = reference(q, k, v, spans, window, sinks, 1 / math.sqrt(d))
    bound = bound16(want, mass, score, dtype, length)
    v[0, 0, sinks - 1, 5] = float("inf")
    v[0, 0, 395, 9] = float("nan")   # queries sit at 330 .. 399: the last five see it
    v[0, 0, 300, 11] = float("-inf")  # seen by 330 .. 339
    out = window_attention(q, k, v, window=window, sinks=sinks)
    assert (out[..., 5] == float("inf")).all()
    assert torch.isnan(out[:, :, 65:, 9]).all() and torch.isfinite(out[:, :, :65, 9]).all()
    assert (out[:, :, :10, 11] == float("-inf")).all() and torch.isfinite(out[:, :, 10:, 11]).all()
    keep = [c for c in range(d) if c not in (5, 9, 11)]
    check(out[..., keep], want[..., keep], bound[..., keep], spans, 7.0)
    error = (out[:, :, :65, 9].double() - want[:, :, :65, 9]).abs()
    assert (error <= bound[:, :, :65, 9]).all()
