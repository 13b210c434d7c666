"""window_attention, kv4_attention and Int4KVCache where they can go wrong: infinities in joined
splits, weights far below a row's largest, the ends of the types' ranges, addresses past 2^32
bytes, calls that cannot be recorded."""
import math

import pytest
import torch

from marlin_style_fluxbin_amd import Int4KVCache, _lib, kv4_attention, window_attention
from tests.attention_bounds import Cache, reference_and_bound
from tests.test_cached_attention_gpu import BF, HF, check, int32, make

pytestmark = pytest.mark.gpu
INF = float("inf")


def splits_of(dtype, b, hk, g, t, length, d, window=0, sinks=0, kv4=0):
    nbytes = _lib.library().fx_cached_attention_workspace_bytes(b, hk * g, hk, t, length, d, window, sinks,
                                                                _lib.dtype_code(dtype), kv4)
    return max(1, nbytes // (b * hk * g * t * (d + 2) * 4))


# ------------------------------------------------------------------ visible infinities
@pytest.mark.parametrize("dtype,b,hk,g,t,length,d", [
    (BF, 24, 8, 4, 1, 300, 128),   # one split
    (BF, 1, 8, 4, 1, 700, 128), (BF, 1, 8, 4, 1, 1500, 128), (HF, 1, 2, 3, 2, 1700, 64),  # joined by one wave a row
    (HF, 1, 4, 2, 1, 1800, 256), (BF, 1, 2, 4, 1, 5000, 128),  # 16; 40, joined by four
    (BF, 2, 2, 5, 70, 900, 128), (BF, 2, 5, 2, 70, 700, 256), (HF, 1, 1, 4, 33, 6000, 128)])  # the rows kernel
def test_infinities_in_every_split(dtype, b, hk, g, t, length, d):
    """Every 64 keys one value's column holds an infinity that every row sees: it reaches each
    of them, whichever split it lies in, and nothing else changes."""
    q, k, v = make(dtype, b, hk, g, t, length, d)
    scale = 1 / math.sqrt(d)
    want, bound = reference_and_bound(q, Cache(k, v, 16), [(length, t)] * b, None, 0, scale)
    keys = range(5, length - t, 64)
    assert len(keys) <= d - 8
    for c, j in enumerate(keys):
        v[:, :, j, c] = -INF if c % 3 == 0 else INF
    out = window_attention(q, k, v)
    for c in range(len(keys)):
        assert (out[..., c] == (-INF if c % 3 == 0 else INF)).all(), (c, splits_of(dtype, b, hk, g, t, length, d))
    rest = slice(len(keys), None)
    check(out[..., rest], want[..., rest], bound[..., rest], [(length, t)] * b, 7.0)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,length", [(1, 300), (1, 2000), (150, 400), (60, 3000)])
@pytest.mark.parametrize("top,at", [(70, 10), (10, 70), (130, 200), (20, 10), (20, 40), (40, 20)])
def test_an_infinity_of_little_weight(dtype, d, t, length, top, at):
    """One key outweighs the others by e^40 (their p is no fp16 number): their infinite values
    still reach the rows that see them."""
    q, k, v = make(dtype, 1, 1, 2, t, length, d)
    q.fill_(1.0)
    k.zero_()
    k[:, :, top] = 40.0
    v[:, :, at, 3], v[:, :, at + 1, 5] = INF, -INF
    got = window_attention(q, k, v, scale=1 / d)
    see = torch.arange(length - t, length, device="cuda") >= max(top, at + 1)  # rows that see all three
    assert (got[:, :, see, 3] == INF).all() and (got[:, :, see, 5] == -INF).all()
    rest = [c for c in range(d) if c not in (3, 5)]
    assert torch.equal(got[:, :, see][..., rest], v[:, :, top, None][..., rest].expand(-1, 2, int(see.sum()), -1))


# ------------------------------------------------------------------ weights far below the largest
@pytest.mark.parametrize("gap", [18.3, 22.6, 28.7])
@pytest.mark.parametrize("b,hk,t,length,d", [(32, 16, 1, 1000, 128), (1, 1, 1, 3000, 64), (16, 16, 1, 900, 256),
                                             (2, 1, 150, 1000, 128), (2, 1, 150, 1000, 256)])
def test_small_fp16_weights_count(gap, b, hk, t, length, d):
    """A key of value zero outweighs the others by 2^gap; what they hold is the output.  p is
    fp16: 2^15 at the row's largest in the few-rows kernel, 2^7 at least in the rows kernel, so
    that it is off by half a step, 2^-11 of itself or 2^-40 (2^-32) of the largest."""
    q, k, v = make(HF, b, hk, 1, t, length, d)
    q.fill_(1.0)
    k.zero_()
    k[:, :, 37] = gap * math.log(2)
    v.abs_().add_(1).mul_(50)
    v[:, :, 37] = 0
    got = window_attention(q, k, v, scale=1 / d).double()
    score = k[0, 0, 37, 0].double()  # as fp16 holds it
    p = torch.arange(length - t, length, device="cuda")
    weight = torch.exp(-score) / (1 + p * torch.exp(-score))
    sums = v.double().cumsum(2)[:, :, p]
    want = sums * weight[:, None]
    step = 2.0**-40 if t == 1 else 2.0**-32
    bound = want * (2.0**-10 + 2.0**-16) + step * sums + 2.0**-25
    error = (got - want).abs()
    assert (error <= bound).all(), (error / bound).max().item()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("power", range(0, 16, 3))
@pytest.mark.parametrize("t,length,d", [(1, 700, 128), (20, 300, 64), (150, 400, 128), (70, 300, 256)])
def test_scores_of_any_size(dtype, bits, power, t, length, d):
    """Queries of 2^power, keys of 0 and 2^power, scores up to 2^37 and more: the mean of the
    values whose keys are largest (of all of them where the scores are 1 apart)."""
    q, k, v = make(dtype, 1, 1, 2, t, length, d)
    q.fill_(2.0**power)
    k.zero_()
    g = torch.Generator().manual_seed(power)
    k[:, :, torch.randperm(length, generator=g)[:length // 2]] = 2.0**power
    k[:, :, 0] = 2.0**power
    scale = 1 / d if power == 0 else 1.0
    spans = [(length, t)]
    want, bound = reference_and_bound(q, Cache(k, v, bits), spans, None, 0, scale)
    if bits == 16:
        got = window_attention(q, k, v, scale=scale)
    else:
        cache = Int4KVCache(1, 1, length, d)
        cache.append(k, v, 0)
        got = kv4_attention(q, cache, scale=scale)
    check(got, want, bound, spans, 7.0)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("power", [0, -6, -10, -14])
@pytest.mark.parametrize("b,hk,t,length,d", [(16, 8, 1, 2000, 128), (1, 1, 1, 5000, 128), (8, 8, 1, 900, 256),
                                             (1, 1, 20, 700, 128), (1, 1, 150, 700, 128)])
def test_kv4_groups_of_mixed_size(dtype, power, b, hk, t, length, d):
    """A strong key, and value groups 2^power as large as their neighbours: each group is as
    exact as if it were alone."""
    q, k, v = make(dtype, b, hk, 1, t, length, d)
    q.fill_(1.0)
    k.zero_()
    k[:, :, 37] = 12 * math.log(2)
    v[..., 64:128] *= 2.0**power
    cache = Int4KVCache(b, hk, length, d)
    cache.append(k, v, 0)
    spans = [(length, t)] * b
    want, bound = reference_and_bound(q, Cache(k, v, 4), spans, None, 0, 1 / d)
    check(kv4_attention(q, cache, scale=1 / d), want, bound, spans, 7.0)


# ------------------------------------------------------------------ the ends of the ranges
@pytest.mark.parametrize("bits,q_value,scale", [(4, 2.0**-133, 1e-3), (4, 2.0**-126, 1e-6), (16, 1.0, 1e-42),
                                                (4, 1.0, 1e-42)])
@pytest.mark.parametrize("t", [1, 150])
def test_scores_that_vanish(bits, q_value, scale, t):
    """Queries and scales so small that every score is zero: the mean of the visible values."""
    b, hk, g, length, d = 1, 2, 2, 260, 128
    q, k, v = make(BF, b, hk, g, t, length, d)
    q.fill_(q_value)
    spans = [(length, t)]
    want, bound = reference_and_bound(q, Cache(k, v, bits), spans, None, 0, scale)
    if bits == 16:
        got = window_attention(q, k, v, scale=scale)
    else:
        cache = Int4KVCache(b, hk, length, d)
        cache.append(k, v, 0)
        got = kv4_attention(q, cache, scale=scale)
    check(got, want, bound, spans, 7.0)


# ------------------------------------------------------------------ calls that are refused
def test_what_a_kernel_cannot_record_is_refused():
    """Forward-mode tangents and tracers: the kernels would drop the one and leave no trace of
    themselves in the other's record."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    q, k, v = make(BF, 1, 2, 2, 3, 40, 64)
    want = window_attention(q, k, v)
    cache = Int4KVCache(1, 2, 40, 64)
    cache.append(k, v, 0)
    want4 = kv4_attention(q, cache)
    out = torch.zeros_like(q)
    before = [x.clone() for x in cache._parts()]
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: window_attention(dual(q), k, v), lambda: window_attention(q, dual(k), v),
                     lambda: window_attention(q, k, dual(v)), lambda: window_attention(q, k, v, out=dual(out)),
                     lambda: kv4_attention(dual(q), cache), lambda: kv4_attention(q, cache, out=dual(out)),
                     lambda: cache.append(dual(k), v, 0), lambda: cache.append(k, dual(v), 0)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        assert torch.equal(window_attention(q, k, v), want)  # no tangent: as ever
        assert torch.equal(kv4_attention(q, cache), want4)
        cache.append(k, v, 0)
    for call in (lambda x: window_attention(x, k, v), lambda x: kv4_attention(x, cache),
                 lambda x: cache.append(k, v, 0) or x + 1, lambda x: cache.restore()[0]):
        with pytest.raises(ValueError, match="trac"):
            torch.jit.trace(call, (q,))
        with pytest.raises(ValueError, match="trac"):
            make_fx(call)(q)
    for call in (lambda x: window_attention(x, k, v), lambda x: kv4_attention(x, cache)):
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.jvp(call, (q,), (torch.ones_like(q),))
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.vmap(call)(torch.stack((q, q)))
    assert (out == 0).all() and all(torch.equal(x, y) for x, y in zip(before, cache._parts()))
    assert torch.equal(window_attention(q, k, v), want)


def test_a_compiled_caller_runs_the_call_as_it_is():
    q, k, v = make(BF, 1, 2, 2, 3, 40, 64)
    cache = Int4KVCache(1, 2, 40, 64)

    def step(q, k, v):
        cache.append(k * 1, v, 0)
        return window_attention(q * 1, k, v, window=9), kv4_attention(q, cache) * 1, cache.restore()[0]

    want = step(q, k, v)
    got = torch.compile(step, backend="eager")(q, k, v)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_an_output_whose_rows_overlap_is_refused():
    q, k, v = make(BF, 2, 2, 2, 5, 40, 64)
    want = window_attention(q, k, v)
    memory = torch.zeros(2 * 4 * 5 * 64, dtype=BF, device="cuda")
    for bad in ((1280, 320, 32, 1), (1280, 64, 64, 1), (640, 320, 64, 1), (8, 320, 64, 1), (1280, 0, 64, 1)):
        with pytest.raises(ValueError, match="its own memory"):
            window_attention(q, k, v, out=memory.as_strided(q.shape, bad))
    assert (memory == 0).all()
    for good in ((1280, 320, 64, 1), (1280, 64, 256, 1), (320, 640, 64, 1), (64, 128, 512, 1), (256, 64, 512, 1)):
        assert torch.equal(window_attention(q, k, v, out=memory.as_strided(q.shape, good)), want)


# ------------------------------------------------------------------ large addresses
def test_16_bit_caches_past_2_to_32_bytes():
    """Keys, values, queries and outputs beyond 2^32 bytes of their tensors' starts, in both
    kernels, and read by append."""
    b, hk, g, n, d, tail, window = 18, 8, 4, 131072, 128, 300, 200
    k, v = (torch.zeros(b, hk, n, d, dtype=BF, device="cuda") for _ in range(2))
    assert k[-1].data_ptr() - k.data_ptr() > 2**32
    for t in (1, 100):
        q, kk, vv = make(BF, 1, hk, g, t, tail, d)
        k[-1:, :, -tail:], v[-1:, :, -tail:] = kk, vv
        want, bound = reference_and_bound(q, Cache(kk, vv, 16), [(tail, t)], window, 0, 1 / math.sqrt(d))
        got = window_attention(q.expand(b, -1, -1, -1), k, v, window=window)
        check(got[-1:], want, bound, [(tail, t)], 7.0)
        assert (got[:-1] == 0).all()
        # two sequences' q and out 2^32 bytes apart
        apart = (2**31, d, hk * g * d, 1)
        far = [torch.zeros(2**31 + t * hk * g * d, dtype=BF, device="cuda").as_strided((2, hk * g, t, d), apart)
               for _ in range(2)]
        far[0][1:] = q
        got = window_attention(far[0], k[-2:], v[-2:], window=window, out=far[1])
        check(got[1:], want, bound, [(tail, t)], 7.0)
        assert (got[0] == 0).all()
    cache, small = Int4KVCache(b, hk, n, d), Int4KVCache(1, hk, tail, d)
    cache.append(k, v, 0)
    small.append(kk, vv, 0)
    assert all(torch.equal(x[-1:, :, -tail:], y) for x, y in zip(cache._parts(), small._parts()))
    assert all((x[:-1] == 0).all() for x in cache._parts())


def test_4_bit_caches_past_2_to_32_bytes():
    b, hk, g, n, d, tail, window = 68, 8, 4, 131072, 128, 300, 200
    cache = Int4KVCache(b, hk, n, d)
    assert cache.k_codes[-1].data_ptr() - cache.k_codes.data_ptr() > 2**32
    start = torch.full((b,), n, dtype=torch.int32, device="cuda")
    start[-1] = n - tail
    for dtype, t in ((BF, 1), (BF, 100), (HF, 100)):  # the rows kernel: bf16's 100 tokens
        q, kk, vv = make(dtype, 1, hk, g, t, tail, d)
        small = Int4KVCache(1, hk, tail, d)
        small.append(kk, vv, 0)
        cache.append(kk.expand(b, -1, -1, -1), vv.expand(b, -1, -1, -1), start)  # the other positions do not exist
        assert all(torch.equal(x[-1:, :, -tail:], y) for x, y in zip(cache._parts(), small._parts()))
        want, bound = reference_and_bound(q, Cache(kk, vv, 4), [(tail, t)], window, 0, 1 / math.sqrt(d))
        got = kv4_attention(q.expand(b, -1, -1, -1), cache, window=window)
        check(got[-1:], want, bound, [(tail, t)], 7.0)
        assert (got[:-1] == 0).all()
    for x, y in zip(cache.restore(dtype=HF), small.restore(dtype=HF)):
        assert x[-1].data_ptr() - x.data_ptr() > 2**34
        assert torch.equal(x[-1:, :, -tail:], y) and (x[-1, :, :-tail] == 0).all() and not x[:-1].any()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,length", [(1, 300), (4, 700), (150, 400)])
def test_rows_of_minus_infinity_beside_infinite_values(dtype, d, t, length):
    """A head whose scores are all -inf is NaN, beside one that sees an infinite value."""
    q, k, v = make(dtype, 1, 1, 2, t, length, d)
    q[:, 0], q[:, 1] = -1.0, 0.0
    k.fill_(1.0)
    k[..., 0] = INF
    q[:, 1, :, 0] = 1.0  # +inf against +inf
    k2 = k.clone()
    k2[..., 0] = 1.0
    v[:, :, 20, 3] = INF
    got = window_attention(q, k, v)
    assert torch.isnan(got).all()
    got = window_attention(q, k2, v)
    assert (got[..., 3] == INF).all() and torch.isfinite(got[..., 4:]).all()
    q[:, 1] = 0.0
    k3 = torch.zeros_like(k)
    k3[..., 1] = -INF
    q[:, 0], q[:, 1] = 1.0, 0.0  # the second: 0 times -inf, NaN
    assert torch.isnan(window_attention(q, k3, v)).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t,length,d", [(1, 3000, 128), (150, 1000, 128), (150, 1000, 256)])
def test_finite_columns_beside_infinite_ones(dtype, t, length, d):
    """What an infinity in one column costs the others' exactness: nothing."""
    q, k, v = make(dtype, 1, 2, 2, t, length, d)
    spans = [(length, t)]
    want, bound = reference_and_bound(q, Cache(k, v, 16), spans, None, 0, 1 / math.sqrt(d))
    v[:, :, ::50, 3] = INF
    v[:, :, 7::50, 4] = float("nan")
    got = window_attention(q, k, v)
    assert (got[..., 3] == INF).all() and torch.isnan(got[..., 4]).all()
    check(got[..., 5:], want[..., 5:], bound[..., 5:], spans, 7.0)
