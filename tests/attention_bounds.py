"""Per-element error bounds of the cached attention, close enough to see a lost tile.

With w_j the softmax weights, o = sum_j w_j v_j the output and, over a 4-bit cache, v_j = a_j +
minimum_j (a_j = code * scale; over a 16-bit one a_j = v_j):

* the output's rounding, half a step of |o|, is counted whole; fp16's steps stay 2^-24 below
  2^-14, so half a step is 2^-25 = 2^-11 2^-14 there;
* everything else is a sum of many roundings that have nothing to do with each other, each
  at most h of what it rounds, so of variance at most h^2 / 3 of its square.  Their sum is
  counted as Z = 8 times its standard deviation (10^6 elements exceed that once in 10^9 runs):
    - p, or p times the scale, rounded to 16 bits before the product: h_p w_j a_j;
    - a widened value: h_v w_j v_j;
    - a score's error d_j moves o by w_j d_j (v_j - o): a widened key, h_k of every term
      scale q_d k_jd; the fp32 sum of D products, sqrt(D + 8) 2^-24 of the sum of its terms'
      magnitudes; the exponent's argument and 2^x, 2^-23 (|terms| log2(e) + 4);
    - the fp32 sums over the keys and their joins, sqrt(n + 128) 2^-24 of sum_j w_j |terms|;
    - 16-bit weights that sink into the subnormals: at most `step` of the row's largest
      (fp16 alone).

The few-rows kernel multiplies 4-bit codes as fp16 subnormals, code * 2^-24.  The matrix unit
aligns the eight terms of a step to the largest exponent among them, where a subnormal counts
as 2^-14, and cuts them 24 bits below (measured: 2^14 * 8 * 2^-24 beside 2^-1 * 2^-24 loses the
latter; beside 2^0 * 2^-24 both are held).  So a term is off by less than 2^-24 2^-14 / 2^-24 =
2^-14 of the largest p * scale of its eight, one code's worth, always towards the same side:
7 2^-14 sum_j w_j scale_j in all, counted whole; and a score by 2^-14 of the row's largest |q|
times the key's scale for each of its D terms, of either sign.

fp16 queries over a 4-bit cache weigh the rounding of p * scale at the codes' middle, so that
a_j is (code - 8) * scale there.
"""
import math

import torch

from tests.attention_reference import half_step, quantize

Z = 8.0
FP16_HALF = 2.0**-11


def visible(n, m, window, sinks, device):
    """[m, n]: the keys that each query of a sequence sees."""
    p = torch.arange(n - m, n, device=device)[:, None]
    j = torch.arange(n, device=device)[None, :]
    see = j <= p
    if window:
        see = see & ((j > p - window) | (j < sinks))
    return see


def attend(q, k, v, see, scale):
    """64 bits: q [G, m, D] of one KV head, k, v [n, D], see [m, n] -> (o [G, m, D], w [G, m, n])."""
    s = torch.matmul(q.double(), k.double().t().contiguous()) * scale
    s = s.masked_fill(~see, -math.inf)
    w = torch.softmax(s, -1)
    w = torch.where(see.any(-1)[:, None], w, torch.zeros_like(w))
    return torch.matmul(w, v.double()), w


def few_rows(dtype, bits, rows):
    """Which of the two kernels a call takes, as their comments say (for what each rounds)."""
    return rows <= 16 or (bits == 4 and (dtype == torch.float16 or rows <= 64))


class Cache:
    """A cache's keys and values in 64 bits, in the parts that the bounds ask for."""

    def __init__(self, k, v, bits):
        self.bits = bits
        device = k.device
        if bits == 16:
            self.k, self.v = k.double(), v.double()
            self.v_part, self.v_mid = self.v, self.v
            self.k_terms, self.v_terms = self.k.abs(), self.v.abs()
            self.v_scale = None
            return

        def parts(x):
            codes, scales, minima, value = quantize(x)
            scales, minima = (y.double().repeat_interleave(64, -1).to(device) for y in (scales, minima))
            return codes.double().to(device), scales, minima, value.to(device)

        codes, scales, minima, self.k = parts(k)
        self.k_terms = codes * scales + minima.abs()
        self.k_unit = scales.amax(-1)  # [B, Hk, L]
        codes, scales, minima, self.v = parts(v)
        self.v_part, self.v_mid = codes * scales, (codes - 8) * scales
        self.v_terms = self.v_part + minima.abs()
        self.v_unit, self.v_scale = scales, scales.amax(-1)


def reference_and_bound(q, cache, spans, window, sinks, scale):
    """q [B, Hq, T, D] over a Cache -> (out, bound), zeros for rows that are not computed."""
    b, hq, t, d = q.shape
    hk = cache.k.shape[1]
    g, dtype = hq // hk, q.dtype
    few = few_rows(dtype, cache.bits, t * g)
    h_p = half_step(dtype) if cache.bits == 16 else FP16_HALF
    h_kv = FP16_HALF if cache.bits == 4 and not few else 0.0
    part = cache.v_part if few or cache.bits == 16 else cache.v
    if few and cache.bits == 4 and dtype == torch.float16:
        part = cache.v_mid
    step = 2.0**-39 if few else 2.0**-32
    if cache.bits == 16 and dtype == torch.bfloat16:
        step = 0.0  # bf16 has fp32's range
    out = torch.zeros(b, hq, t, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for i, (n, m) in enumerate(spans):
        if m == 0 or n == 0:
            continue
        rows = max(1, (1 << 24) // (g * n))
        for h in range(hk):
            heads = slice(h * g, h * g + g)
            k, v, a = cache.k[i, h, :n], cache.v[i, h, :n], part[i, h, :n]
            kt, vt = cache.k_terms[i, h, :n], cache.v_terms[i, h, :n]
            for t0 in range(0, m, rows):
                t1 = min(m, t0 + rows)
                see = visible(n, m, window, sinks, q.device)[t0:t1]
                qq = q[i, heads, t0:t1].double()
                o, w = attend(qq, k, v, see, scale)
                terms = torch.matmul(qq.abs(), kt.t().contiguous()) * scale
                delta = (math.sqrt(d + 8) * 2.0**-24 * terms).square()
                delta += (2.0**-23 * (terms / math.log(2) + 4)).square()
                if h_kv:
                    delta += h_kv**2 / 3 * scale**2 * torch.matmul(qq.square(), k.square().t().contiguous())
                if cache.bits == 4 and few:
                    cut = 2.0**-14 * scale * qq.abs().amax(-1, keepdim=True) * cache.k_unit[i, h, :n]
                    delta += d / 3 * cut.square()
                w2 = w.square()
                wd = w2 * delta
                var = torch.matmul(wd, v.square()) - 2 * o * torch.matmul(wd, v) + o.square() * wd.sum(-1, keepdim=True)
                var = var.clamp_min(0) + h_p**2 / 3 * torch.matmul(w2, a.square())
                if h_kv:
                    var += h_kv**2 / 3 * torch.matmul(w2, v.square())
                var += ((n + 128) * 2.0**-48) * torch.matmul(w, vt).square()
                if step:
                    largest, size = w, v
                    if cache.bits == 4 and few:  # p * scale, over codes
                        largest, size = w * cache.v_scale[i, h, :n], torch.full_like(v, 15.0)
                    lost = step * largest.amax(-1, keepdim=True)
                    var += lost.square() / 3 * torch.matmul(see.double(), size.square())
                out[i, heads, t0:t1] = o
                smallest = 2.0**-14 if dtype == torch.float16 else 0.0
                bound[i, heads, t0:t1] = half_step(dtype) * o.abs().clamp_min(smallest) + Z * var.sqrt()
                if cache.bits == 4 and few:
                    bound[i, heads, t0:t1] += 7 * 2.0**-14 * torch.matmul(w, cache.v_unit[i, h, :n])
    return out, bound
