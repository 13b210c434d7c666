"""The cached attention's definition in 64 bits, with the error bounds of its kernels.

Bounds count roundings only.  For one output element, with w_j the softmax weights,
A = sum_j w_j |v_j| and S = max_j scale sum_d |q_d k_jd| (what a score's fp32 sum is made of):

* the output's rounding: half a step, eps(out) / 2 of |o|;
* p rounded to 16 bits before the product with V: eps(p) / 2 of A;
* a score's error d: the fp32 sum of D products, (D + 8) 2^-24 S, and the exponent's argument
  and 2^x, 2^-23 (S log2(e) + 4); it enters numerator and denominator, 2 d A;
* the fp32 sums over n keys and the joins of up to 64 splits: (n + 128) 2^-24 A.
"""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(q, k, v, spans, window, sinks, scale):
    """q [B, Hq, T, D], k, v [B, Hk, L, D] -> (out, A, S), zeros for rows that are not computed.
    Hidden keys never enter: each row is computed from the keys that it sees alone."""
    b, hq, t, d = q.shape
    g = hq // k.shape[1]
    out = torch.zeros(b, hq, t, d, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    score = torch.zeros(b, hq, t, 1, dtype=torch.float64, device=q.device)
    for i, (n, m) in enumerate(spans):
        for row in range(m):
            p = n - m + row
            if p < 0:
                continue
            seen = torch.arange(p + 1, device=q.device)
            if window:
                seen = seen[(seen > p - window) | (seen < sinks)]
            kk = k[i][:, seen].double().repeat_interleave(g, 0)  # [Hq, keys, D]
            vv = v[i][:, seen].double().repeat_interleave(g, 0)
            qq = q[i, :, row].double()[:, :, None]
            s = torch.matmul(kk, qq)[..., 0] * scale
            w = torch.softmax(s, -1)[:, None]
            out[i, :, row] = torch.matmul(w, vv)[:, 0]
            mass[i, :, row] = torch.matmul(w, vv.abs())[:, 0]
            score[i, :, row, 0] = torch.matmul(kk.abs(), qq.abs())[..., 0].amax(-1) * scale
    return out, mass, score


def bound16(out, mass, score, dtype, keys):
    """16-bit cache: p has the cache's type."""
    d = out.shape[-1]
    delta = (d + 8) * 2.0**-24 * score + 2.0**-23 * (score / math.log(2) + 4)
    return half_step(dtype) * (out.abs() + mass) * (1 + half_step(dtype)) + (2 * delta + (keys + 128) * 2.0**-24) * mass


def bound4(out, score, dtype, keys, values, minima):
    """4-bit cache: fp16 products.  q is exact or within 2^-12 of a bf16 / fp16 element that is
    2^-23 of the row's largest (counted as 2^-12 S); a widened key or value, or p times a scale, is
    rounded to fp16 once, 2^-12 of itself: of the score 2^-12 S, of the value at most 2^-12 of
    R = max |v| + 2 max |minimum| (codes * scale = v - minimum)."""
    d = out.shape[-1]
    size = values + 2 * minima
    delta = (d + 8) * 2.0**-24 * 3 * score + 2.0**-23 * (score / math.log(2) + 4) + 2.0**-11 * score
    return (half_step(dtype) * out.abs() + (2.0**-12 + 2.0**-12 + 2 * delta + (keys + 128) * 2.0**-24) * size)


GROUP = 64


def quantize(x):
    """Codes, scales and minima of the 4-bit format by its definition (one fp32 operation a
    step, on the CPU), and the values they stand for in 64 bits."""
    x = x.detach().cpu().float()
    groups = x.unflatten(-1, (-1, GROUP))
    lo, hi = groups.amin(-1, keepdim=True), groups.amax(-1, keepdim=True)
    minimum = lo.half()
    scale = ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32)).half()
    inverse = torch.where(scale > 0, 1 / scale.float(), torch.zeros_like(lo))
    codes = ((groups - minimum.float()) * inverse).round().clamp(0, 15)
    bad = ~(groups.abs() <= 32768).all(-1, keepdim=True)
    scale = torch.where(bad, torch.zeros_like(scale), scale)
    minimum = torch.where(bad, torch.full_like(minimum, float("nan")), minimum)
    value = codes.double() * scale.double() + minimum.double()
    return codes.flatten(-2).to(torch.uint8), scale[..., 0], minimum[..., 0], value.flatten(-2)


def packed(codes):
    """The cache's code bytes: word [c, g] of 16 x D / 64 holds columns 64 g + 4 c + k at bits 4 k."""
    d = codes.shape[-1]
    c = codes.to(torch.int32).reshape(*codes.shape[:-1], d // GROUP, 16, 4)
    word = c[..., 0] | c[..., 1] << 4 | c[..., 2] << 8 | c[..., 3] << 12
    word = word.transpose(-1, -2).reshape(*codes.shape[:-1], d // 4)
    return torch.stack((word & 255, word >> 8), -1).flatten(-2).to(torch.uint8)
