"""Attention over long caches: what a user runs, as cases that can be timed and checked.

Three operators, each through the framework's public entry points:

* ``window``: ``window_attention``, causal attention of T new tokens over 16-bit keys
  and values with a sliding window and a few first tokens that stay visible (sinks).
* ``kv4``: ``kv4_attention``, the same over an ``Int4KVCache`` (4-bit codes, a scale and a
  minimum per 64 columns); with ``append`` the new tokens' keys and values are written
  into the cache first, as a decode step does.
* ``append``: a prompt's keys and values written into an ``Int4KVCache`` and the cache
  read back to 16 bits.

The arithmetic.  Sequence b holds ``n`` keys, the last ``m`` of which belong to the call's
queries: query t < m sits at position p = n - m + t and sees the keys j <= p with
j > p - window or j < sinks.  out = softmax(scale q . k_j) v_j over them; a row that sees
nothing is zero, rows t >= m stay as they were.  A 4-bit group of 64 columns holds
minimum = fp16(lo), scale = fp16(fp32(hi - lo) * fp32(1 / 15)) and
code = clamp(round(fp32(x - minimum) * fp32(1 / scale)), 0, 15), ties to even, in fp32
(a zero scale gives code 0), and stands for code * scale + minimum.
"""
from __future__ import annotations

import math

import torch

own = False  # False: the plain forms below; True: the framework's operators

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 64


def listed():
    return [
        # one chat sequence decoding with a window: the smallest call, latency is what it costs
        {"name": "window_decode_1", "op": "window", "dtype": "bf16", "batch": 1, "tokens": 1, "length": 2000,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 1024, "sinks": 4, "ragged": False, "layout": "heads"},
        # a serving batch at ragged lengths
        {"name": "window_decode_batch", "op": "window", "dtype": "bf16", "batch": 24, "tokens": 1, "length": 16384,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 4096, "sinks": 4, "ragged": True, "layout": "heads"},
        # a padded batch of short odd prompts behind a cached prefix; keys stored token by token
        {"name": "window_padded_odd", "op": "window", "dtype": "f16", "batch": 3, "tokens": 301, "length": 1501,
         "heads": 14, "kv_heads": 2, "dim": 64, "window": 257, "sinks": 3, "ragged": True, "layout": "tokens"},
        # an ordinary prompt's prefill with a window
        {"name": "window_prefill", "op": "window", "dtype": "bf16", "batch": 1, "tokens": 4096, "length": 4096,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 1024, "sinks": 4, "ragged": False, "layout": "tokens"},
        # the largest: a long prompt without a window
        {"name": "causal_prefill_long", "op": "window", "dtype": "bf16", "batch": 1, "tokens": 16384,
         "length": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "ragged": False,
         "layout": "tokens"},
        # a decode step (append, then attend) of one short sequence on the 4-bit cache
        {"name": "kv4_step_short", "op": "kv4", "dtype": "bf16", "batch": 1, "tokens": 1, "length": 700,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "ragged": False, "append": True},
        # one very long sequence: what the 4-bit cache is for
        {"name": "kv4_decode_long", "op": "kv4", "dtype": "bf16", "batch": 1, "tokens": 1, "length": 131072,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "ragged": False, "append": False},
        # a serving batch's decode step
        {"name": "kv4_step_batch", "op": "kv4", "dtype": "bf16", "batch": 32, "tokens": 1, "length": 32768,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "ragged": True, "append": True},
        # a few drafted tokens per sequence verified at once, odd head groups, windowed
        {"name": "kv4_verify", "op": "kv4", "dtype": "f16", "batch": 8, "tokens": 5, "length": 12289,
         "heads": 28, "kv_heads": 4, "dim": 128, "window": 4096, "sinks": 4, "ragged": True, "append": True},
        # a chunk of a prompt that continues a cached one
        {"name": "kv4_chunk", "op": "kv4", "dtype": "bf16", "batch": 1, "tokens": 1024, "length": 9000,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "ragged": False, "append": True},
        # a prompt into the cache and back
        {"name": "append_prompt", "op": "append", "dtype": "bf16", "batch": 1, "tokens": 8192, "length": 8192,
         "kv_heads": 8, "dim": 128, "ragged": False},
        # a batch's odd chunks behind ragged prefixes
        {"name": "append_chunks", "op": "append", "dtype": "f16", "batch": 16, "tokens": 77, "length": 1000,
         "kv_heads": 2, "dim": 64, "ragged": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: decode, a few tokens, a chunk or a prompt; any head grouping, both
    types, with and without a window; bounded by the largest listed cases' work."""
    limit = [work(c) for c in listed()]
    max_bytes, max_flops = max(w["bytes"] for w in limit), max(w["flops"] for w in limit)
    op = rng.choice(["window", "window", "kv4", "kv4", "append"])
    case = {"op": op, "dtype": rng.choice(["bf16", "f16"])}
    case["kv_heads"], groups = rng.choice([(8, 4), (8, 4), (4, 7), (2, 5), (1, 8), (8, 1), (2, 16), (6, 3)])
    case["dim"] = rng.choice([64, 128, 128, 256])
    case["tokens"] = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 8192)])
    case["length"] = case["tokens"] + rng.choice([0, _log_int(rng, 1, 65536)])
    case["batch"] = _log_int(rng, 1, 32)
    case["ragged"] = rng.random() < 0.6
    if op != "append":
        case["heads"] = case["kv_heads"] * groups
        case["window"] = rng.choice([0, _log_int(rng, 1, 8192)])
        case["sinks"] = rng.choice([0, 1, 4, _log_int(rng, 1, 200)]) if case["window"] else 0
        if op == "window":
            case["layout"] = rng.choice(["heads", "tokens"])
        else:
            case["append"] = rng.random() < 0.5
    while True:
        cost = work(case)
        if cost["bytes"] <= max_bytes and cost["flops"] <= max_flops / 2:
            return case
        if case["batch"] > 1:
            case["batch"] //= 2
        else:
            case["length"] -= case["tokens"] // 2
            case["tokens"] -= case["tokens"] // 2
            if case["tokens"] == 1:
                case["length"] = max(1, case["length"] // 2)


def _spans(case):
    """(keys, queries) of each sequence: ragged batches fall to about half."""
    b, t, length = case["batch"], case["tokens"], case["length"]
    if not case["ragged"]:
        return [(length, t)] * b
    spans = []
    for i in range(b):
        m = max(1, t - (i * t) // (2 * b))
        past = (length - t) - (i * (length - t)) // (2 * b)
        spans.append((m + past, m))
    return spans


def _visible(case):
    """Over the batch: (query, key) pairs, keys that some query sees, queries."""
    pairs = keys = queries = 0
    w, s = case["window"], case["sinks"]
    for n, m in _spans(case):
        first = n - m
        queries += m
        if not w:
            pairs += m * first + m * (m + 1) // 2
            keys += n
            continue
        for p in range(first, n):
            lo = max(0, p - w + 1)
            pairs += p + 1 - lo + min(s, lo)
        lo = max(0, first - w + 1)
        keys += n - lo + min(s, lo)
    return pairs, keys, queries


def work(case):
    d, hk = case["dim"], case["kv_heads"]
    packed = 2 * (d // 2 + d // GROUP * 4)  # bytes of one head's key and value in 4 bits
    if case["op"] == "append":
        written = sum(m for _, m in _spans(case))
        total = case["batch"] * case["length"]
        # read and pack the new tokens; read the whole cache and widen it
        return {"bytes": written * hk * (4 * d + packed) + total * hk * (packed + 4 * d),
                "flops": 6 * d * hk * (written + total)}
    pairs, keys, queries = _visible(case)
    per_key = packed if case["op"] == "kv4" else 4 * d
    nbytes = keys * hk * per_key + 4 * queries * case["heads"] * d
    if case.get("append"):
        nbytes += queries * hk * 4 * d
    return {"bytes": nbytes, "flops": 4 * d * case["heads"] * pairs}


def _inputs(case, seed):
    """q, k, v of the case: normalised heads, a few strong key channels, values of mixed size."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    b, t, length, hk, d = (case[x] for x in ("batch", "tokens", "length", "kv_heads", "dim"))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)

    channel = torch.exp(0.5 * normal(hk, 1, d))
    token_major = case.get("layout") == "tokens"
    shape = (b, length, hk, d) if token_major else (b, hk, length, d)
    k = torch.empty(shape, dtype=dtype, device=DEVICE)
    v = torch.empty(shape, dtype=dtype, device=DEVICE)
    k, v = (x.transpose(1, 2) if token_major else x for x in (k, v))
    for i in range(b):
        k[i] = (normal(hk, length, d) * channel).to(dtype)
        v[i] = (normal(hk, length, d) * torch.exp(0.3 * normal(hk, length, 1))).to(dtype)
    q = None
    if "heads" in case:
        q = normal(b, t, case["heads"], d).to(dtype).transpose(1, 2)
    return q, k, v


# ------------------------------------------------------------------ plain forms
def _quantize_plain(x):
    """[..., D] -> packed codes [..., D / 2], scales and minima [..., D / 64]."""
    groups = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = groups.amin(-1), groups.amax(-1)
    minimum = lo.half()
    scale = ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)).half()
    inverse = torch.where(scale > 0, 1 / scale.float(), torch.zeros_like(lo))
    code = ((groups - minimum.float()[..., None]) * inverse[..., None]).round().clamp(0, 15)
    code = code.to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale, minimum


def _widen_plain(codes, scale, minimum):
    code = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).float()
    return (code.unflatten(-1, (-1, GROUP)) * scale.float()[..., None] + minimum.float()[..., None]).flatten(-2)


class _PlainCache:
    def __init__(self, b, hk, length, d):
        self.k = self._empty(b, hk, length, d)
        self.v = self._empty(b, hk, length, d)

    @staticmethod
    def _empty(b, hk, length, d):
        return [torch.zeros(b, hk, length, d // 2, dtype=torch.uint8, device=DEVICE),
                torch.zeros(b, hk, length, d // GROUP, dtype=torch.float16, device=DEVICE),
                torch.zeros(b, hk, length, d // GROUP, dtype=torch.float16, device=DEVICE)]

    def append(self, k, v, spans):
        """Sequence i's first m rows of k, v to its positions n - m .. n."""
        for store, x in ((self.k, k), (self.v, v)):
            for i, (n, m) in enumerate(spans):
                for part, value in zip(store, _quantize_plain(x[i, :, :m])):
                    part[i, :, n - m:n] = value

    def sequence(self, i, n):
        return (_widen_plain(*(p[i, :, :n] for p in self.k)), _widen_plain(*(p[i, :, :n] for p in self.v)))


def _attend_plain(q, k, v, n, m, window, sinks, scale, out):
    """One sequence in fp32: q [Hq, T, D], k, v [Hk, >= n, D] -> out[:, :m]."""
    hq, _, d = q.shape
    hk = k.shape[0]
    block = max(16, min(1024, (1 << 28) // (hq * max(1, n))))
    for t0 in range(0, m, block):
        t1 = min(m, t0 + block)
        p = torch.arange(n - m + t0, n - m + t1, device=q.device)
        first, last = n - m + t0, n - m + t1
        lo = max(0, first - window + 1) if window else 0
        keep = min(sinks, lo)
        j = torch.arange(lo, last, device=q.device)
        kk, vv = k[:, lo:last], v[:, lo:last]
        if keep:
            j = torch.cat((torch.arange(keep, device=q.device), j))
            kk, vv = torch.cat((k[:, :keep], kk), 1), torch.cat((v[:, :keep], vv), 1)
        kk, vv = kk.float(), vv.float()
        mask = j[None, :] <= p[:, None]
        if window:
            mask = mask & ((j[None, :] > p[:, None] - window) | (j[None, :] < sinks))
        qq = q[:, t0:t1].float().reshape(hk, hq // hk, t1 - t0, d)
        s = torch.matmul(qq.flatten(1, 2), kk.transpose(1, 2).contiguous()) * scale
        s = s.view(hk, hq // hk, t1 - t0, -1).masked_fill(~mask, float("-inf"))
        e = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(e.flatten(1, 2), vv).view(hk, hq // hk, t1 - t0, d) / e.sum(-1, keepdim=True)
        out[:, t0:t1] = o.reshape(hq, t1 - t0, d).to(out.dtype)


# ------------------------------------------------------------------ the cases' state and passes
def prepare(case, seed):
    q, k, v = _inputs(case, seed)
    spans = _spans(case)
    b, hk, length, d = k.shape
    state = {"case": case, "spans": spans}
    dtype = k.dtype
    lengths = torch.tensor([n for n, _ in spans], dtype=torch.int32, device=DEVICE)
    counts = torch.tensor([m for _, m in spans], dtype=torch.int32, device=DEVICE)
    state.update(lengths=lengths, counts=counts, start=lengths - counts)
    if q is not None:
        state.update(q=q, out=torch.zeros(b, case["tokens"], case["heads"], d, dtype=dtype,
                                          device=DEVICE).transpose(1, 2))
    if case["op"] == "window":
        state.update(k=k, v=v)
        return state
    # the new tokens' rows, as the projections give them
    t = case["tokens"]
    new_k, new_v = (torch.empty(b, t, hk, d, dtype=dtype, device=DEVICE).transpose(1, 2) for _ in range(2))
    for i, (n, m) in enumerate(spans):
        for dst, src in ((new_k, k), (new_v, v)):
            dst[i, :, :m] = src[i, :, n - m:n]
            dst[i, :, m:] = 0
    state.update(new_k=new_k, new_v=new_v)
    if own:
        from marlin_style_fluxbin_amd import Int4KVCache

        cache = Int4KVCache(b, hk, length, d, device=DEVICE)
        if case["op"] == "kv4":
            cache.append(k, v, 0, counts=lengths)
    else:
        cache = _PlainCache(b, hk, length, d)
        if case["op"] == "kv4":
            cache.append(k, v, [(n, n) for n, _ in spans])
    state["cache"] = cache
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from marlin_style_fluxbin_amd import kv4_attention, window_attention

    case = state["case"]
    ragged = {"query_lengths": state["counts"]} if case["ragged"] else {}
    mask = {} if case["op"] == "append" else {"window": case["window"] or None, "sinks": case["sinks"]}
    if case["op"] == "window":
        return window_attention(state["q"], state["k"], state["v"], lengths=state["lengths"], out=state["out"],
                                **mask, **ragged)
    cache = state["cache"]
    if case["op"] == "append":
        cache.append(state["new_k"], state["new_v"], state["start"], counts=state["counts"])
        return cache.restore(dtype=state["new_k"].dtype)
    if case["append"]:
        cache.append(state["new_k"], state["new_v"], state["start"], counts=state["counts"])
    return kv4_attention(state["q"], cache, lengths=state["lengths"], out=state["out"], **mask, **ragged)


def _run_plain(state):
    case, spans = state["case"], state["spans"]
    if case["op"] != "window" and (case["op"] == "append" or case["append"]):
        state["cache"].append(state["new_k"], state["new_v"], spans)
    if case["op"] == "append":
        dtype = state["new_k"].dtype
        return tuple(_widen_plain(*part).to(dtype) for part in (state["cache"].k, state["cache"].v))
    out = state["out"]
    for i, (n, m) in enumerate(spans):
        k, v = (state["k"][i], state["v"][i]) if case["op"] == "window" else state["cache"].sequence(i, n)
        _attend_plain(state["q"][i], k, v, n, m, case["window"], case["sinks"], 1 / math.sqrt(case["dim"]), out[i])
    return out


# ------------------------------------------------------------------ 64 bits
def _stands_for(x):
    """The 64-bit value that each element's 4-bit group holds for it; the stored scale and
    minimum are rounded as the format says, the rest is exact."""
    x = x.to(torch.float64)
    shape = x.shape
    x = x.reshape(*shape[:-1], shape[-1] // GROUP, GROUP)
    lo, hi = torch.aminmax(x, dim=-1, keepdim=True)
    minimum = lo.to(torch.float32).to(torch.float16).to(torch.float64)
    step = (hi - lo).to(torch.float32) * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)
    step = step.to(torch.float16)
    safe = torch.where(step > 0, step, torch.ones_like(step)).to(torch.float32)
    quotient = (x - minimum).to(torch.float32) * (1 / safe)
    code = torch.clamp(torch.round(quotient.to(torch.float64)), 0, 15)
    code = torch.where(step > 0, code, torch.zeros_like(code))
    return (code * step.to(torch.float64) + minimum).reshape(shape)


def exact(case, seed):
    cost = work(case)
    if cost["flops"] > 5e12 or cost["bytes"] > 8e9:
        return None
    q, k, v = _inputs(case, seed)
    spans = _spans(case)
    d = case["dim"]
    if case["op"] == "append":
        results = []
        for x in (k, v):
            y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
            for i, (n, m) in enumerate(spans):
                y[i, :, n - m:n] = _stands_for(x[i, :, n - m:n])
            results.append(y)
        return tuple(results)
    group = case["heads"] // case["kv_heads"]
    result = torch.zeros(case["batch"], case["heads"], case["tokens"], d, dtype=torch.float64, device=q.device)
    for i, (n, m) in enumerate(spans):
        position = torch.arange(n - m, n, device=q.device)
        for h in range(case["heads"]):
            kh, vh = k[i, h // group, :n], v[i, h // group, :n]
            if case["op"] == "kv4":
                kh, vh = _stands_for(kh), _stands_for(vh)
            kh, vh = kh.to(torch.float64), vh.to(torch.float64)
            rows = max(1, (1 << 25) // n)
            for t0 in range(0, m, rows):
                p = position[t0:t0 + rows, None]
                key = torch.arange(n, device=q.device)[None, :]
                hidden = key > p
                if case["window"]:
                    hidden |= (key <= p - case["window"]) & (key >= case["sinks"])
                logit = q[i, h, t0:min(t0 + rows, m)].to(torch.float64) @ kh.t() / math.sqrt(d)
                logit[hidden] = -math.inf
                result[i, h, t0:min(t0 + rows, m)] = torch.softmax(logit, dim=-1) @ vh
    return result
