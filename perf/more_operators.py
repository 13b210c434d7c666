"""Products in 8-bit integers and the operators that feed them, as cases that can be timed and checked.

Four kinds of work, each through the framework's public entry points:

* ``norm``: ``rms_norm_int8`` / ``add_rms_norm_int8``: RMSNorm (after the residual's addition) whose
  output is 8-bit codes with a scale per row; read back by ``dequantize_int8``.
* ``linear``: ``PackedInt8Linear``: the rows quantized (``quantize_int8``), then ``int8_matmul``.
* ``matmul``: ``int8_matmul`` on codes that are there already (several Linears read one input).
* ``mlp``: a decoder layer's MLP: ``add_rms_norm_int8``, the gate|up product, ``silu_mul_int8``, the
  down product.

The arithmetic.  A row p of K values is held as codes = round(127 p / a), ties to even, and the scale
a / 127, a = max|p|.  The norm has s = x, or x + residual rounded to its type, p = weight s
/ sqrt(mean(s^2) + eps); SwiGLU p = gate / (1 + exp(-gate)) up.  The product is
(sum_k a[m, k] w[n, k]) a_scale[m] w_scale[n] + bias[n], the sum in whole numbers.
"""
from __future__ import annotations

import math

import torch

own = False  # False: the plain forms below; True: the framework's operators

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # a decode step's norm of one token behind the residual: latency is what it costs
        {"name": "norm_step", "op": "norm", "dtype": "bf16", "rows": 1, "hidden": 4096, "residual": True},
        # the norm of a long prompt
        {"name": "norm_prompt", "op": "norm", "dtype": "bf16", "rows": 8192, "hidden": 4096, "residual": True},
        # an odd batch of an odd width, without a residual
        {"name": "norm_odd", "op": "norm", "dtype": "f16", "rows": 1001, "hidden": 2077, "residual": False},
        # an attention output through o_proj for one token: the smallest product
        {"name": "linear_step", "op": "linear", "dtype": "bf16", "rows": 1, "in": 4096, "out": 4096, "bias": False},
        # the same Linear on a prompt, with a bias
        {"name": "linear_prompt", "op": "linear", "dtype": "bf16", "rows": 2048, "in": 4096, "out": 4096, "bias": True},
        # an odd Linear on a padded batch
        {"name": "linear_odd", "op": "linear", "dtype": "f16", "rows": 301, "in": 2000, "out": 1001, "bias": True},
        # a serving batch's q|k|v on codes that the norm left
        {"name": "matmul_batch", "op": "matmul", "dtype": "bf16", "rows": 24, "in": 4096, "out": 6144, "bias": False},
        # a chunk of a prompt through the down projection: a long sum
        {"name": "matmul_chunk", "op": "matmul", "dtype": "f16", "rows": 512, "in": 12288, "out": 4096, "bias": False},
        # the largest single product: a long prompt through one gate projection
        {"name": "matmul_prompt", "op": "matmul", "dtype": "bf16", "rows": 8192, "in": 4096, "out": 12288,
         "bias": False},
        # the MLP of a decode step
        {"name": "mlp_step", "op": "mlp", "dtype": "bf16", "rows": 1, "hidden": 4096, "inter": 12288},
        # the MLP of a batch of sequences with a few drafted tokens each
        {"name": "mlp_batch", "op": "mlp", "dtype": "bf16", "rows": 48, "hidden": 4096, "inter": 12288},
        # the MLP of a prompt: the largest
        {"name": "mlp_prompt", "op": "mlp", "dtype": "bf16", "rows": 4096, "hidden": 4096, "inter": 12288},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, hi):
    """A Linear's width: mostly whole groups of 128, some odd."""
    n = _log_int(rng, 32, hi)
    return n if rng.random() < 0.25 else max(16, n // 16 * 16) if n < 512 else n // 128 * 128


def draw(rng):
    """One more case: one token to a prompt, any width, both types; bounded by the largest listed work."""
    limit = [work(c) for c in listed()]
    max_bytes, max_flops = max(w["bytes"] for w in limit), max(w["flops"] for w in limit)
    op = rng.choice(["norm", "linear", "matmul", "matmul", "mlp"])
    case = {"op": op, "dtype": rng.choice(["bf16", "f16"]),
            "rows": rng.choice([1, _log_int(rng, 1, 64), _log_int(rng, 1, 8192), _log_int(rng, 1, 8192)])}
    if op == "norm":
        case.update(hidden=_width(rng, 16384), residual=rng.random() < 0.6)
    elif op == "mlp":
        case.update(hidden=_width(rng, 8192), inter=_width(rng, 16384))
    else:
        case.update({"in": _width(rng, 16384), "out": _width(rng, 16384), "bias": rng.random() < 0.4})
    while True:
        cost = work(case)
        if cost["bytes"] <= max_bytes and cost["flops"] <= max_flops:
            return case
        case["rows"] = max(1, case["rows"] // 2)


def work(case):
    m = case["rows"]
    if case["op"] == "norm":
        h = case["hidden"]
        # x (and the residual in and out), the norm's weight; codes and scales written, read again, widened
        return {"bytes": m * h * (2 + 4 * case["residual"]) + 2 * h + 2 * (m * h + 4 * m) + 2 * m * h,
                "flops": m * h * (6 + case["residual"])}
    if case["op"] == "mlp":
        h, i = case["hidden"], case["inter"]
        # x, the residual in and out, the weights; y.  What lies between fits no user's eye
        return {"bytes": 6 * m * h + 2 * h + 3 * h * i + 4 * (2 * i + h) + 2 * m * h, "flops": 6 * m * h * i}
    k, n = case["in"], case["out"]
    codes = m * k + 4 * m if case["op"] == "matmul" else 2 * m * k
    return {"bytes": codes + n * k + 4 * n + 2 * n * case["bias"] + 2 * m * n, "flops": 2 * m * n * k}


def _inputs(case, seed):
    """Tensors of the case: hidden states with a few strong channels, weights as they are trained."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)

    def states(rows, width):
        channel = torch.exp(0.4 * normal(width))
        channel[:: max(1, width // 7)] *= 6.0
        return (normal(rows, width) * channel).to(dtype)

    def weight(out, width):
        """A Linear's weight quantized per output channel, as a checkpoint holds it."""
        w = normal(out, width) * 0.02 * torch.exp(0.2 * normal(out, 1))
        scale = w.abs().amax(1) / 127
        return torch.round(w / scale[:, None]).to(torch.int8), scale

    made = {}
    if case["op"] in ("norm", "mlp"):
        h = case["hidden"]
        made.update(x=states(case["rows"], h), norm=(1 + 0.1 * normal(h)).to(dtype))
        if case.get("residual", True):
            made["residual"] = states(case["rows"], h)
        if case["op"] == "mlp":
            made["gate_up"], made["gate_up_scales"] = weight(2 * case["inter"], h)
            made["down"], made["down_scales"] = weight(h, case["inter"])
        return made
    x = states(case["rows"], case["in"])
    made["weight"], made["weight_scales"] = weight(case["out"], case["in"])
    if case["bias"]:
        made["bias"] = (0.5 * normal(case["out"])).to(dtype)
    if case["op"] == "linear":
        made["x"] = x
    else:
        x = x.float()
        made["scales"] = x.abs().amax(1) / 127
        made["codes"] = torch.round(x / made["scales"][:, None]).to(torch.int8)
    return made


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own and case["op"] == "linear":
        from marlin_style_fluxbin_amd import PackedInt8Linear

        state["linear"] = PackedInt8Linear(state["weight"], state["weight_scales"], bias=state.get("bias"))
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ the framework's calls
def _run_own(state):
    from marlin_style_fluxbin_amd import (add_rms_norm_int8, dequantize_int8, int8_matmul, rms_norm_int8,
                                          silu_mul_int8)

    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    with torch.no_grad():
        if case["op"] == "linear":
            return state["linear"](state["x"])
        if case["op"] == "matmul":
            return int8_matmul(state["codes"], state["scales"], state["weight"], state["weight_scales"],
                               bias=state.get("bias"), dtype=dtype)
        if case["op"] == "norm" and not case["residual"]:
            codes, scales = rms_norm_int8(state["x"], state["norm"], EPS)
            return dequantize_int8(codes, scales, dtype=dtype)
        codes, scales, stream = add_rms_norm_int8(state["x"], state["residual"], state["norm"], EPS)
        if case["op"] == "norm":
            return dequantize_int8(codes, scales, dtype=dtype), stream
        both = int8_matmul(codes, scales, state["gate_up"], state["gate_up_scales"], dtype=dtype)
        codes, scales = silu_mul_int8(both[:, :case["inter"]], both[:, case["inter"]:])
        return int8_matmul(codes, scales, state["down"], state["down_scales"], dtype=dtype), stream


# ------------------------------------------------------------------ plain forms
def _quantize_plain(p):
    """fp32 [M, K] -> whole fp32 values, fp32 scales [M, 1]."""
    top = p.abs().amax(1, keepdim=True)
    return torch.round(p * 127 / top.clamp_min(1e-30)), top / 127


def _matmul_plain(codes, scales, weight, weight_scales, bias, dtype):
    # (partial sums of such codes stay below 2^24, where fp32 holds every whole number)
    y = torch.mm(codes.float(), weight.float().t()) * scales.view(-1, 1) * weight_scales
    return (y if bias is None else y + bias.float()).to(dtype)


def _norm_plain(state, dtype):
    s = state["x"].float()
    if "residual" in state:
        s = (s + state["residual"].float()).to(dtype).float()
    p = s * torch.rsqrt(s.square().mean(1, keepdim=True) + EPS) * state["norm"].float()
    return (*_quantize_plain(p), s.to(dtype))


def _run_plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        return _matmul_plain(*_quantize_plain(state["x"].float()), state["weight"], state["weight_scales"],
                             state.get("bias"), dtype)
    if case["op"] == "matmul":
        return _matmul_plain(state["codes"], state["scales"], state["weight"], state["weight_scales"],
                             state.get("bias"), dtype)
    codes, scales, stream = _norm_plain(state, dtype)
    if case["op"] == "norm":
        values = (codes * scales).to(dtype)
        return (values, stream) if case["residual"] else values
    both = _matmul_plain(codes, scales, state["gate_up"], state["gate_up_scales"], None, dtype).float()
    gate, up = both[:, :case["inter"]], both[:, case["inter"]:]
    codes, scales = _quantize_plain(gate / (1 + torch.exp(-gate)) * up)
    return _matmul_plain(codes, scales, state["down"], state["down_scales"], None, dtype), stream


# ------------------------------------------------------------------ 64 bits
def _held(p):
    """(whole values, scales) of each row of float64 p."""
    step = torch.linalg.vector_norm(p, ord=math.inf, dim=-1, keepdim=True) / 127
    quotient = torch.where(step > 0, p / step, torch.zeros_like(p))
    return torch.round(quotient), step


def exact(case, seed):
    t = _inputs(case, seed)
    d64 = torch.float64
    dtype = DTYPES[case["dtype"]]

    def product(code, step, weight, weight_scales, bias=None):
        y = (code @ weight.to(d64).T.contiguous()) * step * weight_scales.to(d64)[None, :]
        return y if bias is None else y + bias.to(d64)[None, :]

    if case["op"] == "linear":
        return product(*_held(t["x"].to(d64)), t["weight"], t["weight_scales"], t.get("bias"))
    if case["op"] == "matmul":
        return product(t["codes"].to(d64), t["scales"].to(d64)[:, None], t["weight"], t["weight_scales"],
                       t.get("bias"))
    stream = t["x"].to(d64)
    if "residual" in t:
        stream = (stream + t["residual"].to(d64)).to(dtype).to(d64)  # what is stored
    power = (stream * stream).sum(-1, keepdim=True) / case["hidden"]
    code, step = _held(t["norm"].to(d64) * stream / torch.sqrt(power + EPS))
    if case["op"] == "norm":
        return (code * step, stream) if case["residual"] else code * step
    both = product(code, step, t["gate_up"], t["gate_up_scales"]).to(dtype).to(d64)  # what is stored
    gate, up = both.split(case["inter"], dim=-1)
    code, step = _held(gate * torch.sigmoid(gate) * up)
    return product(code, step, t["down"], t["down_scales"]), stream
