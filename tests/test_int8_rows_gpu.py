"""Rows quantized to 8 bits (as they are, normalised, SwiGLU) against the definition in 64 bits.

Bounds.  Rows as they are and normalised rows: codes equal (the products weight * s are exact in
fp32, the codes those of the exact quotient).  Scales: plain a / 127 is one fp32 division, equal;
normalised within 2^-19: a sum of K squares in fp32 takes at most 32 additions in a thread and 14
between threads (46 * 2^-24, halved by the root), the mean, eps, the root (1 ulp = 2 * 2^-24) and
three products and quotients 2^-24 each.  SwiGLU: exp (2 ulp), the sum, the quotient and the product
leave 2^-21 of a value, a and the quotient's own rounding as much again: a code is at most
1/2 + 127 * 2^-20 from the exact quotient, a scale within 2^-20.
"""
import pytest
import torch

from marlin_style_fluxbin_amd import (add_rms_norm_int8, dequantize_int8, quantize_int8, quantize_weight_int8,
                                      rms_norm_int8, silu_mul_int8)
from tests.int8_reference import HALVES, held, norm_rows, swiglu_rows

pytestmark = pytest.mark.gpu

EPS = 1e-6
# around every kernel's width: 512, 1024, 2048, 4096, 6144, 8192, 12288, 16384, and beyond
SHAPES = [(1, 1), (3, 7), (5, 8), (2, 63), (9, 512), (4, 513), (7, 1000), (5, 1024), (3, 1032), (2, 2047), (3, 2049),
          (4, 4096), (2, 4104), (2, 6144), (3, 6152), (3, 8192), (2, 8200), (300, 4090), (2, 12288), (2, 12296), (2, 16384),
          (2, 16392), (1, 40000)]


def states(rows, columns, dtype, gpu, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * rows + columns)
    x = torch.randn(rows, columns, generator=g) * torch.exp(0.5 * torch.randn(columns, generator=g))
    return x.to(dtype).to(gpu)


def same_scales(got, want, tolerance):
    assert got.dtype is torch.float32 and got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert bool(((got - want).abs()[fine].double() <= tolerance * want[fine].double() + 2.0**-149).all())


def assert_rows(got, p, exact_scale):
    codes, scales = held(p)
    assert got[0].dtype is torch.int8
    assert torch.equal(got[0].double(), codes)
    same_scales(got[1], scales, 0.0 if exact_scale else 2.0**-19)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_plain_rows(gpu, rows, columns, dtype):
    x = states(rows, columns, dtype, gpu)
    got = quantize_int8(x)
    codes, _ = held(x)
    assert torch.equal(got[0].double(), codes)
    # (in 64 bits first: torch divides floats on a GPU by multiplying with the reciprocal.  a / 127
    # repeats every seven bits, so it is near no midpoint of two floats and the second rounding adds none)
    assert torch.equal(got[1], (x.double().abs().amax(-1) / 127).float())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_norm_rows(gpu, rows, columns, dtype):
    x, r = states(rows, columns, dtype, gpu, 1), states(rows, columns, dtype, gpu, 2)
    w = (1 + 0.2 * torch.randn(columns, generator=torch.Generator().manual_seed(3))).to(dtype).to(gpu)
    for residual in (None, r):
        p, inverse, s = norm_rows(x, w, EPS, residual)
        if residual is None:
            got = rms_norm_int8(x, w, EPS)
        else:
            *got, total = add_rms_norm_int8(x, r, w, EPS)
            assert torch.equal(total, s)
        codes, _ = held(p)
        assert torch.equal(got[0].double(), codes)
        same_scales(got[1], held(p * inverse)[1], 2.0**-19)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_swiglu_rows(gpu, rows, columns, dtype):
    both = torch.cat([states(rows, columns, dtype, gpu, 4), states(rows, columns, dtype, gpu, 5)], 1)
    gate, up = both[:, :columns], both[:, columns:]
    codes, scales = silu_mul_int8(gate, up)
    p = swiglu_rows(gate, up)
    same_scales(scales, held(p)[1], 2.0**-20)
    quotient = p * 127 / p.abs().amax(-1, keepdim=True)
    assert float((codes.double() - quotient).abs().max()) <= 0.5 + 127 * 2.0**-20
    assert int(codes.abs().max()) == 127


@pytest.mark.parametrize("dtype", HALVES)
def test_borders_between_codes_go_to_the_even_one(gpu, dtype):
    """Quotients that are exact halves, and their neighbours in the type."""
    x = torch.zeros(64, 256, dtype=dtype)
    for i in range(64):
        # 127 * (k + 1/2) / 127: rows whose largest value is 127, 254, .. have exact halves
        top = 127.0 * 2.0 ** (i % 4 - 1)
        halves = (torch.arange(255) - 127 + 0.5) * top / 127
        x[i, 0] = top
        x[i, 1:] = halves.to(dtype)[:255] if i % 2 else (torch.randn(255, generator=torch.Generator().manual_seed(i)) * top / 4).to(dtype)
    x = x.to(gpu)
    assert_rows(quantize_int8(x), x.double(), True)
    w = (2.0 ** torch.randint(-3, 4, (256,), generator=torch.Generator().manual_seed(9))).to(dtype).to(gpu)
    got = rms_norm_int8(x, w, EPS)
    p, inverse, _ = norm_rows(x, w, EPS)
    assert torch.equal(got[0].double(), held(p)[0])


@pytest.mark.parametrize("columns", [40, 700, 3000, 9000, 20000])
def test_rows_that_a_float_does_not_hold(gpu, columns):
    """Zeros, subnormals, sums of squares beyond the floats, infinities and NaN, row by row among
    ordinary ones; a NaN or infinity in the last column alone."""
    base = states(12, columns, torch.bfloat16, "cpu", 7)
    base[1] = 0
    base[2] = (base[2].double() * 2.0**-120).to(torch.bfloat16)
    base[3] = (base[3].double() * 2.0**-133).to(torch.bfloat16)
    base[4] = (base[4].double() * 2.0**100).to(torch.bfloat16)
    base[5, -1] = float("nan")
    base[6, -1] = float("inf")
    base[7, 0] = float("-inf")
    base[8, columns // 2] = float("nan")
    base[9] = -0.0
    base[10] = float("nan")
    x = base.to(gpu)
    codes, scales = quantize_int8(x)
    want, want_scales = held(x)
    assert torch.equal(codes.double(), want)
    same_scales(scales, want_scales, 2.0**-23)
    w = (1 + 0.2 * torch.randn(columns, generator=torch.Generator().manual_seed(3))).bfloat16().to(gpu)
    for eps in (EPS, 0.0):
        p, inverse, _ = norm_rows(x, w, eps)
        codes, scales = rms_norm_int8(x, w, eps)
        inverse = torch.where(torch.isfinite(inverse), inverse, torch.zeros_like(inverse))  # eps 0, a row of zeros
        want, want_scales = held(torch.where(torch.isfinite(p).all(-1, keepdim=True), p, torch.nan) * inverse)
        assert torch.equal(codes.double(), held(p)[0])
        same_scales(scales, want_scales, 2.0**-19)
    residual = x.clone()
    residual[11, 0] = 2.0**127
    codes, scales, total = add_rms_norm_int8(x, residual, w, EPS)
    p, inverse, s = norm_rows(x, w, EPS, residual)
    assert torch.equal(total.view(torch.int16)[~torch.isnan(s)], s.view(torch.int16)[~torch.isnan(s)])
    assert torch.equal(torch.isnan(total), torch.isnan(s))
    assert torch.equal(codes.double(), held(p)[0])
    gate = base.clone()
    gate[4] = (gate[4].double() * 2.0**-90).to(torch.bfloat16)
    gate[11] = -90 - gate[11].abs()  # every product below the floats that a quotient takes
    gate = gate.to(gpu)
    up = states(12, columns, torch.bfloat16, gpu, 8)
    codes, scales = silu_mul_int8(gate, up)
    p = swiglu_rows(gate, up)
    want, want_scales = held(p)
    same_scales(scales, want_scales, 2.0**-20)
    assert int((codes.double() - want).abs().max()) <= 1
    good = torch.isfinite(want_scales)
    quotient = torch.where(p.abs().amax(-1, keepdim=True) > 0, p * 127 / p.abs().amax(-1, keepdim=True), torch.zeros_like(p))
    assert float((codes.double() - quotient)[good].abs().max()) <= 0.5 + 127 * 2.0**-20
    assert not bool(codes[~good].any())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("columns", [33, 64, 1000, 4096])
def test_strides_and_alignment(gpu, columns, dtype):
    """Rows at odd addresses, far apart, transposed, broadcast; leading shapes; outputs in place and
    in the caller's memory, which is not written beside the rows."""
    wide = states(6, columns + 37, dtype, gpu, 11)
    w = (1 + 0.2 * torch.randn(columns, generator=torch.Generator().manual_seed(3))).to(dtype).to(gpu)
    views = [wide[:, 1:1 + columns], wide[:, 8:8 + columns], wide[::2, 3:3 + columns], wide[:1, 5:5 + columns].expand(4, columns),
             wide[:, :columns].t().contiguous().t(), wide[:, 5:5 + columns].reshape(2, 3, columns),
             wide[:, 5:5 + columns].unflatten(0, (2, 3))[:, :2], wide[0, :columns], wide[:0, :columns]]
    for x in views:
        codes, scales = quantize_int8(x)
        assert codes.shape == x.shape and scales.shape == x.shape[:-1]
        if x.numel():
            assert torch.equal(codes.double(), held(x)[0])
        codes, scales, total = add_rms_norm_int8(x, x, w, EPS)
        p, inverse, s = norm_rows(x, w, EPS, x)
        assert torch.equal(total, s)
        if x.numel():
            assert torch.equal(codes.double(), held(p)[0])
    x = wide[:, 3:3 + columns]
    store = torch.full((6, columns + 9), 99, dtype=torch.int8, device=gpu)
    marks = torch.full((8,), 7.0, device=gpu)
    got = quantize_int8(x, out=(store[:, 5:5 + columns], marks[1:7]))
    assert got[0].data_ptr() == store[:, 5:5 + columns].data_ptr()
    assert torch.equal(got[0].double(), held(x)[0])
    assert bool((store[:, :5] == 99).all()) and bool((store[:, 5 + columns:] == 99).all())
    assert float(marks[0]) == float(marks[7]) == 7.0
    for which in range(3):  # the sum over one of its terms, or beside other memory
        a, r = states(6, columns, dtype, gpu, 20), states(6, columns, dtype, gpu, 21)
        p, inverse, s = norm_rows(a, w, EPS, r)
        target = (a, r, wide[:, 1:1 + columns])[which]
        before = wide.clone()
        codes, scales, total = add_rms_norm_int8(a, r, w, EPS, residual_out=target)
        assert total is target and torch.equal(total, s) and torch.equal(codes.double(), held(p)[0])
        assert torch.equal(wide[:, :1], before[:, :1]) and torch.equal(wide[:, 1 + columns:], before[:, 1 + columns:])


@pytest.mark.parametrize("dtype", HALVES + (torch.float32,))
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 15), (5, 16), (4, 100), (7, 4096), (0, 8)])
def test_dequantize(gpu, rows, columns, dtype):
    g = torch.Generator().manual_seed(rows + columns)
    codes = torch.randint(-128, 128, (rows, columns + 3), generator=g).to(torch.int8).to(gpu)
    scales = torch.rand(rows, generator=g).to(gpu)
    for view in (codes[:, :columns].contiguous(), codes[:, 2:2 + columns], codes[:, :columns].t().contiguous().t()):
        got = dequantize_int8(view, scales, dtype=dtype)
        assert torch.equal(got, (view.float() * scales[:, None]).to(dtype))


def test_a_quantized_row_is_within_half_a_step(gpu):
    x = states(64, 4096, torch.bfloat16, gpu, 12)
    codes, scales = quantize_int8(x)
    back = dequantize_int8(codes, scales, dtype=torch.float32)
    assert bool(((back.double() - x.double()).abs() <= scales.double()[:, None] * (0.5 + 1e-4)).all())


def test_many_rows(gpu):
    """More rows than workgroups run at once, every one of them."""
    x = states(20000, 136, torch.bfloat16, gpu, 13)
    assert_rows(quantize_int8(x), x.double(), True)


def test_refusals(gpu):
    x = states(4, 64, torch.bfloat16, gpu)
    w = torch.ones(64, dtype=torch.bfloat16, device=gpu)
    codes, scales = quantize_int8(x)
    bad = [
        (lambda: quantize_int8(x.float()), "fp16 or bf16"), (lambda: quantize_int8(x[:, :0]), "columns to hold"),
        (lambda: quantize_int8(x[0, 0]), "columns to hold"), (lambda: rms_norm_int8(x, w[:63], EPS), "weight must"),
        (lambda: rms_norm_int8(x, w.half(), EPS), "weight must"), (lambda: rms_norm_int8(x, w.cpu(), EPS), "weight must"),
        (lambda: add_rms_norm_int8(x, x[:3], w, EPS), "residual must"),
        (lambda: add_rms_norm_int8(x, None, w, EPS), "residual must"),
        (lambda: add_rms_norm_int8(x, x.half(), w, EPS), "residual must"),
        (lambda: add_rms_norm_int8(x, x, w, EPS, residual_out=x[:3]), "residual_out must"),
        (lambda: add_rms_norm_int8(x, x, w, EPS, residual_out=x[:1].expand(4, 64)), "residual_out must"),
        (lambda: silu_mul_int8(x, x[:, :63]), "up must"), (lambda: silu_mul_int8(x, x.cpu()), "GPU|up must"),
        (lambda: quantize_int8(x, out=(codes[:3], scales)), "out's codes"),
        (lambda: quantize_int8(x, out=(codes, scales[:3])), "out's scales"),
        (lambda: quantize_int8(x, out=(codes[:1].expand(4, 64), scales)), "out's codes"),
        (lambda: quantize_int8(x, out=(codes, scales.double())), "out's scales"),
        (lambda: dequantize_int8(codes.short(), scales), "int8"), (lambda: dequantize_int8(codes, scales[:2]), "fp32, one"),
        (lambda: dequantize_int8(codes, scales, dtype=torch.float64), "dtype must"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(RuntimeError, match="eps"):
        rms_norm_int8(x, w, -1.0)
    with pytest.raises(ValueError, match="no backward"):
        quantize_int8(x.clone().requires_grad_())
    with torch.no_grad():
        quantize_int8(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(lambda t: quantize_int8(t)[0], (x,), check_trace=False)


def test_streams_and_graphs(gpu):
    """A call on another stream, and one captured and replayed on new contents among other work."""
    x, r = states(70, 1000, torch.float16, gpu, 14), states(70, 1000, torch.float16, gpu, 15)
    w = (1 + 0.2 * torch.randn(1000, generator=torch.Generator().manual_seed(3))).half().to(gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = add_rms_norm_int8(x, r, w, EPS)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0].double(), held(norm_rows(x, w, EPS, r)[0])[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        codes, scales, total = add_rms_norm_int8(x, r, w, EPS)
        act = silu_mul_int8(total[:, :500], total[:, 500:])
    for seed in range(3):
        x.copy_(states(70, 1000, torch.float16, gpu, 50 + seed))
        graph.replay()
        eager = add_rms_norm_int8(x, r, w, EPS)
        act_eager = silu_mul_int8(eager[2][:, :500], eager[2][:, 500:])
        torch.cuda.synchronize()
        assert torch.equal(codes, eager[0]) and torch.equal(scales, eager[1]) and torch.equal(total, eager[2])
        assert torch.equal(act[0], act_eager[0]) and torch.equal(act[1], act_eager[1])


def test_a_weight_that_is_not_finite_is_refused(gpu):
    """As on the CPU: no channel becomes NaN without a word."""
    weight = torch.randn(5, 48, device=gpu, dtype=torch.bfloat16)
    weight[3, 7] = float("nan")
    with pytest.raises(ValueError, match="finite"):
        quantize_weight_int8(weight)
    weight[3, 7] = 0
    codes, scales = quantize_weight_int8(weight)
    assert torch.equal(codes, quantize_int8(weight)[0]) and torch.equal(scales, quantize_int8(weight)[1])
