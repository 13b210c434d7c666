"""The 8-bit operators from their definitions in 64 bits, and the bounds that their roundings allow."""
import torch

HALVES = (torch.bfloat16, torch.float16)


def held(p):
    """Rows of float64 values as (codes, scales): float64 codes, fp32 scales; a row with an infinity
    or NaN has codes 0 and a NaN scale."""
    p = p.double()
    top = p.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(p).all(-1, keepdim=True)
    codes = torch.where(top > 0, torch.round(p * 127 / top), torch.zeros_like(p))
    codes = torch.where(bad, torch.zeros_like(codes), codes)
    scales = torch.where(bad, torch.full_like(top, float("nan")), top / 127)
    return codes, scales[..., 0].float()


def norm_rows(x, weight, eps, residual=None):
    """The unquantized rows of the norm and the stored sum."""
    s = x if residual is None else x + residual  # one rounding, the type's own addition
    wide = s.double()
    inverse = 1 / torch.sqrt(wide.square().mean(-1, keepdim=True) + eps)
    return weight.double() * wide, inverse, s


def swiglu_rows(gate, up):
    g = gate.double()
    return g / (1 + torch.exp(-g)) * up.double()


def product(a, a_scales, w, w_scales, bias=None):
    """(the value, the magnitude that fp32 roundings are relative to), both float64."""
    y = torch.matmul(a.double(), w.double().t().contiguous())
    y = y * a_scales.double()[..., None] * w_scales.double()
    size = y.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def product_bound(y, size, dtype):
    """The sum's float, two products and the last addition round once each in fp32 (2^-24 of `size`
    each, and of what those before left: four cover them with their second order), then once to
    the type (half its eps of the value; half its least step near zero)."""
    info = torch.finfo(dtype)
    last = 0.0 if dtype is torch.float32 else info.eps / 2
    least = 2.0**-150 if dtype is not torch.float16 else 2.0**-25
    return size * (4 * 2.0**-24) * (1 + last) + y.abs() * last + least


def assert_product(got, a, a_scales, w, w_scales, bias=None, context=""):
    y, size = product(a, a_scales, w, w_scales, bias)
    top = torch.finfo(got.dtype).max
    bound = product_bound(y, size, got.dtype)
    finite = y.abs() + bound < top
    wrong = (got.double() - y).abs() > bound
    assert not bool((wrong & finite).any()), (context, float(((got.double() - y).abs() / bound)[finite].max()))
    assert torch.equal(torch.isnan(got.double()), torch.isnan(y)), context
