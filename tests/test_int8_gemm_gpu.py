"""``int8_matmul`` and ``PackedInt8Linear`` against the product in 64 bits (bounds: int8_reference)."""
import pytest
import torch
from torch import nn

from marlin_style_fluxbin_amd import (PackedInt8Linear, add_rms_norm_int8, int8_matmul, quantize_int8, silu_mul_int8)
from tests.int8_reference import HALVES, assert_product, held, norm_rows, product_bound, swiglu_rows

pytestmark = pytest.mark.gpu
ALL = HALVES + (torch.float32,)


def codes(rows, columns, gpu, seed, low=-128, high=128):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.randint(low, high, (rows, columns), generator=g, device=gpu, dtype=torch.int32).to(torch.int8)


def scales(rows, gpu, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.rand(rows, generator=g, device=gpu) * 0.01 + 1e-4


def case(m, n, k, gpu, dtype=torch.bfloat16, bias=False, seed=0):
    made = [codes(m, k, gpu, seed), scales(m, gpu, seed + 1), codes(n, k, gpu, seed + 2), scales(n, gpu, seed + 3)]
    b = torch.randn(n, generator=torch.Generator(device=gpu).manual_seed(seed + 4), device=gpu).to(dtype) if bias else None
    return made, b


ROWS = [1, 2, 7, 16, 17, 31, 32, 33, 48, 49, 64, 65, 100, 128, 129, 200, 256, 257, 300, 513]
WIDTHS = [(1, 16), (15, 64), (16, 48), (64, 80), (100, 128), (257, 144), (1001, 1008), (640, 2000), (1024, 4096)]


@pytest.mark.parametrize("m", ROWS)
def test_products(gpu, m):
    for i, (n, k) in enumerate(WIDTHS):
        dtype, bias = ALL[(m + i) % 3], (m + i) % 2 == 0
        args, b = case(m, n, k, gpu, dtype, bias, seed=m * 100 + i)
        got = int8_matmul(*args, bias=b, dtype=dtype)
        assert got.shape == (m, n) and got.dtype == dtype
        assert_product(got, *args, b, context=(m, n, k, dtype, bias))


@pytest.mark.parametrize("m,n,k", [(1, 6144, 4096), (1, 4096, 12288), (5, 24576, 4096), (24, 4096, 12288), (64, 512, 16384),
                                   (96, 300, 8192), (700, 1000, 5120), (1024, 2048, 4096), (2000, 4096, 1024),
                                   (4100, 1280, 256), (33, 12288, 512), (4000, 4100, 272), (2000, 4090, 528), (1000, 4001, 1040), (3, 64, 131056), (130, 64, 131056)])
def test_larger_products(gpu, m, n, k):
    args, b = case(m, n, k, gpu, torch.bfloat16, True, seed=7)
    assert_product(int8_matmul(*args, bias=b), *args, b, context=(m, n, k))


# every kernel, whole and in K splits (few rows: 16 and 32 rows by 16 and 32 columns, eight and sixteen
# waves, two and four pieces in flight; tiles of 64, 64 x 128, 128, 128 x 256 and 256), its last stage not whole
@pytest.mark.parametrize("m,n,k", [(16, 1000, 528), (9, 1000, 8208), (17, 17, 528), (17, 4097, 1040), (31, 8200, 1040),
                                   (200, 100, 48), (16, 6001, 4112), (90, 17, 12304), (200, 8200, 48), (1300, 1000, 8208),
                                   (90, 4097, 8208), (2050, 2049, 48), (260, 8200, 12304), (130, 6001, 8208),
                                   (1300, 6001, 48), (130, 8200, 16400), (9, 3001, 8208), (200, 8200, 528),
                                   (260, 4097, 8208), (390, 8200, 12304), (3, 300, 3712), (20, 100, 3712),
                                   (20, 5001, 3712), (7, 4000, 12288), (1, 4097, 12304), (40, 4097, 12304),
                                   (130, 6001, 12304), (2050, 4097, 48)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_every_kernel_and_split(gpu, m, n, k, dtype):
    args, b = case(m, n, k, gpu, dtype, True, seed=11)
    assert_product(int8_matmul(*args, bias=b, dtype=dtype), *args, b, context=(m, n, k))


@pytest.mark.parametrize("m", [1, 40, 300])
def test_sums_are_exact_at_their_largest(gpu, m):
    """Every product 2^14 or -127 * 128, as many of them as K may be; scales 1 and fp32 results."""
    k = 131056
    a = torch.full((m, k), -128, dtype=torch.int8, device=gpu)
    w = torch.full((80, k), -128, dtype=torch.int8, device=gpu)
    w[1] = 127
    w[2, : k // 2] = 127
    w[3] = 0
    w[3, -1] = 1
    one, ones = torch.ones(m, device=gpu), torch.ones(80, device=gpu)
    got = int8_matmul(a, one, w, ones, dtype=torch.float32)
    want = torch.matmul(a.double(), w.double().t().contiguous())
    assert torch.equal(got, want.float())


@pytest.mark.parametrize("m", [1, 3, 24, 70, 260])
def test_columns_behind_k_and_rows_behind_m_are_not_read_into_the_sum(gpu, m):
    """Views into larger arrays whose other elements are large; an output in the middle of others."""
    n, k = 200, 208
    store_a = torch.full((m + 2, 512), 127, dtype=torch.int8, device=gpu)
    store_w = torch.full((n + 3, 1024), 127, dtype=torch.int8, device=gpu)
    a, w = store_a[1:1 + m, 64:64 + k], store_w[2:2 + n, 160:160 + k]
    a.copy_(codes(m, k, gpu, 1))
    w.copy_(codes(n, k, gpu, 2))
    sa, sw = scales(m, gpu, 3), scales(n, gpu, 4)
    for dtype in ALL:
        for left in (0, 1, 8):
            out = torch.full((m + 2, n + 24), 5.0, dtype=dtype, device=gpu)
            view = out[1:1 + m, left:left + n]
            assert int8_matmul(a, sa, w, sw, dtype=dtype, out=view) is view
            assert_product(view, a, sa, w, sw, context=(m, dtype, left))
            out[1:1 + m, left:left + n] = 5
            assert bool((out == 5).all())


@pytest.mark.parametrize("m", [1, 3, 16, 17, 32, 33, 130, 300])
@pytest.mark.parametrize("k", [1, 15, 17, 64, 100, 2077, 4090, 8200, 12275])
def test_rows_at_any_address_and_of_any_length(gpu, m, k):
    """Odd K, odd strides and addresses, rows in reverse memory order, broadcast rows; large values around
    every row; an output at an odd address."""
    store = torch.full((m + 2, k + 21), 127, dtype=torch.int8, device=gpu)
    wide = torch.full((72, k + 7), 127, dtype=torch.int8, device=gpu)
    sa, sw = scales(m, gpu, 7), scales(70, gpu, 8)
    bias = torch.randn(70, generator=torch.Generator(device=gpu).manual_seed(9), device=gpu).half()
    for left, off in ((3, 1), (16, 2), (0, 0)):
        a, w = store[1:1 + m, left:left + k], wide[1:71, off:off + k]
        a.copy_(codes(m, k, gpu, left))
        w.copy_(codes(70, k, gpu, off + 50))
        out = torch.full((m, 73), 3.0, dtype=torch.float16, device=gpu)
        int8_matmul(a, sa, w, sw, bias=bias, dtype=torch.float16, out=out[:, 1:71])
        assert_product(out[:, 1:71], a, sa, w, sw, bias, context=(m, k, left))
        assert bool((out[:, 0] == 3).all()) and bool((out[:, 71:] == 3).all())
        aligned = torch.empty(70, -(-k // 16) * 16 + 16, dtype=torch.int8, device=gpu)[:, :k]
        aligned.copy_(w)
        assert torch.equal(int8_matmul(a, sa, aligned, sw), int8_matmul(a.contiguous(), sa, w.contiguous(), sw))
    a = codes(k, m, gpu, 5).t()  # columns far apart: copied by torch
    assert_product(int8_matmul(a, sa, w, sw), a, sa, w, sw)
    flat = codes(1, k, gpu, 6)
    assert torch.equal(int8_matmul(flat.expand(m, k), sa, w, sw), int8_matmul(flat.repeat(m, 1), sa, w, sw))


def test_rows_far_apart(gpu):
    """Strides beyond 2^22 bytes, read in place by few rows and copied for many; a weight of one row."""
    store = torch.zeros(70, (1 << 22) + 32, dtype=torch.int8, device=gpu)
    w = store[:, 16:16 + 256]
    w.copy_(codes(70, 256, gpu, 1))
    sw = scales(70, gpu, 2)
    for m in (3, 20, 100):
        a, sa = codes(m, 256, gpu, 3), scales(m, gpu, 4)
        assert_product(int8_matmul(a, sa, w, sw), a, sa, w, sw)
        assert_product(int8_matmul(a, sa, w[:1], sw[:1]), a, sa, w[:1], sw[:1])


def test_leading_axes_and_no_rows(gpu):
    args, _ = case(24, 70, 64, gpu)
    a, sa, w, sw = args
    flat = int8_matmul(a, sa, w, sw)
    assert torch.equal(int8_matmul(a.view(2, 3, 4, 64), sa.view(2, 3, 4), w, sw), flat.view(2, 3, 4, 70))
    assert torch.equal(int8_matmul(a[0], sa[0], w, sw), flat[0])
    assert int8_matmul(a[:0], sa[:0], w, sw).shape == (0, 70)
    one = a[:1].expand(24, 64)
    assert torch.equal(int8_matmul(one, sa, w, sw), int8_matmul(one.contiguous(), sa, w, sw))


@pytest.mark.parametrize("m", [1, 20, 100, 300])
def test_nan_rows_stay_in_their_row(gpu, m):
    (a, sa, w, sw), b = case(m, 130, 256, gpu, bias=True)
    sa[m // 2] = float("nan")
    sw[7] = float("inf")
    got = int8_matmul(a, sa, w, sw, bias=b)
    assert bool(torch.isnan(got[m // 2]).all())
    keep = [i for i in range(m) if i != m // 2]
    cols = [i for i in range(130) if i != 7]
    sub = got[keep][:, cols]
    if keep:
        assert_product(sub.contiguous(), a[keep], sa[keep], w[cols], sw[cols], b[cols])
        y = torch.matmul(a[keep].double(), w[7].double())
        assert torch.equal(got[keep, 7].double(), y * float("inf"))


def test_results_repeat(gpu):
    for m, n, k in ((1, 1000, 4096), (64, 256, 65536), (300, 500, 4096)):
        args, b = case(m, n, k, gpu, bias=True)
        first = int8_matmul(*args, bias=b)
        for _ in range(3):
            assert torch.equal(int8_matmul(*args, bias=b), first)


def test_refusals(gpu):
    (a, sa, w, sw), b = case(4, 32, 64, gpu, bias=True)
    bad = [
        (lambda: int8_matmul(a.short(), sa, w, sw), "a must be int8"), (lambda: int8_matmul(a, sa[:3], w, sw), "a_scales"),
        (lambda: int8_matmul(a, sa.half(), w, sw), "a_scales"), (lambda: int8_matmul(a, sa, w.t(), sw), "weight"),
        (lambda: int8_matmul(a, sa, w, sw[:5]), "weight_scales"), (lambda: int8_matmul(a, sa, w[None], sw[None]), "weight must"),
        (lambda: int8_matmul(a, sa, w, sw, bias=b[:3]), "bias must"),
        (lambda: int8_matmul(a, sa, w, sw, bias=b.half()), "bias must"),
        (lambda: int8_matmul(a, sa, w, sw, dtype=torch.float64), "dtype must"),
        (lambda: int8_matmul(a[:, :0], sa, w[:, :0], sw), "K must be"), (lambda: int8_matmul(a, sa, w[:0], sw[:0]), "N positive"),
        (lambda: int8_matmul(a, sa, w, sw, out=torch.empty(4, 31, dtype=torch.bfloat16, device=gpu)), "out must"),
        (lambda: int8_matmul(a, sa, w, sw, out=torch.empty(4, 32, device=gpu)), "out must"),
        (lambda: int8_matmul(a, sa, w, sw, out=torch.empty(1, 32, dtype=torch.bfloat16, device=gpu).expand(4, 32)), "out must"),
        (lambda: int8_matmul(a, sa, w, sw, out=torch.empty(32, 4, dtype=torch.bfloat16, device=gpu).t()), "out must"),
        (lambda: int8_matmul(a, sa.clone().requires_grad_(), w, sw), "no backward"),
        (lambda: quantize_int8(b[None], out=(w.view(-1)[:32].view(1, 32), sw[:1].clone().requires_grad_())), "no backward"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
    wide = torch.zeros(2, 131057, dtype=torch.int8, device=gpu)
    with pytest.raises(ValueError, match="K must be"):
        int8_matmul(wide, sa[:2], wide, sw[:2])


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (40, 300, 4096), (64, 256, 65536), (300, 512, 1024)])
def test_graphs_replay_on_new_contents(gpu, m, n, k):
    """Two captured calls (each with its own workspace) and eager work between the replays."""
    (a, sa, w, sw), b = case(m, n, k, gpu, bias=True)
    x = torch.randn(m, k, device=gpu).bfloat16()
    linear = PackedInt8Linear(w, sw, bias=b)
    with torch.no_grad():
        linear(x)
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first):
            y = int8_matmul(a, sa, w, sw, bias=b)
        with torch.cuda.graph(second):
            z = linear(x)
        for seed in range(3):
            a.copy_(codes(m, k, gpu, 90 + seed))
            x.copy_(torch.randn(m, k, device=gpu).bfloat16())
            first.replay()
            second.replay()
            assert_product(y, a, sa, w, sw, b)
            assert torch.equal(z, linear(x))
            torch.cuda.synchronize()


def test_two_streams_at_once(gpu):
    (a, sa, w, sw), _ = case(64, 256, 65536, gpu)
    (c, sc, v, sv), _ = case(64, 256, 65536, gpu, seed=50)
    want = int8_matmul(a, sa, w, sw), int8_matmul(c, sc, v, sv)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(streams[0]):
            one = int8_matmul(a, sa, w, sw)
        with torch.cuda.stream(streams[1]):
            two = int8_matmul(c, sc, v, sv)
        torch.cuda.synchronize()
        assert torch.equal(one, want[0]) and torch.equal(two, want[1])


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("out,width,bias", [(96, 64, True), (40, 77, True), (1024, 1000, False)])
def test_module(gpu, out, width, bias, dtype):
    g = torch.Generator().manual_seed(out)
    linear = nn.Linear(width, out, bias=bias).to(gpu, dtype)
    with torch.no_grad():
        linear.weight.copy_(torch.randn(out, width, generator=g).to(dtype))
        module = PackedInt8Linear.from_linear(linear)
        want, want_scales = held(linear.weight)
        assert torch.equal(module.codes[:, :width].double(), want) and torch.equal(module.scales, want_scales)
        for shape in ((1, width), (1, 1, width), (2, 9, width), (130, width), (0, width)):
            x = torch.randn(*shape, generator=g).to(dtype).to(gpu)
            y = module(x)
            assert y.shape == (*shape[:-1], out) and y.dtype == dtype
            if x.numel():
                a, sa = held(x)
                assert_product(y, a, sa, module.codes[:, :width], module.scales, linear.bias)
        assert module.route_counts == {"packed_m1": 2, "dense_fallback": 0, "packed_small_m": 3}
        x = torch.randn(1, 1, width, generator=g).to(dtype).to(gpu)
        eager = module(x)
        module.bind_prepared_decode(dtype)
        assert torch.equal(module(x), eager) and module(x).data_ptr() == module(x).data_ptr()
        with pytest.raises(ValueError, match="mismatch"):
            module(x[:, :, : width - 1])
        module.clear_prepared_decode()
        with pytest.raises(ValueError, match="fallback"):
            module(x.float())
        strided = torch.randn(4, width, 2, generator=g).to(dtype).to(gpu)[..., 0]
        assert torch.equal(module(strided), module(strided.contiguous()))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m", [1, 7, 48, 200])
def test_a_layers_mlp(gpu, m, dtype):
    """The operators together, as a decoder layer runs them, each against its definition on what the
    one before gave."""
    h, inter = 512, 1376
    g = torch.Generator().manual_seed(m)

    def half(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype).to(gpu)

    x, residual, w = half(m, h), half(m, h), 1 + half(h, scale=0.1)
    gate_up = PackedInt8Linear.from_linear(nn.Linear(h, 2 * inter, bias=False).to(gpu, dtype))
    down = PackedInt8Linear.from_linear(nn.Linear(inter, h, bias=False).to(gpu, dtype))
    with torch.no_grad():
        a, sa, stream = add_rms_norm_int8(x, residual, w, 1e-6)
        both = int8_matmul(a, sa, gate_up.codes, gate_up.scales, dtype=dtype)
        b, sb = silu_mul_int8(both[:, :inter], both[:, inter:])
        y = int8_matmul(b, sb, down.codes, down.scales, dtype=dtype)
    p, inverse, s = norm_rows(x, w, 1e-6, residual)
    assert torch.equal(stream, s) and torch.equal(a.double(), held(p)[0])
    assert_product(both, a, sa, gate_up.codes, gate_up.scales)
    v = swiglu_rows(both[:, :inter], both[:, inter:])
    assert float((b.double() - v * 127 / v.abs().amax(-1, keepdim=True)).abs().max()) <= 0.5 + 127 * 2.0**-20
    assert_product(y, b, sb, down.codes, down.scales)
    # and against the rows that are not quantized: half a step of the row's scale (and what the norm's
    # own roundings leave of it) in every term of the sum, then the product's bound
    weight = gate_up.codes.double() * gate_up.scales.double()[:, None]
    smooth = torch.matmul(p * inverse, weight.t().contiguous())
    slack = sa.double()[:, None] * (0.5 + 127 * 2.0**-19) * weight.abs().sum(1)
    size = smooth.abs() + slack
    assert bool(((both.double() - smooth).abs() <= slack + product_bound(size, size, dtype)).all())
    assert quantize_int8(both)[0].shape == both.shape


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", [(1, 33, 16), (1, 4096, 4096), (2, 1000, 8192), (3, 100, 5000), (4, 64, 4096), (5, 64, 4096),
                                   (1, 50, 16384), (1, 50, 16400), (16, 100, 1000), (17, 5000, 1024), (32, 300, 640), (33, 300, 640)])
def test_module_is_quantize_and_matmul(gpu, m, n, k, dtype):
    """Whichever launches a Linear takes, bit for bit the two operators, rows that no code holds among them."""
    w, sw = codes(n, k, gpu, 1, -127), scales(n, gpu, 2)
    bias = torch.randn(n, generator=torch.Generator(device=gpu).manual_seed(3), device=gpu).to(dtype)
    module = PackedInt8Linear(w, sw, bias=bias)
    x = torch.randn(m, k, generator=torch.Generator(device=gpu).manual_seed(4), device=gpu).to(dtype)
    with torch.no_grad():
        for change in range(4):
            if change == 1:
                x[m // 2] = 0
            if change == 2:
                x[m // 2, -1] = float("inf")
            if change == 3:
                x[0] = (x[0].double() * 2.0**-120).to(dtype)
            a, sa = quantize_int8(x)
            want = int8_matmul(a, sa, w, sw, bias=bias, dtype=dtype)
            got = module(x)
            assert torch.equal(got.view(torch.int16)[~torch.isnan(want)], want.view(torch.int16)[~torch.isnan(want)])
            assert torch.equal(torch.isnan(got), torch.isnan(want)), change
        odd = torch.randn(m, k + 1, device=gpu).to(dtype)[:, 1:]
        a, sa = quantize_int8(odd)
        assert torch.equal(module(odd), int8_matmul(a, sa, w, sw, bias=bias, dtype=dtype))
