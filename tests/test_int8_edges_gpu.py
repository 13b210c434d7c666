"""8-bit operators where a call can go wrong beside its numbers: what records a call, large
addresses, padded batches, host threads."""
import threading

import pytest
import torch

from marlin_style_fluxbin_amd import (PackedInt8Linear, add_rms_norm_int8, dequantize_int8, int8_matmul, quantize_int8,
                                      rms_norm_int8, silu_mul_int8)
from tests.int8_reference import assert_product, held, norm_rows, swiglu_rows

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def make(rows=5, columns=64, n=40, gpu="cuda"):
    g = torch.Generator(device=gpu).manual_seed(rows + columns)
    x = torch.randn(rows, columns, generator=g, device=gpu).to(BF)
    w = (1 + 0.1 * torch.randn(columns, generator=g, device=gpu)).to(BF)
    codes = torch.randint(-127, 128, (n, columns), generator=g, device=gpu, dtype=torch.int8)
    return x, w, codes, torch.rand(n, generator=g, device=gpu) + 0.1


def test_what_a_kernel_cannot_record_is_refused(gpu):
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    x, w, codes, scales = make()
    a, sa = quantize_int8(x)
    bias = torch.zeros(40, dtype=BF, device=gpu)
    linear = PackedInt8Linear(codes, scales)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: quantize_int8(dual(x)), lambda: rms_norm_int8(dual(x), w, 1e-6),
                     lambda: rms_norm_int8(x, dual(w), 1e-6), lambda: add_rms_norm_int8(x, dual(x), w, 1e-6),
                     lambda: silu_mul_int8(x, dual(x)), lambda: dequantize_int8(a, dual(sa)),
                     lambda: int8_matmul(a, dual(sa), codes, scales), lambda: int8_matmul(a, sa, codes, dual(scales)),
                     lambda: int8_matmul(a, sa, codes, scales, bias=dual(bias))):
            with pytest.raises(ValueError, match="tangent"):
                call()
        with pytest.raises(ValueError, match="tangent"), torch.no_grad():
            linear(dual(x))
        assert torch.equal(quantize_int8(x)[0], a)  # no tangent: as ever
    calls = (lambda t: quantize_int8(t)[1], lambda t: rms_norm_int8(t, w, 1e-6)[1], lambda t: silu_mul_int8(t, t)[1],
             lambda t: dequantize_int8(a, sa) + t, lambda t: int8_matmul(a, sa, codes, scales)[:, :1] + t)
    for call in calls:
        with pytest.raises(ValueError, match="trac"):
            torch.jit.trace(call, (x,))
        with pytest.raises(ValueError, match="trac"):
            make_fx(call)(x)
    for call in calls[:3]:
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.vmap(call)(torch.stack((x, x)))
    with pytest.raises(ValueError, match="no backward"):
        dequantize_int8(a, sa.clone().requires_grad_())


def test_a_compiled_caller_runs_the_call_as_it_is(gpu):
    x, w, codes, scales = make()
    linear = PackedInt8Linear(codes, scales)

    def step(x):
        a, sa, total = add_rms_norm_int8(x * 1, x, w, 1e-6)
        y = int8_matmul(a, sa, codes, scales)
        b, sb = silu_mul_int8(y, y * 1)
        return total * 1, y, dequantize_int8(b, sb) * 1, linear(x) * 1

    with torch.no_grad():
        want = step(x)
        got = torch.compile(step, backend="eager")(x)
    assert all(torch.equal(u, v) for u, v in zip(got, want))


@pytest.mark.parametrize("columns", [64, 1000, 4096, 12288])
@pytest.mark.parametrize("dtype", [BF, torch.float16])
def test_padded_batches(gpu, columns, dtype):
    """Rows of zeros and of NaN among others: zeros stay zeros (and NaN NaN) through the whole chain, the
    other rows are what they are alone."""
    x = torch.randn(40, columns, generator=torch.Generator().manual_seed(columns)).to(dtype).to(gpu)
    w = torch.ones(columns, dtype=dtype, device=gpu)
    _, _, codes, scales = make(5, columns, 48)
    x[1::3] = 0
    x[2::6] = float("nan")
    with torch.no_grad():
        a, sa = rms_norm_int8(x, w, 1e-6)
        y = int8_matmul(a, sa, codes, scales, dtype=dtype)
        b, sb = silu_mul_int8(y[:, :24], y[:, 24:])
        z = dequantize_int8(b, sb, dtype=dtype)
        assert bool((sa[1::3] == 0).all()) and not bool(y[1::3].any()) and not bool(z[1::3].any())
        assert bool(torch.isnan(sa[2::6]).all()) and bool(torch.isnan(y[2::6]).all()) and bool(torch.isnan(z[2::6]).all())
        for row in (0, 3, 38 if 38 % 3 == 0 else 39):
            alone = rms_norm_int8(x[row:row + 1].contiguous(), w, 1e-6)
            assert torch.equal(alone[0][0], a[row]) and torch.equal(alone[1][0], sa[row])
            assert torch.equal(int8_matmul(*alone, codes, scales, dtype=dtype)[0], y[row])


def test_a_row_is_the_same_in_any_batch(gpu):
    """Sums are exact, so a row's product does not depend on the kernel that the batch takes."""
    for n, k in ((1000, 1024), (4096, 4096), (300, 2077)):
        a = torch.randint(-127, 128, (2000, k), device=gpu, dtype=torch.int8)
        sa = torch.rand(2000, device=gpu)
        w, sw = torch.randint(-127, 128, (n, k), device=gpu, dtype=torch.int8), torch.rand(n, device=gpu)
        whole = int8_matmul(a, sa, w, sw)
        for m in (1, 16, 17, 40, 100, 300, 700):
            assert torch.equal(int8_matmul(a[:m], sa[:m], w, sw), whole[:m]), (n, k, m)


# ------------------------------------------------------------------ large addresses
@pytest.mark.parametrize("m", [3, 40])
def test_weight_past_2_to_32_bytes(gpu, m):
    n, k = 1 << 20, 4352
    w = torch.randint(-127, 128, (n, k), device=gpu, dtype=torch.int8)
    assert w[-1].data_ptr() - w.data_ptr() > 2**32
    sw = torch.rand(n, device=gpu)
    a, sa = torch.randint(-127, 128, (m, k), device=gpu, dtype=torch.int8), torch.rand(m, device=gpu)
    got = int8_matmul(a, sa, w, sw)
    for part in (slice(0, 300), slice(n - 300, n)):
        assert_product(got[:, part], a, sa, w[part], sw[part])


@pytest.mark.parametrize("k", [4352, 4353])
def test_activations_past_2_to_32_bytes(gpu, k):
    m, n = 1 << 20, 48
    a = torch.randint(-127, 128, (m, k), device=gpu, dtype=torch.int8)
    sa, sw = torch.rand(m, device=gpu), torch.rand(n, device=gpu)
    w = torch.randint(-127, 128, (n, k), device=gpu, dtype=torch.int8)
    got = int8_matmul(a, sa, w, sw)
    for part in (slice(0, 300), slice(m - 300, m)):
        assert_product(got[part], a[part], sa[part], w, sw)


def test_output_past_2_to_32_bytes(gpu):
    m, n, k = 70000, 33001, 64
    a, sa = torch.randint(-127, 128, (m, k), device=gpu, dtype=torch.int8), torch.rand(m, device=gpu)
    w, sw = torch.randint(-127, 128, (n, k), device=gpu, dtype=torch.int8), torch.rand(n, device=gpu)
    got = int8_matmul(a, sa, w, sw)
    assert got[-1].data_ptr() - got.data_ptr() > 2**32
    for part in (slice(0, 300), slice(m - 300, m)):
        assert_product(got[part], a[part], sa[part], w, sw)


def test_rows_past_2_to_32_bytes(gpu):
    m, k = 1 << 20, 4200
    x = torch.randn(m, k, device=gpu, dtype=BF)
    w = torch.ones(k, dtype=BF, device=gpu)
    last = slice(m - 100, m)
    codes, scales = quantize_int8(x)
    assert codes[-1].data_ptr() - codes.data_ptr() > 2**32
    assert torch.equal(codes[last].double(), held(x[last])[0])
    back = dequantize_int8(codes, scales)
    assert torch.equal(back[last], (codes[last].float() * scales[last, None]).to(BF))
    codes, scales = silu_mul_int8(x, back)
    p = swiglu_rows(x[last], back[last])
    assert float((codes[last].double() - p * 127 / p.abs().amax(-1, keepdim=True)).abs().max()) <= 0.5 + 127 * 2.0**-20
    want = norm_rows(x[last], w, 1e-6, back[last])
    codes, scales, total = add_rms_norm_int8(x, back, w, 1e-6, residual_out=x)
    assert torch.equal(total[last], want[2]) and torch.equal(codes[last].double(), held(want[0])[0])


# ------------------------------------------------------------------ host threads
def test_threads_on_their_own_streams(gpu):
    linears = [PackedInt8Linear(*make(5, 4096, n)[2:]) for n in (4096, 1000, 512, 2048)]
    xs = [torch.randn(m, 4096, device=gpu).to(BF) for m in (1, 20, 100, 64)]
    with torch.no_grad():
        want = [linear(x) for linear, x in zip(linears, xs)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.no_grad(), torch.cuda.stream(stream):
            for _ in range(30):
                y = linears[i](xs[i])
                a, sa = quantize_int8(xs[i])
                z = int8_matmul(a, sa, linears[i].codes, linears[i].scales)
                stream.synchronize()
                if not (torch.equal(y, want[i]) and torch.equal(z, want[i])):
                    wrong.append(i)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
