"""Sizes past what one call of the 8-bit operators takes: refused by their whole value, though the
library's size arguments are 32 bits wide.  CPU-only: fake tensors of a GPU device have the sizes,
and no call may reach the library."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from marlin_style_fluxbin_amd import (PackedInt8Linear, add_rms_norm_int8, dequantize_int8, int8_linear, int8_matmul,
                                      quantize_int8, rms_norm_int8, silu_mul_int8)

BF = torch.bfloat16
ROWS, COLUMNS = 1 << 21, 1 << 20


class Reached(Exception):
    """The arguments went on to the library."""


@pytest.fixture
def fake(monkeypatch):
    def launch(name, index, *args):
        raise Reached(name)

    def made(shape, dtype, device):
        raise Reached("an output's memory")

    monkeypatch.setattr(int8_linear, "_launch", launch)
    monkeypatch.setattr(int8_linear, "_new", made)
    with FakeTensorMode():
        yield lambda *shape, dtype=BF: torch.empty(*shape, dtype=dtype, device="cuda:0")


def rows_calls(make, rows, columns):
    x, w = make(rows, columns), make(columns)
    codes, scales = make(rows, columns, dtype=torch.int8), make(rows, dtype=torch.float32)
    return (lambda: quantize_int8(x), lambda: rms_norm_int8(x, w, 1e-6), lambda: add_rms_norm_int8(x, x, w, 1e-6),
            lambda: silu_mul_int8(x, x), lambda: dequantize_int8(codes, scales), lambda: quantize_int8(x.t().contiguous().t()))


@pytest.mark.parametrize("rows,columns", [(ROWS + 1, 8), (2**32, 8), (2**32 + 3, 8), (3, COLUMNS + 1), (3, 2**32),
                                          (3, 2**32 + 64)])
def test_rows_past_one_call(fake, rows, columns):
    for call in rows_calls(fake, rows, columns):
        with pytest.raises(ValueError, match="at most"):
            call()
    with pytest.raises(ValueError, match="at most"):
        quantize_int8(fake(1, columns).expand(rows, columns))
    with pytest.raises(ValueError, match="at most"):
        quantize_int8(fake(2, rows, columns))


@pytest.mark.parametrize("rows,columns", [(ROWS, 8), (3, COLUMNS), (0, 8), (1, 1)])
def test_rows_that_one_call_takes(fake, rows, columns):
    for call in rows_calls(fake, rows, columns):
        with pytest.raises(Reached):
            call()


def product(make, m, n, k):
    return int8_matmul(make(m, k, dtype=torch.int8), make(m, dtype=torch.float32), make(n, k, dtype=torch.int8),
                       make(n, dtype=torch.float32))


@pytest.mark.parametrize("m,n,k", [(ROWS + 1, 8, 16), (2**32 + 5, 8, 16), (2**32, 8, 16), (3, COLUMNS + 1, 16),
                                   (3, 2**32 + 8, 16), (3, 8, 131057), (3, 8, 2**32 + 16), (3, 0, 16), (3, 8, 0)])
def test_products_past_one_call(fake, m, n, k):
    with pytest.raises(ValueError, match="K must be"):
        product(fake, m, n, k)


@pytest.mark.parametrize("m,n,k", [(ROWS, 8, 16), (3, COLUMNS, 16), (3, 8, 131056), (0, 8, 16)])
def test_products_that_one_call_takes(fake, m, n, k):
    with pytest.raises(Reached):
        product(fake, m, n, k)


@pytest.mark.parametrize("out", [COLUMNS + 1, 2**32 + 8])
def test_modules_past_one_call(fake, out):
    with torch.no_grad():
        codes, scales = fake(out, 32, dtype=torch.int8), fake(out, dtype=torch.float32)
        module = PackedInt8Linear(codes, scales)
        with pytest.raises(ValueError, match="fallback"):
            module(fake(3, 32))
        with pytest.raises(ValueError, match="at most"):
            module._packed_kernel(1, codes.device)
        with pytest.raises(ValueError, match="at most"):
            module.bind_prepared_decode(BF)
        dense = PackedInt8Linear(codes, scales, fallback="dense")
        assert dense(fake(3, 32)).shape == (3, out) and dense.route_counts["dense_fallback"] == 1


def test_module_rows_past_one_call(fake):
    with torch.no_grad():
        module = PackedInt8Linear(fake(8, 32, dtype=torch.int8), fake(8, dtype=torch.float32))
        for rows in (ROWS + 1, 2**32 + 3):
            with pytest.raises(ValueError, match="fallback"):
                module(fake(1, 32).expand(rows, 32))
        with pytest.raises(Reached):
            module(fake(ROWS, 32))
