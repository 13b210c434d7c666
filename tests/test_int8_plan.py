"""Every kernel of the 8-bit products at sizes that take it: what the plan chooses is asked of the
library, so that no change of its estimate leaves a kernel without a test.  And the few-rows kernel
on rows at any address, in each of its forms."""
import ctypes
from functools import lru_cache
from itertools import product as combinations

import pytest
import torch

from marlin_style_fluxbin_amd import _lib, int8_matmul
from tests.int8_reference import assert_product

FEW = -1
TILES = {0: "64 x 64", 1: "64 x 128", 2: "128 x 128", 3: "128 x 256", 4: "256 x 256"}
KINDS = [(FEW, False), *combinations(TILES, (False, True))]
ODD = [(m, n, k) for m, n, k in combinations(
    (1, 5, 16, 17, 31, 33, 90, 130, 200, 260, 390, 700, 1300, 2050),
    (17, 100, 300, 1000, 2049, 4097, 6001, 8200),
    (48, 528, 1040, 3712, 4112, 8208, 12304, 16400)) if m * n * k < 5e10]


class Plan(ctypes.Structure):
    _fields_ = [("tile", ctypes.c_int), ("splits", ctypes.c_int), ("k_per_split", ctypes.c_int)]


@lru_cache(maxsize=None)
def plan(m, n, k):
    """The kernel (its index, FEW for the few-rows one) and the K splits of a product of aligned rows:
    fx::plan_int8_gemm, which the library holds as a C++ function."""
    choose = _lib.library()._ZN2fx14plan_int8_gemmEiiib
    choose.restype, choose.argtypes = Plan, [ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_bool]
    chosen = choose(m, n, k, False)
    return chosen.tile, chosen.splits


@lru_cache(maxsize=None)
def sizes(kind):
    """Some of the sizes that take a kernel whole or in K splits: the first, the last and one between."""
    tile, split = kind
    found = [s for s in ODD if plan(*s)[0] == tile and (plan(*s)[1] > 1) is split]
    return sorted({found[0], found[len(found) // 2], found[-1]}) if found else []


@pytest.mark.parametrize("kind", KINDS)
def test_every_kernel_has_sizes(kind):
    assert sizes(kind), kind


def test_a_split_products_workspace_is_asked_for():
    lib = _lib.library()
    split = [s for tile in TILES for s in sizes((tile, True))]
    assert len(split) >= len(TILES)
    address = 1 << 24
    for m, n, k in split:
        nbytes = lib.fx_int8_gemm_workspace_bytes(m, n, k, 0)
        assert nbytes >= plan(m, n, k)[1] * m * n * 4 > 0
        for workspace, given, message in ((None, 0, "workspace needs"), (address, nbytes - 1, "workspace needs"),
                                          (address + 4, 1 << 40, "16-byte aligned")):
            assert lib.fx_int8_gemm(address, k, address, address, k, address, None, address, n, workspace, given, m, n, k,
                                    _lib.dtype_code(torch.bfloat16), None) == 1
            assert message in lib.fx_last_error().decode()


def rows(count, columns, gpu, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    codes = torch.randint(-128, 128, (count, columns), generator=g, device=gpu, dtype=torch.int32).to(torch.int8)
    return codes, torch.rand(count, generator=g, device=gpu) * 0.01 + 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", KINDS, ids=lambda kind: f"{TILES.get(kind[0], 'few')}{' split' if kind[1] else ''}")
def test_every_kernel(gpu, kind, dtype):
    for m, n, k in sizes(kind):
        (a, sa), (w, sw) = rows(m, k, gpu, 1), rows(n, k, gpu, 2)
        bias = torch.randn(n, generator=torch.Generator(device=gpu).manual_seed(3), device=gpu).to(dtype)
        assert_product(int8_matmul(a, sa, w, sw, bias=bias, dtype=dtype), a, sa, w, sw, bias, context=(m, n, k))


# 1 to 16 rows by 16 columns (eight waves with two and with four pieces in flight, sixteen waves), 17 to
# 32 rows by 16 and by 32 columns with two and with four; the last block of columns and of K not whole
@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 16, 17, 31, 32])
@pytest.mark.parametrize("n", [1, 70, 4096, 4097, 8200])
@pytest.mark.parametrize("k", [1, 63, 1041, 4090, 8200, 12275])
def test_few_rows_at_any_address(gpu, m, n, k):
    """Odd lengths and odd addresses, large values around every row, an output among others."""
    store_a = torch.full((m + 2, k + 5), 127, dtype=torch.int8, device=gpu)
    store_w = torch.full((n + 2, k + 9), 127, dtype=torch.int8, device=gpu)
    a, w = store_a[1:1 + m, 3:3 + k], store_w[1:1 + n, 5:5 + k]
    codes, sa = rows(m, k, gpu, 1)
    a.copy_(codes)
    codes, sw = rows(n, k, gpu, 2)
    w.copy_(codes)
    dtype = (torch.bfloat16, torch.float16, torch.float32)[(m + n + k) % 3]
    out = torch.full((m + 2, n + 5), 5.0, dtype=dtype, device=gpu)
    view = out[1:1 + m, 3:3 + n]
    int8_matmul(a, sa, w, sw, dtype=dtype, out=view)
    assert_product(view, a, sa, w, sw, context=(m, n, k, dtype))
    out[1:1 + m, 3:3 + n] = 5
    assert bool((out == 5).all())
    assert bool((store_a[:, :3] == 127).all()) and bool((store_w[:, 5 + k:] == 127).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [16, 17, 32])
@pytest.mark.parametrize("k", [512, 4096])
def test_few_whole_rows_at_odd_addresses(gpu, m, k):
    """K of whole 16 bytes: one operand or both beside its 16-byte boundary."""
    n = 4100
    (a, sa), (w, sw) = rows(m, k, gpu, 1), rows(n, k, gpu, 2)
    want = int8_matmul(a, sa, w, sw)
    assert_product(want, a, sa, w, sw)

    def shifted(t):
        return torch.empty(t.numel() + 1, dtype=torch.int8, device=gpu)[1:].view(t.shape).copy_(t)

    for left, right in ((shifted(a), w), (a, shifted(w)), (shifted(a), shifted(w))):
        assert torch.equal(int8_matmul(left, sa, right, sw), want)  # exact sums, the same roundings
