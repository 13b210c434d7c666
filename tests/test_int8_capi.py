"""The 8-bit entry points on the host: header and binding agree, every bad argument is refused
before a launch, the Python layer refuses what the kernels do not take.  CPU-only; device
pointers are stand-in addresses that no call here reaches."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch
from torch import nn

from marlin_style_fluxbin_amd import (PackedInt8Linear, _lib, add_rms_norm_int8, dequantize_int8, int8_matmul,
                                      quantize_int8, quantize_weight_int8, rms_norm_int8, silu_mul_int8)
from tests.int8_reference import held

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "fluxbin_int8.h"
D = 1 << 24  # a 16-byte aligned stand-in device address


def _parameters():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return {m.group(1): [p.strip().split()[-1].lstrip("*") for p in m.group(2).split(",")]
            for m in re.finditer(r"\b(?:int|size_t)\s+(fx_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", text)}


PARAMS = _parameters()
ROWS = dict(x=D, x_stride=100, codes=D, code_stride=112, scales=D, rows=3, columns=100, code_columns=112, dtype=2,
            stream=None)
DEFAULTS = {
    "fx_int8_quantize": ROWS,
    "fx_int8_rmsnorm": dict(ROWS, residual=D, residual_stride=100, residual_out=D, residual_out_stride=100, weight=D,
                            eps=1e-6),
    "fx_int8_silu_mul": dict(ROWS, gate=D, gate_stride=200, up=D, up_stride=200),
    "fx_int8_restore": dict(codes=D, code_stride=112, scales=D, out=D, out_stride=100, rows=3, columns=100, dtype=2,
                            stream=None),
    "fx_int8_gemm_workspace_bytes": dict(M=1, N=1, K=16, loose=0),
    "fx_int8_linear_workspace_bytes": dict(M=1, N=1, K=16),
    "fx_int8_linear": dict(x=D, x_stride=60, x_dtype=2, w=D, w_stride=64, w_scales=D, bias=D, out=D, out_stride=8,
                           workspace=D, workspace_bytes=1 << 20, M=3, N=8, K=60, out_dtype=2, stream=None),
    "fx_int8_gemm": dict(a=D, a_stride=64, a_scales=D, w=D, w_stride=64, w_scales=D, bias=D, out=D, out_stride=8,
                         workspace=None, workspace_bytes=0, M=3, N=8, K=64, dtype=2, stream=None),
}


def call(name, **over):
    values = {**DEFAULTS[name], **over}
    lib = _lib.library()
    rc = getattr(lib, name)(*[values[p] for p in PARAMS[name]])
    return rc, lib.fx_last_error().decode()


def test_binding_matches_the_header():
    assert set(PARAMS) == set(_lib.INT8_SIGNATURES) == set(DEFAULTS)
    for name, parameters in PARAMS.items():
        assert hasattr(_lib.library(), name)
        assert len(_lib.INT8_SIGNATURES[name][1]) == len(parameters), name
    assert '#include "fluxbin_int8.h"' in (ROOT / "include" / "fluxbin_amd.h").read_text()


def test_header_compiles_alone_as_c_and_cxx(tmp_path):
    for compiler, suffix, flags in (("gcc", "c", ["-std=c99"]), ("g++", "cc", [])):
        if shutil.which(compiler) is None:
            pytest.skip(f"no {compiler}")
        src = tmp_path / f"probe.{suffix}"
        src.write_text('#include "fluxbin_int8.h"\nint main(void) { return (int)fx_int8_gemm_workspace_bytes(1, 1, 16, 0); }\n')
        subprocess.run([compiler, *flags, "-Wall", "-Wextra", "-Werror", "-I", str(ROOT / "include"), "-c", str(src),
                        "-o", str(tmp_path / "probe.o")], check=True)


SHARED = [
    (dict(rows=-1), "rows must be in"), (dict(rows=(1 << 21) + 1), "rows must be in"),
    (dict(columns=0), "columns must be in"), (dict(columns=(1 << 20) + 1, code_columns=(1 << 20) + 1), "columns must be in"),
    (dict(code_columns=99), "code_columns must be in"), (dict(code_columns=228, code_stride=300), "code_columns must be in"),
    (dict(codes=None), "codes and scales must be non-null"), (dict(scales=None), "codes and scales must be non-null"),
    (dict(scales=D + 2), "scales must be 4-byte aligned"), (dict(code_stride=111), "codes stride"),
    (dict(dtype=0), "dtype must be fp16 or bf16"),
]
CASES = [("fx_int8_quantize", *c) for c in SHARED + [
    (dict(x=None), "x must be non-null"), (dict(x=D + 1), "x must be 2-byte aligned"),
    (dict(x_stride=-1), "x stride must be non-negative")]]
CASES += [("fx_int8_rmsnorm", *c) for c in SHARED + [
    (dict(x=None), "x must be non-null"), (dict(weight=None), "weight must be non-null"),
    (dict(weight=D + 1), "weight must be 2-byte aligned"), (dict(residual_out=None), "residual_out must be non-null"),
    (dict(residual=D + 1), "residual must be 2-byte aligned"), (dict(residual_stride=-8), "residual stride"),
    (dict(residual_out_stride=99), "residual_out stride"), (dict(eps=-1.0), "eps must be"),
    (dict(eps=float("nan")), "eps must be"), (dict(eps=float("inf")), "eps must be")]]
CASES += [("fx_int8_silu_mul", *c) for c in SHARED + [
    (dict(gate=None), "gate must be non-null"), (dict(up=None), "up must be non-null"),
    (dict(up=D + 1), "up must be 2-byte aligned"), (dict(up_stride=-1), "up stride")]]
CASES += [("fx_int8_restore", *c) for c in [
    (dict(rows=-1), "rows must be in"), (dict(columns=0), "columns must be in"), (dict(dtype=3), "dtype must be fp32"),
    (dict(rows=1 << 21, columns=1 << 20, out_stride=1 << 20), "too large for one call"),
    (dict(codes=None), "must be non-null"), (dict(scales=None), "must be non-null"), (dict(out=None), "must be non-null"),
    (dict(out=D + 2, dtype=0), "aligned to their elements"), (dict(scales=D + 2), "aligned to their elements"),
    (dict(code_stride=-1), "do not fit rows"), (dict(out_stride=99), "do not fit rows")]]
CASES += [("fx_int8_gemm", *c) for c in [
    (dict(M=-1), "M must be in"), (dict(M=(1 << 21) + 1), "M must be in"), (dict(N=0), "N must be in"),
    (dict(N=(1 << 20) + 1), "N must be in"), (dict(K=0), "K must be"), (dict(K=-16), "K must be"),
    (dict(K=131072, a_stride=131072, w_stride=131072), "K must be in [1, 131056]"), (dict(dtype=3), "dtype must be fp32"),
    (dict(a=None), "a must be non-null"), (dict(w=None), "w must be non-null"),
    (dict(a_stride=48), "a stride must be"), (dict(w_stride=63), "w stride must be"),
    (dict(a=D + 8, M=100), "workspace needs"), (dict(w_stride=72, M=100), "workspace needs"),
    (dict(K=60, M=100, workspace=D, workspace_bytes=64 * 108 - 1), "workspace needs"),
    (dict(w_stride=(1 << 22) + 16, M=100), "workspace needs"),
    (dict(a_stride=-64), "a stride must be"), (dict(a_scales=None), "scales and out must be non-null"),
    (dict(out=None), "scales and out must be non-null"), (dict(w_scales=D + 2), "aligned to their elements"),
    (dict(bias=D + 2, dtype=0), "aligned to their elements"), (dict(out=D + 1), "aligned to their elements"),
    (dict(out_stride=7), "out stride")]]
CASES += [("fx_int8_linear", *c) for c in [
    (dict(M=-1), "M must be in"), (dict(N=0), "N must be in"), (dict(K=0), "K must be in"),
    (dict(K=131057), "K must be in"), (dict(x_dtype=0), "x dtype must be"), (dict(out_dtype=3), "dtype must be fp32"),
    (dict(workspace=None), "workspace needs"), (dict(workspace_bytes=511), "workspace needs"),
    (dict(workspace=D + 8), "workspace must be 16-byte aligned"), (dict(x=None), "x must be non-null"),
    (dict(x_stride=-2), "x stride"), (dict(w=None), "w must be non-null"), (dict(w_stride=48), "w stride"),
    (dict(w=D + 8), "w must have rows of whole 16 bytes"), (dict(w_scales=None), "scales and out must be non-null"),
    (dict(bias=D + 1), "aligned to their elements"), (dict(out_stride=7), "out stride")]]


@pytest.mark.parametrize("name,over,message", CASES, ids=lambda x: x if isinstance(x, str) else None)
def test_refusals(name, over, message):
    rc, error = call(name, **over)
    assert rc == 1 and message in error, (rc, error)


@pytest.mark.parametrize("name", [n for n in DEFAULTS if "gemm" not in n and "linear" not in n])
def test_no_rows_do_nothing(name):
    assert call(name, rows=0, codes=None, scales=None, out=None)[0] == 0 if name == "fx_int8_restore" else (
        call(name, rows=0)[0] == 0)
    assert call("fx_int8_gemm", M=0, a=None, out=None)[0] == 0
    assert call("fx_int8_linear", M=0, x=None, workspace=None)[0] == 0


def test_workspace_query_refuses_bad_sizes():
    size = _lib.library().fx_int8_gemm_workspace_bytes
    assert size(-1, 8, 64, 0) == size(1, 0, 64, 0) == size(1, 8, 0, 0) == size(0, 8, 64, 3) == 0
    # up to 32 rows are read wherever they lie; copies of more are whole 16 bytes wide
    assert size(32, 8, 65, 3) == size(32, 8, 64, 0) == 0
    one = size(100, 8, 64, 0)
    assert size(100, 8, 64, 1) == one + 100 * 64 and size(100, 8, 64, 2) == one + 8 * 64
    assert size(100, 8, 60, 0) == size(100, 8, 60, 3) == one + 108 * 64
    whole = _lib.library().fx_int8_linear_workspace_bytes
    assert whole(-1, 8, 64) == whole(1, 0, 64) == whole(1, 8, 0) == whole(0, 8, 64) == whole(1, 8, 131057) == 0
    # codes padded to whole 16 columns, a scale for each row, the product's own
    assert whole(3, 8, 60) == 256 + 256 + size(3, 8, 64, 0)


def test_a_split_products_workspace_is_checked():
    size = _lib.library().fx_int8_gemm_workspace_bytes
    split = [s for s in ((64, 256, 65536), (128, 1024, 12288), (200, 64, 131056)) if size(*s, 0)]
    for m, n, k in split:
        sizes = dict(M=m, N=n, K=k, a_stride=k, w_stride=k, out_stride=n)
        assert "workspace needs" in call("fx_int8_gemm", **sizes)[1]
        assert "workspace needs" in call("fx_int8_gemm", **sizes, workspace=D, workspace_bytes=size(m, n, k, 0) - 1)[1]
        assert "16-byte aligned" in call("fx_int8_gemm", **sizes, workspace=D + 4, workspace_bytes=1 << 40)[1]


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 32, dtype=torch.bfloat16), torch.ones(32, dtype=torch.bfloat16)
    codes, scales = torch.zeros(2, 32, dtype=torch.int8), torch.ones(2)
    for call_ in (lambda: quantize_int8(x), lambda: rms_norm_int8(x, w, 1e-6), lambda: add_rms_norm_int8(x, x, w, 1e-6),
                  lambda: silu_mul_int8(x, x), lambda: dequantize_int8(codes, scales),
                  lambda: int8_matmul(codes, scales, codes, scales)):
        with pytest.raises(ValueError, match="must be a GPU tensor"):
            call_()


def test_module_on_the_host():
    g = torch.Generator().manual_seed(0)
    linear = nn.Linear(40, 7)
    with torch.no_grad():
        linear.weight.copy_(torch.randn(7, 40, generator=g))
        linear.weight[3] = 0
    codes, scales = quantize_weight_int8(linear.weight)
    want_codes, want_scales = held(linear.weight.double())
    assert torch.equal(codes.double(), want_codes) and torch.equal(scales, want_scales)
    module = PackedInt8Linear.from_linear(linear, fallback="dense")
    assert (module.out_features, module.in_features, module.codes.shape) == (7, 40, (7, 48))
    assert not bool(module.codes[:, 40:].any())
    x = torch.randn(3, 40, generator=g)
    with torch.no_grad():
        weight = codes.float() * scales[:, None]
        assert torch.equal(module(x), torch.nn.functional.linear(x, weight, linear.bias))
        assert module.route_counts["dense_fallback"] == 1
        strict = PackedInt8Linear.from_linear(linear)
        with pytest.raises(ValueError, match="fallback"):
            strict(x)
        with pytest.raises(ValueError, match="expected"):
            strict(x[:, :39])
    with pytest.raises(RuntimeError, match="no_grad"):
        module(x)
    with pytest.raises(ValueError, match="cast"), torch.no_grad():
        PackedInt8Linear.from_linear(linear, fallback="dense").half()(x)
    again = PackedInt8Linear(torch.zeros(7, 40, dtype=torch.int8), torch.ones(7), bias=linear.bias)
    again.load_state_dict(module.state_dict())
    assert torch.equal(again.codes, module.codes) and torch.equal(again.scales, module.scales)


@pytest.mark.parametrize("over", [
    dict(codes=torch.zeros(7, 40)), dict(codes=torch.zeros(7, 0, dtype=torch.int8)),
    dict(codes=torch.zeros(40, dtype=torch.int8)), dict(scales=torch.ones(8)), dict(scales=torch.ones(7).half()),
    dict(bias=torch.ones(8)), dict(codes=torch.zeros(7, 131057, dtype=torch.int8)), dict(fallback="maybe")])
def test_module_refusals(over):
    args = dict(codes=torch.zeros(7, 40, dtype=torch.int8), scales=torch.ones(7), bias=None, fallback="error") | over
    with pytest.raises(ValueError):
        PackedInt8Linear(args["codes"], args["scales"], bias=args["bias"], fallback=args["fallback"])
    with pytest.raises(ValueError, match="nn.Linear"):
        PackedInt8Linear.from_linear(nn.Identity())
    with pytest.raises(ValueError, match="finite"):
        quantize_weight_int8(torch.full((2, 3), float("inf")))
