"""The cached-attention entry points on the host: header and binding agree, every bad argument
is refused before a launch, the workspace query follows the sizes.  CPU-only; device pointers
are stand-in addresses that no call here reaches."""
import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from marlin_style_fluxbin_amd import Int4KVCache, _lib, kv4_attention, window_attention

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "fluxbin_attention.h"
D = 1 << 24  # a 16-byte aligned stand-in device address


def _parameters():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return {m.group(1): [p.strip().split()[-1].lstrip("*") for p in m.group(2).split(",")]
            for m in re.finditer(r"\b(?:int|size_t)\s+(fx_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", text)}


PARAMS = _parameters()


def strides(*rows):
    return (ctypes.c_longlong * (3 * len(rows)))(*[s for r in rows for s in r])


ROW = (8192, 1024, 128)
ATTENTION = dict(q=D, k=D, v=D, out=D, lengths=None, query_lengths=None, workspace=D, workspace_bytes=1 << 30, batch=2,
                 n_q_heads=8, n_kv_heads=2, tokens=4, max_len=100, head_dim=128, window=10, sinks=2, scale=0.1, dtype=2,
                 stream=None, k_codes=D, k_scales=D, v_codes=D, v_scales=D)
DEFAULTS = {
    "fx_window_attention": dict(ATTENTION, strides=strides(ROW, ROW, ROW, ROW)),
    "fx_kv4_attention": dict(ATTENTION, strides=strides(ROW, ROW)),
    "fx_kv4_append": dict(ATTENTION, strides=strides(ROW, ROW), start=None, start_all=0, counts=None),
    "fx_kv4_restore": dict(ATTENTION, k_out=D, v_out=D, rows=100),
}


def call(name, **over):
    values = {**DEFAULTS[name], **over}
    lib = _lib.library()
    rc = getattr(lib, name)(*[values[p] for p in PARAMS[name]])
    return rc, lib.fx_last_error().decode()


def test_binding_matches_the_header():
    assert set(PARAMS) == set(_lib.ATTENTION_SIGNATURES)
    for name, parameters in PARAMS.items():
        assert hasattr(_lib.library(), name)
        assert len(_lib.ATTENTION_SIGNATURES[name][1]) == len(parameters), name
    assert '#include "fluxbin_attention.h"' in (ROOT / "include" / "fluxbin_amd.h").read_text()


def test_header_compiles_alone_as_c_and_cxx(tmp_path):
    for compiler, suffix, flags in (("gcc", "c", ["-std=c99"]), ("g++", "cc", [])):
        if shutil.which(compiler) is None:
            pytest.skip(f"no {compiler}")
        src = tmp_path / f"probe.{suffix}"
        src.write_text('#include "fluxbin_attention.h"\nint main(void) { return (int)fx_cached_attention_workspace_bytes(1, 1, 1, 1, 1, 64, 0, 0, 2, 0); }\n')
        subprocess.run([compiler, *flags, "-Wall", "-Wextra", "-Werror", "-I", str(ROOT / "include"), "-c", str(src),
                        "-o", str(tmp_path / "probe.o")], check=True)


SHARED = [
    (dict(head_dim=96), "head_dim must be 64, 128 or 256"),
    (dict(batch=-1), "batch must be in"),
    (dict(batch=1 << 17), "batch must be in"),
    (dict(n_kv_heads=0), "n_kv_heads must be in"),
    (dict(max_len=-1), "max_len must be in"),
    (dict(dtype=0), "dtype must be fp16 or bf16"),
    (dict(batch=1 << 16, n_kv_heads=256, n_q_heads=256), "too large for one call"),
]
QUERIES = [
    (dict(tokens=-1), "tokens must be in"),
    (dict(n_q_heads=3), "positive multiple"),
    (dict(n_q_heads=0), "positive multiple"),
    (dict(window=-1), "non-negative"),
    (dict(sinks=-1), "non-negative"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=-1.0), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
    (dict(scale=float("inf")), "scale must be positive"),
    (dict(q=None), "q and out must be non-null"),
    (dict(out=None), "q and out must be non-null"),
    (dict(q=D + 8), "q and out must be 16-byte aligned"),
    (dict(out=D + 2), "q and out must be 16-byte aligned"),
    (dict(strides=None), "strides must be non-null"),
    (dict(window=0, batch=1, max_len=100000, workspace=None), "workspace needs"),
    (dict(window=0, batch=1, max_len=100000, workspace_bytes=16), "workspace needs"),
    (dict(window=0, batch=1, max_len=100000, workspace=D + 8), "workspace must be 16-byte aligned"),
]
CACHE = [(dict(**{name: None}), "cache arrays must be non-null") for name in ("k_codes", "k_scales", "v_codes", "v_scales")]
CACHE += [(dict(k_scales=D + 4), "cache arrays must be 16-byte aligned")]
CASES = [("fx_window_attention", *c) for c in SHARED + QUERIES]
CASES += [("fx_window_attention", *c) for c in [
    (dict(k=None), "k and v must be non-null"),
    (dict(v=D + 4), "k and v must be 16-byte aligned"),
    (dict(strides=strides((8192, 1024, 12), ROW, ROW, ROW)), "q strides"),
    (dict(strides=strides(ROW, (-8, 1024, 128), ROW, ROW)), "k strides"),
    (dict(strides=strides(ROW, ROW, (8192, 1024, 1 << 23), ROW)), "v position stride"),
    (dict(strides=strides(ROW, ROW, ROW, (8192, 1025, 128))), "out strides"),
]]
CASES += [("fx_kv4_attention", *c) for c in SHARED + QUERIES + CACHE]
CASES += [("fx_kv4_attention", dict(strides=strides(ROW, (8192, 4, 128))), "out strides")]
CASES += [("fx_kv4_append", *c) for c in SHARED + CACHE + [
    (dict(tokens=-2), "tokens must be in"),
    (dict(k=None), "k and v must be non-null"),
    (dict(k=D + 8), "k and v must be 16-byte aligned"),
    (dict(strides=None), "strides must be non-null"),
    (dict(strides=strides((8192, 1024, 4), ROW)), "k strides"),
    (dict(strides=strides(ROW, (8192, -1024, 128))), "v strides")]]
CASES += [("fx_kv4_restore", *c) for c in SHARED + CACHE + [
    (dict(rows=101), "rows must be in"),
    (dict(rows=-1), "tokens must be in"),
    (dict(k_out=None), "k_out and v_out must be non-null"),
    (dict(v_out=D + 8), "k_out and v_out must be 16-byte aligned")]]


@pytest.mark.parametrize("name,over,message", CASES, ids=lambda x: x if isinstance(x, str) else None)
def test_refusals(name, over, message):
    rc, error = call(name, **over)
    assert rc == 1 and message in error, (rc, error)


def test_every_entry_point_has_a_case():
    assert {c[0] for c in CASES} | {"fx_cached_attention_workspace_bytes"} == set(PARAMS)


@pytest.mark.parametrize("name,over", [
    ("fx_window_attention", dict(batch=0)), ("fx_window_attention", dict(tokens=0, q=None, out=None)),
    ("fx_kv4_attention", dict(batch=0)), ("fx_kv4_append", dict(tokens=0)), ("fx_kv4_append", dict(max_len=0)),
    ("fx_kv4_restore", dict(rows=0))])
def test_empty_calls_do_nothing(name, over):
    assert call(name, **over)[0] == 0


def test_workspace_query():
    size = _lib.library().fx_cached_attention_workspace_bytes
    # one query row over a long cache is split; partials are fp32 [rows, splits, D + 2]
    assert size(1, 32, 8, 1, 100000, 128, 0, 0, 2, 0) == 32 * 64 * 130 * 4
    # a prompt fills the chip by its rows
    assert size(1, 32, 8, 16384, 16384, 128, 0, 0, 2, 0) == 0
    # a window bounds the splits whatever the cache could hold
    assert size(1, 32, 8, 1, 1 << 20, 128, 256, 4, 2, 0) == size(1, 32, 8, 1, 1 << 28, 128, 256, 4, 2, 0) < 32 * 64 * 130 * 4
    for bad in (dict(d=96), dict(dt=0), dict(b=-1), dict(hq=3, hk=2)):
        v = dict(b=1, hq=32, hk=8, t=1, n=100000, d=128, w=0, s=0, dt=2, kv4=0) | bad
        assert size(*v.values()) == 0


def test_cpu_tensors_are_refused():
    q, k = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1, 5, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="q must be a GPU tensor"):
        window_attention(q, k, k)
    with pytest.raises(ValueError, match="GPU"):
        Int4KVCache(1, 1, 5, 64, device="cpu")


@pytest.mark.parametrize("args", [(0, 1, 5, 64), (1, 0, 5, 64), (1, 1, 0, 64), (1, 1, 5, 80)])
def test_cache_sizes_are_checked(args):
    with pytest.raises(ValueError):
        Int4KVCache(*args)
    assert callable(kv4_attention)
