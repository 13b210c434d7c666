"""Attention over long caches: a sliding window with sinks, and a cache held in 4 bits.

No reference counterpart: the reference's decode runs stock SDPA over a full 16-bit
static cache of one sequence (``static_decode.py:67-81``), which this package serves with
``fx_decode_attention``.  The operators here take what that path does not: batches at
ragged lengths, prompts and chunks of any number of tokens, a window of the last keys
with a few first tokens that stay visible, and an :class:`Int4KVCache` in a quarter of the
bytes (4.5 bits a value).  Every call goes to the HIP kernels behind
``include/fluxbin_attention.h`` on the current stream of the tensors' device; there is no
CPU substitute and no backward pass.  Lengths stay on the device, so calls can be captured
into a HIP graph and follow the lengths of each replay.
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch

from . import _lib

_HALF = (torch.float16, torch.bfloat16)
HEAD_DIMS = (64, 128, 256)
KV4_GROUP = 64  # columns that share a scale and a minimum
_LIMIT = 2**31 - 1


@lru_cache(maxsize=256)
def _workspace_bytes(*sizes) -> int:
    return _lib.library().fx_cached_attention_workspace_bytes(*sizes)


def _strides(t: torch.Tensor) -> list[int]:
    """(batch, head, row) strides; an axis of one element never moves."""
    return [0 if n == 1 else s for n, s in zip(t.shape, t.stride()[:3])]


def _rows_ok(t: torch.Tensor) -> bool:
    """16-byte aligned rows of contiguous columns."""
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and not any(s % 8 for s in _strides(t))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a copy of it whose rows the kernels can read."""
    if _rows_ok(t):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_heads(name: str, t: torch.Tensor) -> None:
    if t.ndim != 4:
        raise ValueError(f"{name} must have shape [batch, heads, tokens, head_dim]")
    _lib.require_gpu_tensor(t, name)
    if t.dtype not in _HALF:
        raise ValueError(f"{name} must be fp16 or bf16")
    if t.shape[3] not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {t.shape[3]}")


def _check_counts(name: str, t: torch.Tensor | None, batch: int, device: torch.device) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.int32 or t.shape != (batch,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [batch] tensor on the device of the cache")
    return t.data_ptr()


def _check_inference(*tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError("cached attention has no backward pass; call it under torch.no_grad()")


def _on_device(device: torch.device, call, *args) -> int:
    """Launch with ``device`` current (kernels launch on the current device)."""
    if torch.cuda.current_device() == device.index:
        return call(*args, _lib.stream_handle(device))
    with torch.cuda.device(device):
        return call(*args, _lib.stream_handle(device))


def _attention(name, q, cache, cache_args, cache_strides, lengths, query_lengths, window, sinks, scale, out, kv4):
    """Checks and call shared by the two caches; ``cache`` is (batch, kv heads, max_len)."""
    batch, heads, tokens, dim = q.shape
    kv_heads, max_len = cache[1], cache[2]
    device = q.device
    if cache[0] != batch:
        raise ValueError(f"q and the cache disagree on the batch: {batch} and {cache[0]}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a positive multiple of KV heads ({kv_heads})")
    if window is None:
        window = 0
    elif not isinstance(window, int) or isinstance(window, bool) or not 1 <= window <= _LIMIT:
        raise ValueError("window must be None or a positive integer")
    if not isinstance(sinks, int) or isinstance(sinks, bool) or not 0 <= sinks <= _LIMIT:
        raise ValueError("sinks must be a non-negative integer")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    # no key lies beyond max_len, so neither a window nor sinks need to
    window, sinks = min(window, max_len + 1), min(sinks, max_len)
    lengths_ptr = _check_counts("lengths", lengths, batch, device)
    counts_ptr = _check_counts("query_lengths", query_lengths, batch, device)
    if out is None:
        make = torch.empty if query_lengths is None else torch.zeros
        out = make((batch, tokens, heads, dim), dtype=q.dtype, device=device).transpose(1, 2)
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != device:
            raise ValueError("out must have q's shape, dtype and device")
        if not _rows_ok(out) or any(s == 0 and n > 1 for n, s in zip(out.shape, out.stride())):
            raise ValueError("out must have contiguous 16-byte aligned rows, each its own memory")
    q = _rows(q)
    nbytes = _workspace_bytes(batch, heads, kv_heads, tokens, max_len, dim, window, sinks, kv4)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    strides = (ctypes.c_longlong * (6 + len(cache_strides)))(*_strides(q), *cache_strides, *_strides(out))
    rc = _on_device(device, getattr(_lib.library(), name), q.data_ptr(), *cache_args, out.data_ptr(), strides,
                    lengths_ptr, counts_ptr, _lib.ptr(workspace), nbytes, batch, heads, kv_heads, tokens, max_len, dim,
                    window, sinks, scale, _lib.dtype_code(q.dtype))
    if rc:
        _lib.check(rc, name)
    return out


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, lengths: torch.Tensor | None = None,
                     query_lengths: torch.Tensor | None = None, window: int | None = None, sinks: int = 0,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of ``q [batch, heads, tokens, head_dim]`` over a cache ``k, v
    [batch, kv_heads, max_len, head_dim]`` that already holds the tokens' own keys.

    Sequence b holds ``lengths[b]`` keys (int32 on the device, clamped to ``[0,
    max_len]``; default ``max_len``); its queries are the last ``query_lengths[b]`` of them
    (clamped to ``[0, tokens]``; default ``tokens``), query t at position ``p = lengths[b] -
    query_lengths[b] + t``.  It sees the keys ``j <= p`` with ``j > p - window`` (``window``
    None: all) or ``j < sinks``.  A query in front of the first key gives zeros; rows behind
    ``query_lengths[b]`` stay as they are in ``out`` and are zeros in a new output.  ``scale``
    defaults to ``1 / sqrt(head_dim)``.  fp16 or bf16, head_dim 64, 128 or 256, any strides
    (rows that are not 16-byte aligned are copied first, ``out`` is refused)."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_heads(name, t)
    if k.shape != v.shape or q.shape[3] != k.shape[3]:
        raise ValueError("k and v must have one shape, with q's head_dim")
    if not q.dtype == k.dtype == v.dtype or not q.device == k.device == v.device:
        raise ValueError("q, k and v must share dtype and device")
    _check_inference(q, k, v)
    k, v = _rows(k), _rows(v)
    return _attention("fx_window_attention", q, k.shape, (k.data_ptr(), v.data_ptr()), _strides(k) + _strides(v),
                      lengths, query_lengths, window, sinks, scale, out, 0)


class Int4KVCache:
    """Keys and values of ``batch`` sequences in 4 bits: for each group of 64 columns of a
    position a scale and a minimum in fp16, and codes that stand for ``code * scale +
    minimum`` (``include/fluxbin_attention.h`` has the format).  A new cache stands for
    zeros.  The caller keeps the lengths, as it does for a 16-bit cache."""

    def __init__(self, batch: int, kv_heads: int, max_len: int, head_dim: int, *, device="cuda"):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if batch < 1 or kv_heads < 1 or max_len < 1:
            raise ValueError("batch, kv_heads and max_len must be positive")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("Int4KVCache lives on a GPU")
        self.batch, self.kv_heads, self.max_len, self.head_dim = batch, kv_heads, max_len, head_dim
        rows = (batch, kv_heads, max_len)

        def part(shape, dtype):
            return torch.zeros(rows + shape, dtype=dtype, device=device)

        self.k_codes, self.v_codes = (part((head_dim // 2,), torch.uint8) for _ in range(2))
        self.k_scales, self.v_scales = (part((head_dim // KV4_GROUP, 2), torch.float16) for _ in range(2))

    @property
    def device(self) -> torch.device:
        return self.k_codes.device

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._parts())

    def _parts(self):
        return self.k_codes, self.k_scales, self.v_codes, self.v_scales

    def _pointers(self):
        return tuple(t.data_ptr() for t in self._parts())

    def append(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor | int, *,
               counts: torch.Tensor | None = None) -> None:
        """Quantize tokens ``t < counts[b]`` (int32 on the device; default all) of ``k, v
        [batch, kv_heads, tokens, head_dim]`` into positions ``start[b] + t`` (``start`` int32
        ``[batch]`` on the device, or one integer for all).  Positions outside the cache are
        dropped; nothing else of it changes."""
        for name, t in (("k", k), ("v", v)):
            _check_heads(name, t)
        if k.shape != v.shape or k.dtype != v.dtype or not k.device == v.device == self.device:
            raise ValueError("k and v must share shape and dtype, on the cache's device")
        batch, heads, tokens, dim = k.shape
        if (batch, heads, dim) != (self.batch, self.kv_heads, self.head_dim):
            raise ValueError("k and v must be [batch, kv_heads, tokens, head_dim] of the cache")
        _check_inference(k, v)
        start_ptr, start_all = None, 0
        if isinstance(start, torch.Tensor):
            start_ptr = _check_counts("start", start, batch, self.device)
        elif isinstance(start, int) and not isinstance(start, bool) and 0 <= start <= _LIMIT:
            start_all = start
        else:
            raise ValueError("start must be a non-negative integer or an int32 [batch] tensor")
        counts_ptr = _check_counts("counts", counts, batch, self.device)
        k, v = _rows(k), _rows(v)
        strides = (ctypes.c_longlong * 6)(*_strides(k), *_strides(v))
        rc = _on_device(self.device, _lib.library().fx_kv4_append, k.data_ptr(), v.data_ptr(), strides, start_ptr,
                        start_all, counts_ptr, *self._pointers(), batch, heads, tokens, self.max_len, dim,
                        _lib.dtype_code(k.dtype))
        if rc:
            _lib.check(rc, "fx_kv4_append")

    def restore(self, *, length: int | None = None, dtype: torch.dtype = torch.bfloat16):
        """The values that the first ``length`` positions (default all) stand for, as new
        ``k, v [batch, kv_heads, length, head_dim]`` tensors of ``dtype`` (fp16 or bf16)."""
        length = self.max_len if length is None else length
        if not isinstance(length, int) or isinstance(length, bool) or not 0 <= length <= self.max_len:
            raise ValueError("length must be an integer in [0, max_len]")
        if dtype not in _HALF:
            raise ValueError("dtype must be fp16 or bf16")
        shape = (self.batch, self.kv_heads, length, self.head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        rc = _on_device(self.device, _lib.library().fx_kv4_restore, *self._pointers(), k.data_ptr(), v.data_ptr(),
                        self.batch, self.kv_heads, self.max_len, length, self.head_dim, _lib.dtype_code(dtype))
        if rc:
            _lib.check(rc, "fx_kv4_restore")
        return k, v


def kv4_attention(q: torch.Tensor, cache: Int4KVCache, *, lengths: torch.Tensor | None = None,
                  query_lengths: torch.Tensor | None = None, window: int | None = None, sinks: int = 0,
                  scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`window_attention` over the values that an :class:`Int4KVCache` stands for."""
    _check_heads("q", q)
    if q.shape[3] != cache.head_dim or q.device != cache.device:
        raise ValueError("q must have the cache's head_dim and device")
    _check_inference(q)
    return _attention("fx_kv4_attention", q, (cache.batch, cache.kv_heads, cache.max_len), cache._pointers(), [],
                      lengths, query_lengths, window, sinks, scale, out, 1)
