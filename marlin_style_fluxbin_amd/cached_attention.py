"""Attention over long caches: a sliding window with sinks, and a cache held in 4 bits.

No reference counterpart: the reference's decode runs stock SDPA over a full 16-bit
static cache of one sequence (``static_decode.py:67-81``), which this package serves with
``fx_decode_attention``.  The operators here take what that path does not: batches at
ragged lengths, prompts and chunks of any number of tokens, a window of the last keys
with a few first tokens that stay visible, and an :class:`Int4KVCache` in a quarter of the
bytes (4.5 bits a value).  Every call goes to the HIP kernels behind
``include/fluxbin_attention.h`` on the current stream of the tensors' device; there is no
CPU substitute, no backward pass and no forward-mode derivative, and calls are not traced
(what would need one of them is refused).  Lengths stay on the device, so calls can be captured
into a HIP graph and follow the lengths of each replay.
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch
from torch.autograd import forward_ad

from . import _lib

_HALF = (torch.float16, torch.bfloat16)
HEAD_DIMS = (64, 128, 256)
KV4_GROUP = 64  # columns that share a scale and a minimum
_LIMIT = 2**31 - 1


@lru_cache(maxsize=256)
def _workspace_bytes(*sizes) -> int:
    return _lib.library().fx_cached_attention_workspace_bytes(*sizes)


def _strides(t: torch.Tensor) -> tuple[int, ...]:
    """(batch, head, row) strides; an axis of one element never moves."""
    return tuple(0 if n == 1 else s for n, s in zip(t.shape, t.stride()[:3]))


def _rows(t: torch.Tensor, copy: bool = True):
    """``t`` (or a copy of it, or None without ``copy``) as the kernels read it, rows of
    contiguous columns at 16-byte boundaries: the tensor, its address and its strides."""
    s, p = t.stride(), t.data_ptr()
    lazy = t.is_neg()
    if s[3] == 1 and not (s[0] | s[1] | s[2]) & 7 and not p & 15 and not lazy:
        return t, p, s[:3]
    s = _strides(t)
    if t.stride(3) != 1 or (s[0] | s[1] | s[2]) & 7 or p & 15 or lazy:
        if not copy:
            return None
        t = t.resolve_neg()
        t = t.contiguous()
        t = t.clone() if t.data_ptr() & 15 else t
        s = _strides(t)
    return t, t.data_ptr(), s


def _disjoint(shape, strides) -> bool:
    """No element of the rows at these (batch, head, row) strides is another's memory."""
    b, h, t, dim = shape
    s0, s1, s2 = strides
    if dim <= s1 and h * s1 <= s2 and t * s2 <= s0 or dim <= s2 and t * s2 <= s1 and h * s1 <= s0:
        return True  # in the order of the axes, either way
    axes = sorted((s, n) for s, n in ((s0, b), (s1, h), (s2, t)) if n != 1)
    extent = dim
    for s, n in axes:  # each axis behind all that lies within its step
        if s < extent:
            break
        extent += s * (n - 1)
    else:
        return True
    if any(n == 0 for _, n in axes):
        return True
    starts = torch.zeros(1, dtype=torch.int64, device="cpu")
    for s, n in axes:  # rows in each other's gaps: every one of them
        starts = (starts[:, None] + s * torch.arange(n, dtype=torch.int64, device="cpu")).flatten()
    return bool((starts.sort().values.diff() >= dim).all())


_BF16, _FP16 = torch.bfloat16, torch.float16


def _check_heads(**tensors: torch.Tensor) -> torch.dtype:
    """Four axes, one GPU, one half dtype (returned); the message names what is not."""
    first = next(iter(tensors.values()))
    for name, t in tensors.items():
        if t.ndim != 4:
            raise ValueError(f"{name} must have shape [batch, heads, tokens, head_dim]")
        _lib.require_gpu_tensor(t, name)
        if t.dtype not in _HALF:
            raise ValueError(f"{name} must be fp16 or bf16")
        if t.dtype != first.dtype or t.device != first.device:
            raise ValueError(f"{' and '.join(tensors)} must share dtype and device")
    return first.dtype


def _check_head_dim(dim: int) -> None:
    if dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {dim}")


def _counts(name: str, t: torch.Tensor, batch: int, index: int) -> int:
    if t.dtype is not torch.int32 or t.shape != (batch,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [batch] tensor on the device of the cache")
    return t.data_ptr()


def _no_gradient() -> None:
    raise ValueError("cached attention has no backward pass; call it under torch.no_grad()")


# torch's own queries of what records a call: jit.trace, make_fx and its pre-dispatch form.
# They are internal; a torch without one has nothing of its kind in force.
_PROXY = getattr(getattr(torch._C, "_TorchDispatchModeKey", None), "PROXY", None)
_PRE_DISPATCH = getattr(getattr(torch._C, "DispatchKey", None), "PreDispatch", None)
_jit_tracer = getattr(torch._C, "_get_tracing_state", lambda: None)
_mode_count = getattr(torch._C, "_len_torch_dispatch_stack", lambda: 0)
_mode_of = getattr(torch._C, "_get_dispatch_mode", lambda key: None)
_key_included = getattr(torch._C, "_dispatch_tls_is_dispatch_key_included", lambda key: False)


def _refuse_records(*tensors: torch.Tensor | None, what: str = "cached attention") -> None:
    """What a kernel called by address writes carries no tangent, and a tracer's record of the
    call would hold its output's allocation alone.  (torch.compile breaks its graph at the call
    and runs it as it is.)"""
    if torch.compiler.is_dynamo_compiling():
        return
    if (_jit_tracer() is not None or (_mode_count() and _mode_of(_PROXY) is not None)
            or _key_included(_PRE_DISPATCH)):
        raise ValueError(f"{what} cannot be traced: its kernels would be missing from the record")
    if getattr(forward_ad, "_current_level", -1) >= 0:
        if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
            raise ValueError(f"{what} has no forward-mode derivative: an argument carries a tangent")


# (the arguments are on a GPU, so torch has initialised it)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(name: str, device: torch.device, *args) -> None:
    """The library call with ``device`` current (kernels launch on the current device)."""
    call = getattr(_lib.library(), name)
    if _current_device() == device.index:
        rc = call(*args, _lib.stream_handle(device))
    else:
        with torch.cuda.device(device):
            rc = call(*args, _lib.stream_handle(device))
    if rc:
        _lib.check(rc, name)


_Strides6, _Strides12 = ctypes.c_longlong * 6, ctypes.c_longlong * 12


def _attention(name, q, cache, cache_args, cache_strides, lengths, query_lengths, window, sinks, scale, out, kv4):
    """Checks and call shared by the two caches; ``cache`` is (batch, kv heads, max_len)."""
    shape, dtype, device = q.shape, q.dtype, q.device
    batch, heads, tokens, dim = shape
    cache_batch, kv_heads, max_len = cache
    if cache_batch != batch:
        raise ValueError(f"q and the cache disagree on the batch: {batch} and {cache_batch}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a positive multiple of KV heads ({kv_heads})")
    if window is None:
        window = 0
    elif type(window) is not int or window < 1:
        raise ValueError("window must be None or a positive integer")
    if type(sinks) is not int or sinks < 0:
        raise ValueError("sinks must be a non-negative integer")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    elif not 0.0 < float(scale) < 3.4e38:
        raise ValueError("scale must be positive and finite")
    # no key lies beyond max_len, so neither a window nor sinks need to
    window, sinks = min(window, max_len + 1), min(sinks, max_len)
    index = device.index
    lengths_ptr = None if lengths is None else _counts("lengths", lengths, batch, index)
    counts_ptr = None if query_lengths is None else _counts("query_lengths", query_lengths, batch, index)
    if out is None:
        make = torch.empty if query_lengths is None else torch.zeros
        out = make((batch, tokens, heads, dim), dtype=dtype, device=device).transpose(1, 2)
    elif out.shape != shape or out.dtype is not dtype or out.get_device() != index:
        raise ValueError("out must have q's shape, dtype and device")
    elif out.requires_grad and torch.is_grad_enabled():
        _no_gradient()
    rows = _rows(out, copy=False)
    if rows is None or not _disjoint(shape, rows[2]):
        raise ValueError("out must have contiguous 16-byte aligned rows, each its own memory")
    _, out_ptr, out_strides = rows
    q, q_ptr, q_strides = _rows(q)
    code = _lib.dtype_code(dtype)
    nbytes = _workspace_bytes(batch, heads, kv_heads, tokens, max_len, dim, window, sinks, code, kv4)
    workspace = workspace_ptr = None
    if nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        workspace_ptr = workspace.data_ptr()
    strides = (_Strides6 if kv4 else _Strides12)(*q_strides, *cache_strides, *out_strides)
    _launch(name, device, q_ptr, *cache_args, out_ptr, strides, lengths_ptr, counts_ptr, workspace_ptr, nbytes,
            batch, heads, kv_heads, tokens, max_len, dim, window, sinks, scale, code)
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
    (rows that are not 16-byte aligned are copied first, ``out`` is refused; positions of a cache
    at most 2^22 elements apart)."""
    dtype, index = q.dtype, q.get_device()
    if not (q.ndim == k.ndim == v.ndim == 4 and index >= 0 and (dtype is _BF16 or dtype is _FP16)
            and k.dtype is dtype and v.dtype is dtype and k.get_device() == index and v.get_device() == index):
        _check_heads(q=q, k=k, v=v)
    shape = k.shape
    if v.shape != shape or q.shape[3] != shape[3]:
        raise ValueError("k and v must have one shape, with q's head_dim")
    _check_head_dim(shape[3])
    if (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        _no_gradient()
    _refuse_records(q, k, v, out)
    k, k_ptr, k_strides = _rows(k)
    v, v_ptr, v_strides = _rows(v)
    return _attention("fx_window_attention", q, shape[:3], (k_ptr, v_ptr), (*k_strides, *v_strides), lengths,
                      query_lengths, window, sinks, scale, out, 0)


class Int4KVCache:
    """Keys and values of ``batch`` sequences in 4 bits: for each group of 64 columns of a
    position a scale and a minimum in fp16, and codes that stand for ``code * scale +
    minimum`` (``include/fluxbin_attention.h`` has the format).  A new cache stands for
    zeros.  The caller keeps the lengths, as it does for a 16-bit cache."""

    def __init__(self, batch: int, kv_heads: int, max_len: int, head_dim: int, *, device="cuda"):
        _check_head_dim(head_dim)
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
        return (self.k_codes.data_ptr(), self.k_scales.data_ptr(), self.v_codes.data_ptr(), self.v_scales.data_ptr())

    def append(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor | int, *,
               counts: torch.Tensor | None = None) -> None:
        """Quantize tokens ``t < counts[b]`` (int32 on the device; default all) of ``k, v
        [batch, kv_heads, tokens, head_dim]`` into positions ``start[b] + t`` (``start`` int32
        ``[batch]`` on the device, or one integer for all).  Positions outside the cache are
        dropped; nothing else of it changes."""
        dtype, device = k.dtype, self.device
        index = device.index
        if not (k.ndim == v.ndim == 4 and k.get_device() == index and v.get_device() == index
                and (dtype is _BF16 or dtype is _FP16) and v.dtype is dtype):
            _check_heads(k=k, v=v)
            raise ValueError("k and v must be on the cache's device")
        shape = k.shape
        if v.shape != shape:
            raise ValueError("k and v must share their shape")
        batch, heads, tokens, dim = shape
        if (batch, heads, dim) != (self.batch, self.kv_heads, self.head_dim):
            raise ValueError("k and v must be [batch, kv_heads, tokens, head_dim] of the cache")
        if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
            _no_gradient()
        _refuse_records(k, v)
        start_ptr, start_all = None, 0
        if isinstance(start, torch.Tensor):
            start_ptr = _counts("start", start, batch, index)
        elif type(start) is int and 0 <= start <= _LIMIT:
            start_all = start
        else:
            raise ValueError("start must be a non-negative integer or an int32 [batch] tensor")
        counts_ptr = None if counts is None else _counts("counts", counts, batch, index)
        k, k_ptr, k_strides = _rows(k)
        v, v_ptr, v_strides = _rows(v)
        _launch("fx_kv4_append", device, k_ptr, v_ptr, _Strides6(*k_strides, *v_strides), start_ptr, start_all,
                counts_ptr, *self._pointers(), batch, heads, tokens, self.max_len, dim, _lib.dtype_code(dtype))

    def restore(self, *, length: int | None = None, dtype: torch.dtype = torch.bfloat16):
        """The values that the first ``length`` positions (default all) stand for, as new
        ``k, v [batch, kv_heads, length, head_dim]`` tensors of ``dtype`` (fp16 or bf16)."""
        length = self.max_len if length is None else length
        if type(length) is not int or not 0 <= length <= self.max_len:
            raise ValueError("length must be an integer in [0, max_len]")
        if dtype not in _HALF:
            raise ValueError("dtype must be fp16 or bf16")
        _refuse_records()
        shape = (self.batch, self.kv_heads, length, self.head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        _launch("fx_kv4_restore", self.device, *self._pointers(), k.data_ptr(), v.data_ptr(), self.batch, self.kv_heads,
                self.max_len, length, self.head_dim, _lib.dtype_code(dtype))
        return k, v


def kv4_attention(q: torch.Tensor, cache: Int4KVCache, *, lengths: torch.Tensor | None = None,
                  query_lengths: torch.Tensor | None = None, window: int | None = None, sinks: int = 0,
                  scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`window_attention` over the values that an :class:`Int4KVCache` stands for."""
    dtype = q.dtype
    if not (q.ndim == 4 and q.get_device() == cache.device.index and (dtype is _BF16 or dtype is _FP16)):
        _check_heads(q=q)
        raise ValueError("q must be on the cache's device")
    if q.shape[3] != cache.head_dim:
        raise ValueError("q must have the cache's head_dim")
    if q.requires_grad and torch.is_grad_enabled():
        _no_gradient()
    _refuse_records(q, out)
    return _attention("fx_kv4_attention", q, (cache.batch, cache.kv_heads, cache.max_len), cache._pointers(), (),
                      lengths, query_lengths, window, sinks, scale, out, 1)
