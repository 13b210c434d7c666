"""Linears whose activations and weights are 8-bit integers, and the rows that feed them.

No reference counterpart: the reference's Linears keep 16-bit activations
(``w3_lut_deployment.py:190-359``, ``deployment.py:182-297``).  Here a row of activations (a
token) and a row of the weight (an output channel) are 8-bit codes with an fp32 scale each, the
products run on the int8 matrix cores with exact sums, and what produces a Linear's input can
write it as codes at once: :func:`add_rms_norm_int8` in front of q|k|v and gate|up,
:func:`silu_mul_int8` in front of down, :func:`quantize_int8` elsewhere.
:class:`PackedInt8Linear` is the module, which quantizes its own 16-bit input: a model of them
does so in every Linear, ``NativeDecodeSession``'s steps take the operators instead.
``include/fluxbin_int8.h`` has the format.

Every call goes to the HIP kernels on the current stream of the tensors' device; there is no
CPU substitute, no backward pass and no forward-mode derivative, and calls are not traced.
Nothing synchronises, so calls can be captured into a HIP graph.
"""
from __future__ import annotations

from functools import lru_cache

import torch
from torch import nn
from torch.autograd.graph import increment_version
from torch.nn import functional as F

from . import _lib
from .cached_attention import _current_device, _refuse_records
from .packed_linear import PACKED_M1, PACKED_SMALL_M, DENSE_FALLBACK, PackedLinearBase, replace_linears_atomically

_HALF = (torch.float16, torch.bfloat16)
_OUT = (torch.float16, torch.bfloat16, torch.float32)
MAX_IN_FEATURES = 131056  # sums of so many products of codes stay within 32 bits
# The library's limits, checked here on the whole number: its size arguments are 32 bits wide, and
# the binding would drop the bits above them without a word.
MAX_ROWS, MAX_COLUMNS = 1 << 21, 1 << 20
MAX_OUT_FEATURES = 1 << 20
_STEP = 16                # the module's rows are whole 16 bytes
_ROW_LIMIT = 1 << 22      # bytes between two rows that every product reads in place
_WHAT = "an 8-bit operator"

_BF16, _FP16, _INT8, _FP32 = torch.bfloat16, torch.float16, torch.int8, torch.float32
_CODES = {dtype: _lib.dtype_code(dtype) for dtype in _OUT}


@lru_cache(maxsize=4096)
def _workspace_bytes(m: int, n: int, k: int, loose: int) -> int:
    return _lib.library().fx_int8_gemm_workspace_bytes(m, n, k, loose)


@lru_cache(maxsize=4096)
def _linear_workspace_bytes(m: int, n: int, k: int) -> int:
    return _lib.library().fx_int8_linear_workspace_bytes(m, n, k)


def _new(shape, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """``torch.empty``, whose own way to the same memory takes 0.9 us longer."""
    if len(shape) == 2:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=device)
    if len(shape) == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def _launch(name: str, index: int, *args) -> None:
    """The library call on GPU ``index`` and its current stream."""
    call = getattr(_lib.library(), name)
    if _current_device() == index:
        rc = call(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, _stream_of(index))
    if rc:
        _lib.check(rc, name)


_stream_of = _lib._raw_stream or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _refuse(*tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("8-bit operators have no backward pass; call them under torch.no_grad()")
    _refuse_records(*tensors, what=_WHAT)


def _rows_of(t: torch.Tensor) -> tuple[int, int] | None:
    """(rows, elements between rows) of ``t [..., columns]`` where its rows lie evenly in memory
    with contiguous columns, else None."""
    shape = t.shape
    columns = shape[-1]
    if t.is_contiguous():
        return t.numel() // columns, columns
    strides = t.stride()
    if strides[-1] != 1 and columns > 1:
        return None
    if len(shape) == 2:
        return shape[0], strides[0]
    rows, step = 1, columns
    for n, s in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n == 1:
            continue
        if rows == 1:
            step = s
        elif s != rows * step:
            return None
        rows *= n
    return rows, step


def _check_sizes(t: torch.Tensor, name: str) -> None:
    """``t [..., columns]``, columns not 0, is within what one call takes."""
    columns = t.shape[-1]
    if columns > MAX_COLUMNS or t.numel() > MAX_ROWS * columns:
        raise ValueError(f"{name} must have at most {MAX_ROWS} rows of at most {MAX_COLUMNS} columns, "
                         f"got {t.numel() // columns} of {columns}")


def _half_input(t: torch.Tensor, name: str, like: torch.Tensor | None = None) -> tuple[torch.Tensor, int, int]:
    """``t`` or a copy of it as the kernels read it, its row count and row stride."""
    dtype, shape = t.dtype, t.shape
    if not t.is_cuda or (dtype is not _BF16 and dtype is not _FP16):
        _lib.require_gpu_tensor(t, name)
        raise ValueError(f"{name} must be fp16 or bf16")
    if not shape or shape[-1] < 1:
        raise ValueError(f"{name} must have shape [..., columns] with columns to hold")
    if like is not None and (shape != like.shape or dtype is not like.dtype or t.get_device() != like.get_device()):
        raise ValueError(f"{name} must have the input's shape, dtype and device")
    _check_sizes(t, name)
    if t.is_neg():
        t = t.resolve_neg()
    found = _rows_of(t)
    if found is None:
        t = t.contiguous()
        found = _rows_of(t)
    return t, *found


def _code_outputs(shape: torch.Size, device: torch.device, out) -> tuple[torch.Tensor, torch.Tensor, int]:
    """codes, scales and the codes' row stride: new ones, or the caller's checked."""
    if out is None:
        return _new(shape, _INT8, device), _new(shape[:-1], _FP32, device), shape[-1]
    codes, scales = out
    _refuse(scales)
    if codes.shape != shape or codes.dtype is not _INT8 or codes.device != device:
        raise ValueError("out's codes must be int8 of the input's shape on its device")
    if (scales.shape != shape[:-1] or scales.dtype is not _FP32 or scales.device != device
            or not scales.is_contiguous() or scales.is_neg()):
        raise ValueError("out's scales must be contiguous fp32 of the input's leading shape on its device")
    found = _rows_of(codes)
    if found is None or (found[0] > 1 and found[1] < shape[-1]):
        raise ValueError("out's codes must have contiguous rows, each its own memory")
    return codes, scales, found[1]


def quantize_int8(x: torch.Tensor, *, out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Each row of ``x [..., columns]`` (fp16 or bf16) as ``codes`` (int8, x's shape) and ``scales``
    (fp32, x's leading shape): with a the row's largest magnitude, code = round(127 x / a), ties to
    even, scale = a / 127.  A row with an infinity or NaN stands for NaN (its scale is NaN).  At most
    2^21 rows of 2^20 columns, here and in the calls below.  ``out`` gives both their memory, none of
    it an input's."""
    _refuse(x)
    x, rows, stride = _half_input(x, "x")
    shape, device = x.shape, x.device
    codes, scales, code_stride = _code_outputs(shape, device, out)
    columns = shape[-1]
    _launch("fx_int8_quantize", device.index, x.data_ptr(), stride, codes.data_ptr(), code_stride, scales.data_ptr(), rows,
            columns, columns, _CODES[x.dtype])
    if out is not None:
        increment_version((codes, scales))  # a graph that saved the memory before refuses its backward, as for torch's own out=
    return codes, scales


def dequantize_int8(codes: torch.Tensor, scales: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that rows of codes stand for: ``codes * scales[..., None]`` as a new ``dtype`` (fp16,
    bf16 or fp32) tensor."""
    _check_codes(codes, scales, "codes", "scales")
    if dtype not in _OUT:
        raise ValueError("dtype must be fp16, bf16 or fp32")
    _refuse(codes, scales)
    if codes.shape[-1] < 1:
        raise ValueError("codes must have shape [..., columns] with columns to hold")
    _check_sizes(codes, "codes")
    found = _rows_of(codes)
    if found is None:
        codes = codes.contiguous()
        found = _rows_of(codes)
    scales = scales.resolve_neg().contiguous()
    out = _new(codes.shape, dtype, codes.device)
    columns = codes.shape[-1]
    _launch("fx_int8_restore", codes.get_device(), codes.data_ptr(), found[1], scales.data_ptr(), out.data_ptr(), columns,
            found[0], columns, _lib.dtype_code(dtype))
    return out


def _norm(x, residual, weight, eps, residual_out, out):
    _refuse(x, residual, weight, residual_out)
    x, rows, stride = _half_input(x, "hidden_states")
    shape, dtype, device = x.shape, x.dtype, x.device
    columns = shape[-1]
    if weight.shape != (columns,) or weight.dtype is not dtype or weight.get_device() != device.index:
        raise ValueError("weight must have shape [hidden] and the input's dtype and device")
    if weight.is_neg() or not weight.is_contiguous():
        weight = weight.resolve_neg().contiguous()
    r_ptr = s_ptr = None
    r_stride = s_stride = 0
    written = ()
    if residual is not None:
        residual, _, r_stride = _half_input(residual, "residual", x)
        if residual_out is None:
            residual_out, s_stride = _new(shape, dtype, device), columns
        else:
            if residual_out.shape != shape or residual_out.dtype is not dtype or residual_out.device != device:
                raise ValueError("residual_out must have the input's shape, dtype and device")
            found = None if residual_out.is_neg() else _rows_of(residual_out)
            if found is None or (found[0] > 1 and found[1] < columns):
                raise ValueError("residual_out must have contiguous rows, each its own memory")
            s_stride = found[1]
            written += (residual_out,)
        r_ptr, s_ptr = residual.data_ptr(), residual_out.data_ptr()
    codes, scales, code_stride = _code_outputs(shape, device, out)
    if out is not None:
        written += (codes, scales)
    _launch("fx_int8_rmsnorm", device.index, x.data_ptr(), stride, r_ptr, r_stride, s_ptr, s_stride, weight.data_ptr(),
            codes.data_ptr(), code_stride, scales.data_ptr(), rows, columns, columns, float(eps), _CODES[dtype])
    if written:
        increment_version(written)
    return codes, scales, residual_out


def rms_norm_int8(hidden_states: torch.Tensor, weight: torch.Tensor, eps: float, *,
                  out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """:func:`quantize_int8` of ``weight * x * rsqrt(mean(x^2) + eps)`` over the last axis, in one launch
    and without the rounding to 16 bits between the two: ``(codes, scales)``."""
    return _norm(hidden_states, None, weight, eps, None, out)[:2]


def add_rms_norm_int8(hidden_states: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, *,
                      residual_out: torch.Tensor | None = None,
                      out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """:func:`rms_norm_int8` of ``residual_out = round(hidden_states + residual)``, which is written too:
    ``(codes, scales, residual_out)``.  ``residual_out`` may be ``hidden_states`` or ``residual`` itself;
    otherwise it shares no memory with them."""
    if residual is None:
        raise ValueError("residual must be a tensor")
    return _norm(hidden_states, residual, weight, eps, residual_out, out)


def silu_mul_int8(gate: torch.Tensor, up: torch.Tensor, *, out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """:func:`quantize_int8` of ``silu(gate) * up`` (formed in fp32), in one launch.  ``gate`` and ``up``
    may be the halves of one product's output."""
    _refuse(gate, up)
    gate, rows, stride = _half_input(gate, "gate")
    up, _, up_stride = _half_input(up, "up", gate)
    shape, device = gate.shape, gate.device
    codes, scales, code_stride = _code_outputs(shape, device, out)
    columns = shape[-1]
    _launch("fx_int8_silu_mul", device.index, gate.data_ptr(), stride, up.data_ptr(), up_stride, codes.data_ptr(), code_stride,
            scales.data_ptr(), rows, columns, columns, _CODES[gate.dtype])
    if out is not None:
        increment_version((codes, scales))
    return codes, scales


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, name: str, scales_name: str) -> None:
    if codes.dtype is not _INT8 or not codes.is_cuda or not codes.shape:
        _lib.require_gpu_tensor(codes, name)
        raise ValueError(f"{name} must be int8 [..., columns]")
    if scales.dtype is not _FP32 or scales.shape != codes.shape[:-1] or scales.get_device() != codes.get_device():
        raise ValueError(f"{scales_name} must be fp32, one for each row of {name}, on its device")


def _code_rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int, bool]:
    """``t`` (or a copy whose rows lie evenly), its rows and row stride, and whether the products
    read its rows in place however many they are (whole 16 bytes at 16-byte boundaries)."""
    found = _rows_of(t)
    if found is None or (found[0] > 1 and 0 != found[1] < t.shape[-1]):
        t = t.contiguous()
        found = _rows_of(t)
    rows, stride = found
    loose = (t.shape[-1] | t.data_ptr()) & 15 or (rows > 1 and (stride & 15 or stride > _ROW_LIMIT))
    return t, rows, stride, bool(loose)


def int8_matmul(a: torch.Tensor, a_scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *,
                bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[..., n] = (sum_k a[..., k] weight[n, k]) * a_scales[...] * weight_scales[n] + bias[n]``.

    ``a [..., K]`` and ``weight [N, K]`` int8, their scales fp32 (one per row), ``bias [N]`` and the
    result of ``dtype`` (fp16, bf16 or fp32).  The sum is exact (K up to 131056); scales and bias are
    applied in fp32, rounded once.  At most 2^21 rows and N up to 2^20.  Rows that lie at 16-byte
    boundaries are read in place where K is a multiple of 16, and any where ``a`` has at most 32; others
    are copied in every call (512 x 4096 x 4090 31 us, 4096 columns 18).  ``out`` shares no memory with
    the inputs."""
    shape, wide, index = a.shape, weight.shape, a.get_device()
    if not (a.dtype is _INT8 and weight.dtype is _INT8 and a_scales.dtype is _FP32 and weight_scales.dtype is _FP32
            and index >= 0 and a_scales.get_device() == index and weight.get_device() == index
            and weight_scales.get_device() == index and shape and len(wide) == 2 and shape[-1] == wide[1]
            and a_scales.shape == shape[:-1] and weight_scales.shape == wide[:1]):
        _check_codes(a, a_scales, "a", "a_scales")
        _check_codes(weight, weight_scales, "weight", "weight_scales")
        raise ValueError("weight must be [N, K] with a's K, on a's device")
    n, k = wide
    device = a.device
    if not 1 <= k <= MAX_IN_FEATURES or not 1 <= n <= MAX_OUT_FEATURES or a.numel() > MAX_ROWS * k:
        raise ValueError(f"K must be in [1, {MAX_IN_FEATURES}], N positive and at most {MAX_OUT_FEATURES} and a of at "
                         f"most {MAX_ROWS} rows, got K {k}, N {n} and {a.numel() // max(k, 1)} rows")
    code = _CODES.get(dtype)
    if code is None:
        raise ValueError("dtype must be fp16, bf16 or fp32")
    if bias is not None:
        if bias.shape != (n,) or bias.dtype is not dtype or bias.get_device() != index:
            raise ValueError("bias must have shape [N], the result's dtype and a's device")
        bias = bias.resolve_neg().contiguous()
    _refuse(a_scales, weight_scales, bias, out)
    shape = (*shape[:-1], n)
    given = out is not None
    if not given:
        out = _new(shape, dtype, device)
        out_stride = n
    else:
        if out.shape != shape or out.dtype is not dtype or out.get_device() != index or out.is_neg():
            raise ValueError("out must have shape [..., N], the result's dtype and a's device")
        found = _rows_of(out)
        if found is None or (found[0] > 1 and found[1] < n):
            raise ValueError("out must have contiguous rows, each its own memory")
        out_stride = found[1]
    a_ptr, w_ptr = a.data_ptr(), weight.data_ptr()
    loose = 0
    if a.is_contiguous() and weight.is_contiguous() and not (k | a_ptr | w_ptr) & 15:
        rows, a_stride, w_stride = a.numel() // k, k, k
    else:
        a, rows, a_stride, a_loose = _code_rows(a)
        weight, _, w_stride, w_loose = _code_rows(weight)
        a_ptr, w_ptr, loose = a.data_ptr(), weight.data_ptr(), a_loose + 2 * w_loose
    if not a_scales.is_contiguous() or a_scales.is_neg():
        a_scales = a_scales.resolve_neg().contiguous()
    if not weight_scales.is_contiguous() or weight_scales.is_neg():
        weight_scales = weight_scales.resolve_neg().contiguous()
    nbytes = _workspace_bytes(rows, n, k, loose)
    workspace = _new((nbytes,), torch.uint8, device) if nbytes else None
    _launch("fx_int8_gemm", index, a_ptr, a_stride, a_scales.data_ptr(), w_ptr, w_stride,
            weight_scales.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), out_stride,
            None if workspace is None else workspace.data_ptr(), nbytes, rows, n, k, code)
    if given:
        increment_version(out)
    return out


def quantize_weight_int8(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A Linear's weight ``[O, K]`` as codes and scales, one scale per output channel: the kernel's
    codes for a 16-bit weight on a GPU, the same formula in 64 bits elsewhere."""
    if weight.ndim != 2:
        raise ValueError("weight must have shape [O, K]")
    weight = weight.detach()
    if weight.is_cuda and weight.dtype in _HALF:
        codes, scales = quantize_int8(weight)
        if not bool(torch.isfinite(scales).all()):
            raise ValueError("weight must be finite")
        return codes, scales
    wide = weight.double()
    top = wide.abs().amax(1, keepdim=True)
    if not bool(torch.isfinite(top).all()):
        raise ValueError("weight must be finite")
    codes = torch.round(wide * 127 / torch.where(top > 0, top, torch.ones_like(top))).to(torch.int8)
    return codes, (top[:, 0] / 127).float()


class PackedInt8Linear(PackedLinearBase):
    """Linear with 8-bit weights (a scale per output channel) and activations (a scale per row,
    formed in the call).

    ``codes [O, K]`` int8 and ``scales [O]`` fp32 stand for the weight ``codes * scales[:, None]``; the
    module holds copies of them (and of a bias, which is rounded to the result's type where its own is
    another).
    fp16 or bf16 rows on the GPU, up to 2^21 of them, take the kernels, by up to 2^20 outputs; the rest
    is refused unless ``fallback='dense'`` (``F.linear`` with the weight that the codes stand for).  Routes, counters
    and the bound one-row decode call are those of ``packed_linear.PackedLinearBase``."""

    max_packed_rows = MAX_ROWS
    bias_in_kernel = True

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, *, bias: torch.Tensor | None = None,
                 fallback: str = "error"):
        super().__init__()
        if codes.ndim != 2 or codes.dtype is not torch.int8 or not 1 <= codes.shape[1] <= MAX_IN_FEATURES or (
                codes.shape[0] < 1):
            raise ValueError(f"codes must be int8 [O, K], K at most {MAX_IN_FEATURES}")
        self.out_features, self.in_features = codes.shape
        if scales.shape != (self.out_features,) or scales.dtype is not torch.float32 or scales.device != codes.device:
            raise ValueError("scales must be fp32 [O] on the codes' device")
        if bias is not None and (bias.shape != (self.out_features,) or bias.device != codes.device):
            raise ValueError("bias must have shape [O] on the codes' device")
        self._init_protocol(fallback=fallback, bias=bias)
        # rows of whole 16 bytes, the columns behind K zero, as the kernels read them
        self._width = -(-self.in_features // _STEP) * _STEP
        padded = self._width != self.in_features
        codes = F.pad(codes.detach(), (0, self._width - self.in_features)) if padded else codes.detach()
        self.register_buffer("codes", codes.contiguous() if padded else codes.clone(memory_format=torch.contiguous_format))
        self.register_buffer("scales", scales.detach().clone(memory_format=torch.contiguous_format))

    @classmethod
    def from_linear(cls, linear: nn.Linear, *, fallback: str = "error") -> "PackedInt8Linear":
        """The Linear with its weight quantized per output channel."""
        if not isinstance(linear, nn.Linear):
            raise ValueError("from_linear takes an nn.Linear")
        codes, scales = quantize_weight_int8(linear.weight)
        return cls(codes, scales, bias=linear.bias, fallback=fallback)

    def _payload_device(self) -> torch.device:
        return self.codes.device

    def _dense_weight(self, dtype: torch.dtype) -> torch.Tensor:
        return (self.codes[:, :self.in_features].float() * self.scales[:, None]).to(dtype)

    def _load_from_state_dict(self, *args, **kwargs):
        """Tensors that ``assign=True`` puts in place of the buffers are held as the kernels read them, and
        a decode binding of the old ones ends."""
        before = list(self._buffers.values())  # (held, so that no new tensor is taken for a freed one)
        super()._load_from_state_dict(*args, **kwargs)
        for name in ("codes", "scales", "bias"):
            t = self._buffers[name]
            if t is not None and (not t.is_contiguous() or t.is_neg() or t.data_ptr() % 16):
                self._buffers[name] = t.detach().clone(memory_format=torch.contiguous_format)
        if any(t is not b for t, b in zip(self._buffers.values(), before)):
            self.clear_prepared_decode()

    def _check_before_call(self) -> None:
        codes, scales, bias = self._tensor("codes"), self._tensor("scales"), self._tensor("bias")
        if scales.dtype is not torch.float32 or codes.dtype is not torch.int8:
            raise ValueError("codes or scales were cast; move devices without dtype conversion")
        index = codes.get_device()
        if scales.get_device() != index or (bias is not None and bias.get_device() != index):
            raise ValueError("codes, scales and bias must be on one device")

    def _check_before_bind(self, device: torch.device) -> None:
        if self.scales.device != device or not self.codes.is_contiguous():
            raise ValueError("contiguous same-device codes and scales required")
        self._check_before_call()

    def _packed_kernel(self, rows: int, device: torch.device):
        """The rows quantized and multiplied, through a workspace of this callable's own."""
        codes, scales, bias = self._tensor("codes"), self._tensor("scales"), self._tensor("bias")
        width, k, o = self._width, self.in_features, self.out_features
        if rows > MAX_ROWS or o > MAX_OUT_FEATURES:
            raise ValueError(f"at most {MAX_ROWS} rows by {MAX_OUT_FEATURES} outputs take the kernels, got {rows} by {o}")
        nbytes = _linear_workspace_bytes(rows, o, k)
        workspace = _new((nbytes,), torch.uint8, device) if nbytes else None
        index = device.index

        def run(x2: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
            code = _CODES[x2.dtype]
            added = bias if bias is None or bias.dtype == out.dtype else bias.to(out.dtype)
            _launch("fx_int8_linear", index, x2.data_ptr(), x2.stride(0), code, codes.data_ptr(), width,
                    scales.data_ptr(), None if added is None else added.data_ptr(), out.data_ptr(), o,
                    workspace if workspace is None else workspace.data_ptr(), nbytes, rows, o, k, _CODES[out.dtype])
            return out
        return run

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self._decode_binding is not None:
            _refuse_records(x, what=_WHAT)
            return self._decode_binding(x.resolve_neg() if x.is_neg() else x)
        if torch.is_grad_enabled():
            raise RuntimeError("packed inference requires no_grad/inference_mode")
        shape, k, dtype = x.shape, self.in_features, x.dtype
        if len(shape) < 2 or shape[-1] != k:
            raise ValueError("expected [...,K] input")
        self._check_before_call()
        device = self._tensor("codes").device
        rows = x.numel() // k
        if (not x.is_cuda or (dtype is not _BF16 and dtype is not _FP16) or x.get_device() != device.index
                or rows > self.max_packed_rows or self.out_features > MAX_OUT_FEATURES):
            if self.fallback != "dense":
                raise ValueError("unsupported input; enable explicit dense fallback if needed")
            self._count(DENSE_FALLBACK)
            return self._dense_linear(x)
        _refuse_records(x, what=_WHAT)
        self._count(PACKED_M1 if rows == 1 else PACKED_SMALL_M)
        out = _new((*shape[:-1], self.out_features), dtype, device)
        if rows:
            if x.is_neg():
                x = x.resolve_neg()
            if len(shape) != 2 or not x.is_contiguous():
                x = x.reshape(rows, k).contiguous()
            self._packed_kernel(rows, device)(x, out)
        return out


def replace_int8_block_linears(block: nn.Module, *, fallback: str = "error") -> list[str]:
    """Replace the seven Qwen3 Linears of one block by :class:`PackedInt8Linear` of their weights;
    every replacement is built before the block is touched.  Returns their names."""
    from .qwen3 import QWEN3_LINEAR_MODULES

    return replace_linears_atomically(
        block, [(name, PackedInt8Linear.from_linear(block.get_submodule(name), fallback=fallback))
                for name in QWEN3_LINEAR_MODULES])
