"""8-bit integer operators of the encoder's layers on torch device tensors.

``quantize_rows`` (an activation and int8 rows with a scale each), ``norm_quantize`` (the
residual's addition, LayerNorm or RMS norm, int8 rows) and ``int8_linear`` (the product of int8
rows) are the pieces that ``BertEncoder(dtype="i8")`` runs its layers on; they bind
``hcr_quant_rows_device``, ``hcr_norm_quant_rows_device``, ``hcr_dequant_rows_device`` and
``hcr_int8_linear_device`` (include/hcrag.h).

Every call is enqueued on torch's current stream of the tensors' device and returns at once;
calls can be captured into graphs.  They compute no gradients: a tensor that asks for one is
refused while gradients are recorded, a forward-mode dual tensor always, and what a call writes
into (``out``, ``sum_out``, ``norm_out``) counts as modified in place.  No CPU fallback: without the
HIP library they raise.

    w = quantize_rows(weight)                       # [features, depth], once
    x = norm_quantize(y, gain, bias, residual=r, norm_out=r)
    y = int8_linear(x, w, bias=b, dtype=torch.float16)
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.autograd.forward_ad as _forward

from ._lib import (HCR_ACT_GELU, HCR_ACT_NONE, HCR_BF16, HCR_F16, HCR_F32, HCR_NORM_LAYER,
                   HCR_NORM_RMS, NORM_QUANT_ARGS, check, lib)

_DTYPE = {torch.float16: HCR_F16, torch.bfloat16: HCR_BF16, torch.float32: HCR_F32}
_ACT = {"none": HCR_ACT_NONE, "gelu": HCR_ACT_GELU}
_NORM = {"layer": HCR_NORM_LAYER, "rms": HCR_NORM_RMS}
_I8, _F32, _Tensor = torch.int8, torch.float32, torch.Tensor
_grad_on = torch.is_grad_enabled
_current_device = torch._C._cuda_getDevice            # (torch.cuda.current_device without its init check:
_current_stream = torch._C._cuda_getCurrentRawStream  # the operands are device tensors; 0.1 us against 1.4)
_new = object.__new__
_wrote = torch._C._increment_version                  # (torch.autograd.graph.increment_version of several tensors)
_pack_norm = NORM_QUANT_ARGS.pack


def _tangent(t) -> bool:
    """Whether t carries a forward-mode tangent."""
    return _forward._current_level >= 0 and _forward.unpack_dual(t).tangent is not None


# A single token's call is bound by what the host does, so the checks are one expression per
# operand, the error message is put together only when it fails, and the C functions are looked up
# once.
def _ok(t, dtypes, dim: int, device: int) -> bool:
    return (isinstance(t, _Tensor) and t.dtype in dtypes and t.dim() == dim and t.get_device() == device >= 0
            and (t.is_contiguous() or t.shape[-1] <= 1 or t.stride(-1) == 1)
            and not (t.requires_grad and _grad_on()) and (_forward._current_level < 0 or not _tangent(t)))


class _Entry:
    """A C entry point, called with torch's current stream of ``device`` as its last argument."""

    __slots__ = ("name", "fn")

    def __init__(self, name: str):
        self.name, self.fn = name, None

    def __call__(self, device: int, *args) -> None:
        fn = self.fn
        if fn is None:
            fn = self.fn = getattr(lib(), self.name)
        if device == _current_device():
            rc = fn(*args, _current_stream(device))
        else:
            with torch.cuda.device(device):
                rc = fn(*args, _current_stream(device))
        if rc:
            check(rc)


_quant = _Entry("hcr_quant_rows_device")
_norm_quant = _Entry("hcr_norm_quant_rows_device")
_dequant = _Entry("hcr_dequant_rows_device")
_linear = _Entry("hcr_int8_linear_device")


def _refuse(t, name: str, dtypes, dim: int, device: Optional[int] = None) -> None:
    """Raise what is wrong with an operand that ``_ok`` turned down."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype} is not supported here")
    if t.dim() != dim:
        raise ValueError(f"{name}: expected {dim} dimension(s), got shape {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a device tensor")
    if device is not None and t.get_device() != device:
        raise ValueError(f"{name}: on {t.device}, other operands on cuda:{device}")
    if t.requires_grad and _grad_on() or _tangent(t):
        raise ValueError(f"{name}: requires a gradient, which the int8 operators do not compute")
    raise ValueError(f"{name}: elements of a row must be contiguous")


def _device(t, name: str, dtypes, dim: int) -> int:
    """The device index of a call's first operand, checked."""
    device = t.get_device() if isinstance(t, torch.Tensor) else -1
    if not _ok(t, dtypes, dim, device):
        _refuse(t, name, dtypes, dim)
    return device


def _rows_device(r: "Int8Rows", name: str) -> int:
    """The device index of int8 rows, which a loader may have restored to the host and whose scales may
    ask for a gradient since they were wrapped."""
    device = r._q.get_device()
    if device < 0:
        _refuse(r._q, name, (_I8,), 2)
    scale = r._scale
    if scale.get_device() != device or scale.requires_grad and _grad_on() or _forward._current_level >= 0 and _tangent(scale):
        _refuse(scale, name + ".scale", (_F32,), 1, device)
    return device


def _ld(t) -> int:
    """Row stride in elements; of at most one row, any that its width allows."""
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else (cols + 15) // 16 * 16


class Int8Rows:
    """int8 rows with a scale each: ``q`` int8 [rows, cols], ``scale`` float32 [rows]; an element
    stands for ``q * scale``.  Rows start on 16 bytes (``q[:, :cols]`` of a buffer whose row length
    is a multiple of 16); what lies between a row's end and the next row is never read as a value.
    """

    __slots__ = ("_q", "_scale")
    q = property(lambda self: self._q)
    scale = property(lambda self: self._scale)

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        device = _device(q, "q", (_I8,), 2)
        if not _ok(scale, (_F32,), 1, device):
            _refuse(scale, "scale", (_F32,), 1, device)
        rows, cols = q.shape
        if scale.shape[0] != rows:
            raise ValueError(f"{rows} rows and {scale.shape[0]} scales")
        if (q.data_ptr() | (q.stride(0) if rows > 1 else 0)) & 15:
            raise ValueError("q: rows must start on 16 bytes (aligned storage, row stride a multiple of 16)")
        self._q, self._scale = q, scale

    @classmethod
    def empty(cls, rows: int, cols: int, device) -> "Int8Rows":
        """Uninitialised rows on a GPU, laid out as the operators want them."""
        self = _empty_rows(cls, rows, cols, device)
        _rows_device(self, "rows")
        return self

    @property
    def shape(self):
        return self._q.shape

    @property
    def device(self):
        return self._q.device

    def dequantize(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """[rows, cols] of the values that the rows stand for, rounded to ``dtype``."""
        if dtype not in _DTYPE:
            raise ValueError(f"dtype {dtype} is not supported here")
        device = _rows_device(self, "rows")
        q = self._q
        rows, cols = q.shape
        out = q.new_empty((rows, cols), dtype=dtype)
        if rows:
            _dequant(device, q.data_ptr(), _ld(q), self._scale.data_ptr(), rows, cols, out.data_ptr(),
                     _DTYPE[dtype], cols)
        return out


def _empty_rows(cls, rows: int, cols: int, device) -> Int8Rows:
    self = _new(cls)
    self._q = torch.empty_strided((rows, cols), ((cols + 15) // 16 * 16, 1), dtype=_I8, device=device)
    self._scale = torch.empty(rows, dtype=_F32, device=device)
    return self


def _int8_out(out: Optional[Int8Rows], rows: int, cols: int, like: torch.Tensor) -> Int8Rows:
    if out is None:
        return _empty_rows(Int8Rows, rows, cols, like.device)
    if tuple(out._q.shape) != (rows, cols) or _rows_device(out, "out") != like.get_device():
        raise ValueError(f"out: {tuple(out._q.shape)} on {out._q.device}, expected {(rows, cols)} on {like.device}")
    return out


def quantize_rows(x: torch.Tensor, act: str = "none", out: Optional[Int8Rows] = None) -> Int8Rows:
    """int8 rows of ``act(x)``; x [rows, cols] float16 / bfloat16 / float32, act "none" or "gelu"
    (exact-erf form).  Weights [features, depth] are quantised per channel by the same call."""
    device = _device(x, "x", _DTYPE, 2)
    if act not in _ACT:
        raise ValueError(f"unknown activation {act!r} (none | gelu)")
    rows, cols = x.shape
    given, out = out, _int8_out(out, rows, cols, x)
    _quant(device, x.data_ptr(), _DTYPE[x.dtype], _ld(x), rows, cols, _ACT[act], out._q.data_ptr(), _ld(out._q),
           out._scale.data_ptr())
    if given is not None:
        _wrote((out._q, out._scale))
    return out


def norm_quantize(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  residual: Optional[torch.Tensor] = None, norm: str = "layer", eps: float = 1e-12,
                  sum_out: Optional[torch.Tensor] = None, norm_out: Optional[torch.Tensor] = None,
                  out: Optional[Int8Rows] = None) -> Int8Rows:
    """int8 rows of ``norm(x + residual) * weight + bias``.

    x, residual: [rows, cols] float16 / bfloat16 / float32, each of its own type; weight, bias:
    float32 [cols]; norm "layer" or "rms".  ``sum_out`` (the residual's type) receives
    ``x + residual``, ``norm_out`` (any of the three types) the normalised rows before they are
    quantised.  sum_out may be the residual itself, norm_out x or the residual itself; other
    operands must not overlap.
    """
    device = _device(x, "x", _DTYPE, 2)
    if norm not in _NORM:
        raise ValueError(f"unknown norm {norm!r} (layer | rms)")
    shape = x.shape
    rows, cols = shape
    if not _ok(weight, (_F32,), 1, device):
        _refuse(weight, "weight", (_F32,), 1, device)
    if weight.shape[0] != cols:
        raise ValueError(f"weight: {weight.shape[0]} elements, expected {cols}")
    bias_p = resid_p = sum_p = norm_p = 0
    resid_t = norm_t = HCR_F32
    resid_ld = sum_ld = norm_ld = 0
    if bias is not None:
        if not _ok(bias, (_F32,), 1, device):
            _refuse(bias, "bias", (_F32,), 1, device)
        if bias.shape[0] != cols:
            raise ValueError(f"bias: {bias.shape[0]} elements, expected {cols}")
        bias_p = bias.data_ptr()
    if residual is not None:
        resid_t, resid_ld = _rows_operand(residual, "residual", shape, device)
        resid_p = residual.data_ptr()
    if sum_out is not None:
        if residual is None or sum_out.dtype != residual.dtype:
            raise ValueError("sum_out needs a residual of the same dtype")
        _, sum_ld = _rows_operand(sum_out, "sum_out", shape, device)
        sum_p = sum_out.data_ptr()
    if norm_out is not None:
        norm_t, norm_ld = _rows_operand(norm_out, "norm_out", shape, device)
        norm_p = norm_out.data_ptr()
    given, out = out, _int8_out(out, rows, cols, x)
    q = out._q
    _norm_quant(device, _pack_norm(x.data_ptr(), _ld(x), resid_p, resid_ld, weight.data_ptr(), bias_p, sum_p, sum_ld,
                                   norm_p, norm_ld, q.data_ptr(), _ld(q), out._scale.data_ptr(), rows, cols,
                                   _DTYPE[x.dtype], resid_t, norm_t, _NORM[norm], eps))
    if given is not None:
        _wrote((q, out._scale))
    if sum_out is not None:
        _wrote((sum_out,))
    if norm_out is not None:
        _wrote((norm_out,))
    return out


def _rows_operand(t, name: str, shape, device: int):
    """(dtype, row stride) of a [rows, cols] operand of a floating type."""
    if not _ok(t, _DTYPE, 2, device):
        _refuse(t, name, _DTYPE, 2, device)
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    return _DTYPE[t.dtype], _ld(t)


def int8_linear(x: Int8Rows, w: Int8Rows, bias: Optional[torch.Tensor] = None,
                dtype: torch.dtype = torch.float16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x . w^T + bias``: x [rows, depth], w [features, depth], bias float32 [features] ->
    [rows, features] in ``dtype`` (or into ``out``).  The integer sums are exact."""
    if not isinstance(x, Int8Rows) or not isinstance(w, Int8Rows):
        raise ValueError("x and w: expected Int8Rows (quantize_rows makes them)")
    xq, wq = x._q, w._q
    rows, depth = xq.shape
    features, depth_w = wq.shape
    device = _rows_device(x, "x")
    if depth_w != depth:
        raise ValueError(f"x has depth {depth}, w {depth_w}")
    if _rows_device(w, "w") != device:
        raise ValueError(f"w: on {wq.device}, x on {xq.device}")
    bias_p = None
    if bias is not None:
        if not _ok(bias, (_F32,), 1, device):
            _refuse(bias, "bias", (_F32,), 1, device)
        if bias.shape[0] != features:
            raise ValueError(f"bias: {bias.shape[0]} elements, expected {features}")
        bias_p = bias.data_ptr()
    if out is None:
        code = _DTYPE.get(dtype)
        if code is None:
            raise ValueError(f"dtype {dtype} is not supported here")
        given, out = False, xq.new_empty((rows, features), dtype=dtype)
        ldo = features
    else:
        given = True
        code, ldo = _rows_operand(out, "out", (rows, features), device)
    _linear(device, xq.data_ptr(), _ld(xq), x._scale.data_ptr(), rows, wq.data_ptr(), _ld(wq), w._scale.data_ptr(),
            features, depth, bias_p, out.data_ptr(), code, ldo)
    if given:
        _wrote((out,))
    return out


__all__ = ["Int8Rows", "quantize_rows", "norm_quantize", "int8_linear"]
