"""8-bit integer operators of the encoder's layers on torch device tensors.

``quantize_rows`` (an activation and int8 rows with a scale each), ``norm_quantize`` (the
residual's addition, LayerNorm or RMS norm, int8 rows) and ``int8_linear`` (the product of int8
rows) are the pieces that ``BertEncoder(dtype="i8")`` runs its layers on; they bind
``hcr_quant_rows_device``, ``hcr_norm_quant_rows_device``, ``hcr_dequant_rows_device`` and
``hcr_int8_linear_device`` (include/hcrag.h).

Every call is enqueued on torch's current stream of the tensors' device and returns at once;
calls can be captured into graphs.  They compute no gradients: a tensor that asks for one is
refused while gradients are recorded.  No CPU fallback: without the HIP library they raise.

    w = quantize_rows(weight)                       # [features, depth], once
    x = norm_quantize(y, gain, bias, residual=r, norm_out=r)
    y = int8_linear(x, w, bias=b, dtype=torch.float16)
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import (HCR_ACT_GELU, HCR_ACT_NONE, HCR_BF16, HCR_F16, HCR_F32, HCR_NORM_LAYER,
                   HCR_NORM_RMS, check, lib)

_DTYPE = {torch.float16: HCR_F16, torch.bfloat16: HCR_BF16, torch.float32: HCR_F32}
_ACT = {"none": HCR_ACT_NONE, "gelu": HCR_ACT_GELU}
_NORM = {"layer": HCR_NORM_LAYER, "rms": HCR_NORM_RMS}


def _check(t, name: str, dtypes, dim: int, device=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype} is not supported here")
    if t.dim() != dim:
        raise ValueError(f"{name}: expected {dim} dimension(s), got shape {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a device tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, other operands on {device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: elements of a row must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: requires a gradient, which the int8 operators do not compute")


def _ld(t) -> int:
    """Row stride in elements; of at most one row, any that its width allows."""
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16


def _call(device, fn, *args) -> None:
    """``fn`` with torch's current stream of ``device`` as its last argument."""
    index = device.index
    if index == torch.cuda.current_device():
        check(fn(*args, torch.cuda.current_stream(index).cuda_stream))
    else:
        with torch.cuda.device(index):
            check(fn(*args, torch.cuda.current_stream(index).cuda_stream))


class Int8Rows:
    """int8 rows with a scale each: ``q`` int8 [rows, cols], ``scale`` float32 [rows]; an element
    stands for ``q * scale``.  Rows start on 16 bytes (``q[:, :cols]`` of a buffer whose row length
    is a multiple of 16); what lies between a row's end and the next row is never read as a value.
    """

    __slots__ = ("q", "scale")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        _check(q, "q", (torch.int8,), 2)
        _check(scale, "scale", (torch.float32,), 1, q.device)
        if scale.shape[0] != q.shape[0]:
            raise ValueError(f"{q.shape[0]} rows and {scale.shape[0]} scales")
        if q.data_ptr() & 15 or _ld(q) & 15:
            raise ValueError("q: rows must start on 16 bytes (aligned storage, row stride a multiple of 16)")
        self.q, self.scale = q, scale

    @classmethod
    def empty(cls, rows: int, cols: int, device) -> "Int8Rows":
        """Uninitialised rows, laid out as the operators want them."""
        q = torch.empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=device)
        return cls(q[:, :cols], torch.empty(rows, dtype=torch.float32, device=device))

    @property
    def shape(self):
        return self.q.shape

    @property
    def device(self):
        return self.q.device

    def dequantize(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """[rows, cols] of the values that the rows stand for, rounded to ``dtype``."""
        if dtype not in _DTYPE:
            raise ValueError(f"dtype {dtype} is not supported here")
        rows, cols = self.q.shape
        out = torch.empty((rows, cols), dtype=dtype, device=self.q.device)
        if rows:
            _call(self.q.device, lib().hcr_dequant_rows_device, self.q.data_ptr(), _ld(self.q),
                  self.scale.data_ptr(), rows, cols, out.data_ptr(), _DTYPE[dtype], cols)
        return out


def _int8_out(out: Optional[Int8Rows], rows: int, cols: int, device) -> Int8Rows:
    if out is None:
        return Int8Rows.empty(rows, cols, device)
    if tuple(out.q.shape) != (rows, cols) or out.q.device != device:
        raise ValueError(f"out: {tuple(out.q.shape)} on {out.q.device}, expected {(rows, cols)} on {device}")
    return out


def quantize_rows(x: torch.Tensor, act: str = "none", out: Optional[Int8Rows] = None) -> Int8Rows:
    """int8 rows of ``act(x)``; x [rows, cols] float16 / bfloat16 / float32, act "none" or "gelu"
    (exact-erf form).  Weights [features, depth] are quantised per channel by the same call."""
    _check(x, "x", _DTYPE, 2)
    if act not in _ACT:
        raise ValueError(f"unknown activation {act!r} (none | gelu)")
    rows, cols = x.shape
    out = _int8_out(out, rows, cols, x.device)
    _call(x.device, lib().hcr_quant_rows_device, x.data_ptr(), _DTYPE[x.dtype], _ld(x), rows, cols,
          _ACT[act], out.q.data_ptr(), _ld(out.q), out.scale.data_ptr())
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
    _check(x, "x", _DTYPE, 2)
    if norm not in _NORM:
        raise ValueError(f"unknown norm {norm!r} (layer | rms)")
    rows, cols = x.shape
    dev = x.device
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None or name == "weight":
            _check(t, name, (torch.float32,), 1, dev)
            if t.shape[0] != cols:
                raise ValueError(f"{name}: {t.shape[0]} elements, expected {cols}")
    for t, name in ((residual, "residual"), (sum_out, "sum_out"), (norm_out, "norm_out")):
        if t is not None:
            _check(t, name, _DTYPE, 2, dev)
            if t.shape != x.shape:
                raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {(rows, cols)}")
    if sum_out is not None and (residual is None or sum_out.dtype != residual.dtype):
        raise ValueError("sum_out needs a residual of the same dtype")
    out = _int8_out(out, rows, cols, dev)
    _call(dev, lib().hcr_norm_quant_rows_device, x.data_ptr(), _DTYPE[x.dtype], _ld(x),
          residual.data_ptr() if residual is not None else None,
          _DTYPE[residual.dtype] if residual is not None else HCR_F32,
          _ld(residual) if residual is not None else 0, rows, cols, _NORM[norm],
          weight.data_ptr(), bias.data_ptr() if bias is not None else None, eps,
          sum_out.data_ptr() if sum_out is not None else None,
          _ld(sum_out) if sum_out is not None else 0,
          norm_out.data_ptr() if norm_out is not None else None,
          _DTYPE[norm_out.dtype] if norm_out is not None else HCR_F32,
          _ld(norm_out) if norm_out is not None else 0,
          out.q.data_ptr(), _ld(out.q), out.scale.data_ptr())
    return out


def int8_linear(x: Int8Rows, w: Int8Rows, bias: Optional[torch.Tensor] = None,
                dtype: torch.dtype = torch.float16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x . w^T + bias``: x [rows, depth], w [features, depth], bias float32 [features] ->
    [rows, features] in ``dtype`` (or into ``out``).  The integer sums are exact."""
    if not isinstance(x, Int8Rows) or not isinstance(w, Int8Rows):
        raise ValueError("x and w: expected Int8Rows (quantize_rows makes them)")
    rows, depth = x.q.shape
    features = w.q.shape[0]
    dev = x.q.device
    if w.q.shape[1] != depth:
        raise ValueError(f"x has depth {depth}, w {w.q.shape[1]}")
    if w.q.device != dev:
        raise ValueError(f"w: on {w.q.device}, x on {dev}")
    if bias is not None:
        _check(bias, "bias", (torch.float32,), 1, dev)
        if bias.shape[0] != features:
            raise ValueError(f"bias: {bias.shape[0]} elements, expected {features}")
    if out is None:
        if dtype not in _DTYPE:
            raise ValueError(f"dtype {dtype} is not supported here")
        out = torch.empty((rows, features), dtype=dtype, device=dev)
    else:
        _check(out, "out", _DTYPE, 2, dev)
        if tuple(out.shape) != (rows, features):
            raise ValueError(f"out: shape {tuple(out.shape)}, expected {(rows, features)}")
    _call(dev, lib().hcr_int8_linear_device, x.q.data_ptr(), _ld(x.q), x.scale.data_ptr(), rows,
          w.q.data_ptr(), _ld(w.q), w.scale.data_ptr(), features, depth,
          bias.data_ptr() if bias is not None else None, out.data_ptr(), _DTYPE[out.dtype], _ld(out))
    return out


__all__ = ["Int8Rows", "quantize_rows", "norm_quantize", "int8_linear"]
