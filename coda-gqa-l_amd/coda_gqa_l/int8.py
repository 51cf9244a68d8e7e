"""Rows in 8 bits: int8 codes with one scale a row, how they are made, and
the product of two sets of them.

  quantize_rows  - rows of a tensor: a weight's output channels, tokens
  rms_norm_int8  - RMSNorm of tokens, the residual's addition before it
  linear_int8    - tokens times weight, exact int32 sums, a scale for each
                   token and each channel
  Int8Rows       - the codes and scales that these hand on

The layers run their projections on them after use_int8_projections()
(Int8Mixin).  Inference only: no output carries a gradient.  Errors surface
as RuntimeError, like those of the other operators.
"""

from __future__ import annotations

import contextlib
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _hip

__all__ = ["Int8Rows", "quantize_rows", "rms_norm_int8", "linear_int8"]

PAD = 128        # codes of a row are stored up to a multiple of this
MAX_ROW = 32768  # longest row that codes are made of


def _padded(cols: int) -> int:
    return -(-cols // PAD) * PAD


def _on(t: torch.Tensor):
    """Work on t's device, whichever is current."""
    if t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


@dataclass(frozen=True)
class Int8Rows:
    """Rows of 8-bit codes: the value at (row, c) is codes[row, c] *
    scales[row].

    codes (..., P) int8 in [-127, 127], P = cols up to a multiple of 128,
    zeros behind cols; scales (...) float32; dtype: the type that the values,
    and what linear_int8 makes of them, have.  A row of scale NaN (one that
    held an infinity or a NaN) makes NaN of all that is computed from it.
    from_codes() lays out codes of the plain shape (..., cols)."""

    codes: torch.Tensor
    scales: torch.Tensor
    cols: int
    dtype: torch.dtype

    def __post_init__(self):
        c, s = self.codes, self.scales
        if c.dtype != torch.int8 or s.dtype != torch.float32:
            raise RuntimeError(f"Int8Rows: codes must be int8 and scales float32, got {c.dtype} and {s.dtype}")
        if self.cols <= 0 or c.dim() < 1 or c.shape[-1] != _padded(self.cols):
            raise RuntimeError(f"Int8Rows: codes {tuple(c.shape)} for rows of {self.cols}: the last size must be "
                               f"{_padded(max(int(self.cols), 1))} (from_codes() lays out plain codes)")
        if s.shape != c.shape[:-1] or s.device != c.device:
            raise RuntimeError(f"Int8Rows: scales {tuple(s.shape)} on {s.device} for codes {tuple(c.shape)} on {c.device}")
        _hip.dtype_code(self.dtype)

    @staticmethod
    def from_codes(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> "Int8Rows":
        """Rows of plain codes (..., cols), zeros added behind them."""
        cols = codes.shape[-1]
        if codes.dtype == torch.int8 and cols % PAD:
            codes = torch.nn.functional.pad(codes, (0, _padded(cols) - cols))
        return Int8Rows(codes, scales, cols, dtype)

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.cols))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def is_cuda(self) -> bool:
        return self.codes.is_cuda

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values, in `dtype` (None: the rows' own)."""
        dtype = self.dtype if dtype is None else dtype
        codes, scales = _flat(self)
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        with _on(codes):
            _hip.check(_hip.lib().coda_dequantize_rows(
                _hip.dtype_code(dtype), codes.data_ptr(), codes.stride(0), scales.data_ptr(), codes.shape[0], self.cols,
                out.data_ptr(), self.cols, _hip.stream_of(codes)))
        return out


def _flat(r: Int8Rows) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes (rows, P) whose rows lie at 16-byte addresses, scales (rows,)
    without gaps), copied only where they do not lie so."""
    _hip.require_device(r.codes, r.scales)
    c = r.codes.reshape(-1, r.codes.shape[-1])
    if c.stride(1) != 1 or c.stride(0) % 16 or c.data_ptr() % 16:
        c = c.clone(memory_format=torch.contiguous_format)
    return c, r.scales.reshape(-1).contiguous()


def _rows_of(x: torch.Tensor) -> torch.Tensor:
    """x (..., D) as (rows, D) with unit stride over D."""
    x2 = x.reshape(-1, x.shape[-1])
    return x2 if x2.stride(1) == 1 or x2.shape[1] == 1 else x2.contiguous()


def _new_rows(x: torch.Tensor, D: int) -> Tuple[torch.Tensor, torch.Tensor]:
    lead = x.shape[:-1]
    return (torch.empty((*lead, _padded(D)), dtype=torch.int8, device=x.device),
            torch.empty(lead, dtype=torch.float32, device=x.device))


def _check_input(x: torch.Tensor, who: str) -> int:
    _hip.require_device(x)
    if x.dim() < 1 or not 0 < x.shape[-1] <= MAX_ROW:
        raise RuntimeError(f"{who}: rows of 1 to {MAX_ROW} elements, got {tuple(x.shape)}")
    return x.shape[-1]


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """x (..., D) in 8 bits, a scale for each row: scale = max|x| / 127, codes
    the nearest to x / scale (ties to even).  For a weight (out, in) the rows
    are its output channels.  D at most 32768."""
    D = _check_input(x, "quantize_rows")
    x2 = _rows_of(x.detach())
    codes, scales = _new_rows(x, D)
    with _on(x):
        _hip.check(_hip.lib().coda_quantize_rows(
            _hip.dtype_code(x.dtype), x2.data_ptr(), x2.stride(0), x2.shape[0], D, codes.data_ptr(), codes.shape[-1],
            scales.data_ptr(), _hip.stream_of(x)))
    return Int8Rows(codes, scales, D, x.dtype)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None
                  ) -> Union[Int8Rows, Tuple[Int8Rows, torch.Tensor]]:
    """RMSNorm(x) * weight over the last dimension in 8 bits, a scale for each
    token.  With a residual (x's shape) the norm is of s = x + residual,
    rounded to x's type, and (rows, s) is returned: s is the residual of the
    next sublayer.  x, weight (D,) and residual share their type; D at most
    32768."""
    D = _check_input(x, "rms_norm_int8")
    _hip.require_device(weight, residual)
    if tuple(weight.shape) != (D,):
        raise RuntimeError(f"rms_norm_int8: weight {tuple(weight.shape)}, expected ({D},)")
    if residual is not None and residual.shape != x.shape:
        raise RuntimeError(f"rms_norm_int8: residual {tuple(residual.shape)} is not x's shape {tuple(x.shape)}")
    for name, t in (("weight", weight), ("residual", residual)):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise RuntimeError(f"rms_norm_int8: {name} is {t.dtype} on {t.device}, x {x.dtype} on {x.device}")
    if not eps >= 0:
        raise RuntimeError(f"rms_norm_int8: eps={eps} is negative")
    x2, w = _rows_of(x.detach()), weight.detach().contiguous()
    codes, scales = _new_rows(x, D)
    r2 = out = None
    if residual is not None:
        r2 = _rows_of(residual.detach())
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with _on(x):
        _hip.check(_hip.lib().coda_rms_norm_int8(
            _hip.dtype_code(x.dtype), x2.data_ptr(), x2.stride(0), _hip.ptr(r2), 0 if r2 is None else r2.stride(0),
            w.data_ptr(), x2.shape[0], D, float(eps), _hip.ptr(out), D, codes.data_ptr(), codes.shape[-1],
            scales.data_ptr(), _hip.stream_of(x)))
    rows = Int8Rows(codes, scales, D, x.dtype)
    return rows if residual is None else (rows, out)


def linear_int8(x: Int8Rows, weight: Int8Rows, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x (..., K) times weight (N, K), both in 8 bits: the sum of products is
    exact in int32, then times the token's and the channel's scale, plus bias
    (N,), rounded once to x's type.  K at most 130944."""
    if not isinstance(x, Int8Rows) or not isinstance(weight, Int8Rows):
        raise TypeError("linear_int8 takes Int8Rows (quantize_rows, rms_norm_int8 make them)")
    if weight.codes.dim() != 2 or weight.cols != x.cols or weight.codes.shape[0] == 0:
        raise RuntimeError(f"linear_int8: weight {tuple(weight.shape)} does not fit x {tuple(x.shape)}")
    N = weight.codes.shape[0]
    _hip.require_device(x.codes, weight.codes, bias)
    if weight.device != x.device or bias is not None and (bias.device != x.device or bias.dtype != x.dtype or
                                                          tuple(bias.shape) != (N,)):
        raise RuntimeError("linear_int8: weight and bias must be on x's device, bias (N,) of x's type")
    a, sa = _flat(x)
    b, sb = _flat(weight)
    bias = None if bias is None else bias.detach().contiguous()
    out = torch.empty((*x.codes.shape[:-1], N), dtype=x.dtype, device=x.device)
    with _on(a):
        _hip.check(_hip.lib().coda_linear_int8(
            _hip.dtype_code(x.dtype), a.data_ptr(), a.stride(0), sa.data_ptr(), a.shape[0], b.data_ptr(), b.stride(0),
            sb.data_ptr(), N, b.shape[1], _hip.ptr(bias), out.data_ptr(), N, _hip.stream_of(a)))
    return out
