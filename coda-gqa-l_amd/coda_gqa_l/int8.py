"""Rows in 8 bits: int8 codes with one scale a row, how they are made, and
the product of two sets of them.

  quantize_rows  - rows of a tensor: a weight's output channels, tokens
  rms_norm_int8  - RMSNorm of tokens, the residual's addition before it
  linear_int8    - tokens times weight, exact int32 sums, a scale for each
                   token and each channel
  Int8Rows       - the codes and scales that these hand on

The layers run their projections on them after use_int8_projections()
(Int8Mixin), and take Int8Rows in place of a tensor.  Inference only: no output
carries a gradient.  Errors surface as RuntimeError, like those of the other
operators.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn

from . import _hip
from .rows import _Made, _capturing, _version

__all__ = ["Int8Rows", "quantize_rows", "rms_norm_int8", "linear_int8"]

PAD = 128        # codes of a row are stored up to a multiple of this
MAX_ROW = 32768  # longest row that codes are made of
MAX_STRIDE = 1 << 24  # bytes from row to row that the product's kernels span
FLOAT_ROWS = 4  # token rows that a product's launch quantises itself


def _padded(cols: int) -> int:
    return -(-cols // PAD) * PAD


class Int8Rows:
    """Rows of 8-bit codes: the value at (row, c) is codes[row, c] *
    scales[row].

    codes (..., P) int8 in [-127, 127], P = cols up to a multiple of 128,
    zeros behind cols; scales (...) float32; dtype: the type that the values,
    and what linear_int8 makes of them, have.  A row of scale NaN (one that
    held an infinity or a NaN) makes NaN of all that is computed from it.
    from_codes() lays out codes of the plain shape (..., cols)."""

    __slots__ = ("codes", "scales", "cols", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int, dtype: torch.dtype):
        if codes.dtype is not torch.int8 or scales.dtype is not torch.float32:
            raise RuntimeError(f"Int8Rows: codes must be int8 and scales float32, got {codes.dtype} and {scales.dtype}")
        shape = codes.shape
        if cols <= 0 or not shape or shape[-1] != _padded(cols):
            raise RuntimeError(f"Int8Rows: codes {tuple(shape)} for rows of {cols}: the last size must be "
                               f"{_padded(max(int(cols), 1))} (from_codes() lays out plain codes)")
        if scales.shape != shape[:-1] or scales.device != codes.device:
            raise RuntimeError(f"Int8Rows: scales {tuple(scales.shape)} on {scales.device} for codes {tuple(shape)} on "
                               f"{codes.device}")
        _hip.dtype_code(dtype)
        self.codes, self.scales, self.cols, self.dtype = codes, scales, int(cols), dtype

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
        code = _hip.dtype_code(dtype)
        codes, sm, scales = _flat(self)
        cols = self.cols
        if cols == sm and codes is self.codes:
            out = torch.empty_like(codes, dtype=dtype)
        else:
            out = torch.empty(self.shape, dtype=dtype, device=codes.device)
        _call(_hip.lib().coda_dequantize_rows, codes.get_device(), code, codes.data_ptr(), sm, scales.data_ptr(),
              scales.numel(), cols, out.data_ptr(), cols)
        return out


def _made(codes: torch.Tensor, scales: torch.Tensor, cols: int, dtype: torch.dtype) -> Int8Rows:
    """Int8Rows of codes that this module has laid out."""
    r = Int8Rows.__new__(Int8Rows)
    r.codes, r.scales, r.cols, r.dtype = codes, scales, cols, dtype
    return r


# the current stream's address, without the Stream object around it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(fn, index: int, *args) -> None:
    """A library call on device `index`, whichever is current, and its current
    stream."""
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _hip.check(rc)


def _flat(r: Int8Rows) -> Tuple[torch.Tensor, int, torch.Tensor]:
    """(codes whose rows lie at 16-byte addresses, bytes from one to the next,
    scales without gaps), copied only where they do not lie so."""
    c, s = r.codes, r.scales
    if c.is_contiguous() and s.is_contiguous() and not c.data_ptr() % 16 and c.is_cuda:
        return c, c.shape[-1], s
    if s.numel() >= 1 << 31:
        raise RuntimeError(f"Int8Rows: {s.numel()} rows, a call takes less than 2^31")
    _hip.require_device(c, s)
    s, P = s.contiguous(), c.shape[-1]
    c = c.reshape(-1, P)
    if c.stride(1) == 1 and c.stride(0) % 16 == 0 and c.stride(0) <= MAX_STRIDE and c.data_ptr() % 16 == 0:
        return c, c.stride(0), s
    return c.clone(memory_format=torch.contiguous_format), P, s


def _rows_of(x: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """x (..., D) with unit stride over D, and the elements from one row to
    the next."""
    D = x.shape[-1]
    if x.is_contiguous():
        return x, D
    x = x.reshape(-1, D)
    return (x, x.stride(0)) if x.stride(1) == 1 or D == 1 else (x.contiguous(), D)


def _new_rows(x: torch.Tensor, D: int) -> Tuple[torch.Tensor, torch.Tensor, int]:
    """Uninitialised codes and scales of x's rows, and the codes of a row."""
    lead, P, dev = x.shape[:-1], _padded(D), x.device
    if P == D and x.is_contiguous():
        codes = torch.empty_like(x, dtype=torch.int8)
    else:
        codes = torch.empty((*lead, P), dtype=torch.int8, device=dev)
    return codes, torch.empty(lead, dtype=torch.float32, device=dev), P


def _check_input(x: torch.Tensor, who: str) -> int:
    if not x.is_cuda:
        _hip.require_device(x)
    if x.dim() < 1 or not 0 < x.shape[-1] <= MAX_ROW:
        raise RuntimeError(f"{who}: rows of 1 to {MAX_ROW} elements, got {tuple(x.shape)}")
    return x.shape[-1]


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """x (..., D) in 8 bits, a scale for each row: scale = max|x| / 127, codes
    the nearest to x / scale (ties to even).  For a weight (out, in) the rows
    are its output channels.  D at most 32768."""
    D = _check_input(x, "quantize_rows")
    dt = x.dtype
    code = _hip.dtype_code(dt)
    x2, sm = _rows_of(x)
    codes, scales, P = _new_rows(x, D)
    _call(_hip.lib().coda_quantize_rows, x.get_device(), code, x2.data_ptr(), sm, scales.numel(), D, codes.data_ptr(), P,
          scales.data_ptr())
    return _made(codes, scales, D, dt)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None
                  ) -> Union[Int8Rows, Tuple[Int8Rows, torch.Tensor]]:
    """RMSNorm(x) * weight over the last dimension in 8 bits, a scale for each
    token.  With a residual (x's shape) the norm is of s = x + residual,
    rounded to x's type, and (rows, s) is returned: s is the residual of the
    next sublayer.  x, weight (D,) and residual share their type; D at most
    32768."""
    D, dt, index = _check_input(x, "rms_norm_int8"), x.dtype, x.get_device()
    code = _hip.dtype_code(dt)
    if weight.dtype is not dt or weight.get_device() != index or weight.shape != (D,):
        raise RuntimeError(f"rms_norm_int8: weight is {tuple(weight.shape)} {weight.dtype} on {weight.device}, expected "
                           f"({D},) {dt} on {x.device}")
    if not eps >= 0:
        raise RuntimeError(f"rms_norm_int8: eps={eps} is negative")
    x2, sm = _rows_of(x)
    w = weight if weight.is_contiguous() else weight.contiguous()
    codes, scales, P = _new_rows(x, D)
    fn = _hip.lib().coda_rms_norm_int8
    if residual is None:
        _call(fn, index, code, x2.data_ptr(), sm, None, 0, w.data_ptr(), scales.numel(), D, eps, None, 0, codes.data_ptr(),
              P, scales.data_ptr())
        return _made(codes, scales, D, dt)
    if residual.dtype is not dt or residual.get_device() != index or residual.shape != x.shape:
        raise RuntimeError(f"rms_norm_int8: residual is {tuple(residual.shape)} {residual.dtype} on {residual.device}, x "
                           f"{tuple(x.shape)} {dt} on {x.device}")
    r2, rm = _rows_of(residual)
    out = torch.empty_like(x2) if x2 is x else torch.empty(x.shape, dtype=dt, device=x.device)
    _call(fn, index, code, x2.data_ptr(), sm, r2.data_ptr(), rm, w.data_ptr(), scales.numel(), D, eps, out.data_ptr(), D,
          codes.data_ptr(), P, scales.data_ptr())
    return _made(codes, scales, D, dt), out


def linear_int8(x: Union[Int8Rows, torch.Tensor], weight: Int8Rows, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x (..., K) times weight (N, K), both in 8 bits: the sum of products is
    exact in int32, then times the token's and the channel's scale, plus bias
    (N,), rounded once to x's type.  K at most 130944.  A tensor x is
    quantised by rows first (quantize_rows; K at most 32768), up to 4 rows on
    the product's own way through the weights: the same bits."""
    rows = isinstance(x, Int8Rows)
    if not isinstance(weight, Int8Rows) or not rows and not isinstance(x, torch.Tensor):
        raise TypeError("linear_int8 takes a tensor or Int8Rows, and a weight in Int8Rows (quantize_rows makes them)")
    b, bm, sb = _flat(weight)
    N, P = sb.numel(), weight.codes.shape[-1]
    if rows:
        K, lead = x.cols, x.scales.shape
        a, am, sa = _flat(x)
        M, sp = sa.numel(), sa.data_ptr()
    else:
        K, lead = _check_input(x, "linear_int8"), x.shape[:-1]
        M, sp = x.numel() // K, None
        if M <= FLOAT_ROWS:
            a, am = _rows_of(x)
        else:
            x = quantize_rows(x)
            a, am, sa = x.codes, P, x.scales
            sp = sa.data_ptr()
    if weight.cols != K or weight.scales.dim() != 1 or not N:
        raise RuntimeError(f"linear_int8: weight {tuple(weight.shape)} does not fit x {tuple(x.shape)}")
    dt, index = x.dtype, a.get_device()
    if b.get_device() != index or bias is not None and (bias.get_device() != index or bias.dtype is not dt or
                                                        bias.shape != (N,)):
        raise RuntimeError("linear_int8: weight and bias must be on x's device, bias (N,) of x's type")
    if bias is not None:
        bias = bias.contiguous()
    out = torch.empty((*lead, N), dtype=dt, device=a.device)
    _call(_hip.lib().coda_linear_int8, index, _hip.dtype_code(dt), a.data_ptr(), am, sp, M, K, b.data_ptr(), bm,
          sb.data_ptr(), N, P, None if bias is None else bias.data_ptr(), out.data_ptr(), N)
    return out


class Int8Mixin:
    """The projections of a layer in 8 bits: RowsMixin's attributes, and
    _rope_tables."""

    int8_projections = False

    def use_int8_projections(self, on: bool = True) -> "Int8Mixin":
        """Run q / k / v / lambda / gate (one product, with the RoPE of k and
        the sigmoids) and o_proj on 8-bit rows: weights with a scale for each
        output channel, tokens with a scale each.  Results differ from the
        float projections' by the roundings to 8 bits.  The float parameters
        stay; the codes are made of them at the next call and again whenever
        torch counts a change of one (drop_parameter_copies() after one that
        it does not count; a captured graph keeps the codes of its capture).
        The projections have to be plain nn.Linear without hooks."""
        self.int8_projections = bool(on)
        self.__dict__.pop("_fast", None)
        return self

    def _int8_on(self, x) -> bool:
        """Whether a call on x runs on 8-bit rows."""
        if isinstance(x, Int8Rows):
            if not self.int8_projections:
                raise RuntimeError("the layer takes Int8Rows after use_int8_projections()")
            return True
        return self.int8_projections

    def _int8_names(self) -> tuple:
        return ("q_proj", "k_proj", "v_proj", "lambda_proj") + (("write_proj",) if self._has_gate() else ()) + ("o_proj",)

    def _int8_plain(self, name: str) -> bool:
        """Whether a projection's module does what nn.Linear does, and no more."""
        m = self._modules[name]
        return type(m) is nn.Linear and not (m._forward_hooks or m._forward_pre_hooks or "forward" in m.__dict__)

    def _int8_still_plain(self) -> bool:
        """The part of _int8_linears that a cached step does not see in the
        parameters' identities and versions."""
        return nn.Linear.forward.__module__ == "torch.nn.modules.linear" and \
            not nn.modules.module._has_any_global_hook() and all(map(self._int8_plain, self._int8_names()))

    def _int8_linears(self) -> list:
        H, Hkv, Dh, D = self.num_heads, self.num_kv_heads, self.head_dim, self.embed_dim
        shapes = dict(q_proj=(H * Dh, D), k_proj=(Hkv * Dh, D), v_proj=(Hkv * Dh, D), lambda_proj=(H, D), write_proj=(1, D),
                      o_proj=(D, H * Dh))
        lins = []
        plain = nn.Linear.forward.__module__ == "torch.nn.modules.linear" and not nn.modules.module._has_any_global_hook()
        for n in self._int8_names():
            m = self._modules[n]
            if not plain or not self._int8_plain(n) or type(m.weight) is not nn.Parameter or \
                    tuple(m.weight.shape) != shapes[n]:
                raise RuntimeError(f"8-bit projections need {n} to be a plain nn.Linear {shapes[n]} without hooks")
            lins.append(m)
        return lins

    def _int8_weights(self) -> Tuple[torch.Tensor, ...]:
        """(codes, scales, fp32 biases) of q | k | v | lambda | gate in the
        front end's row order, (codes, scales, bias) of o_proj; kept while the
        parameters are what they were."""
        lins = self._int8_linears()
        ps = [t for m in lins for t in (m.weight, m.bias) if t is not None]
        tag = tuple((id(t), _version(t), t.data_ptr(), t.dtype, t.device) for t in ps) + (self.rope_interleaved,)
        hit = self.__dict__.get("_int8_made")
        if hit is not None and hit[0] == tag:
            hit[2].use()
            return self._handed(hit[1])
        Dh, dev = self.head_dim, lins[0].weight.device
        with torch.no_grad():
            rows = [quantize_rows(m.weight) for m in lins[:-1]]
            codes, scales = [r.codes for r in rows], [r.scales for r in rows]
            bias = [torch.zeros(m.out_features, device=dev) if m.bias is None else m.bias.float() for m in lins[:-1]]
            if not self.rope_interleaved:
                # k rows of a head by RoPE pairs (i, i + Dh/2)
                half = torch.arange(Dh // 2, device=dev)
                perm = (torch.arange(self.num_kv_heads, device=dev)[:, None] * Dh +
                        torch.stack([half, half + Dh // 2], 1).reshape(1, -1)).reshape(-1)
                for part in (codes, scales, bias):
                    part[1] = part[1][perm]
            n = sum(m.out_features for m in lins[:-1])
            out = quantize_rows(lins[-1].weight)
            val = (torch.cat(codes), torch.cat(scales), torch.cat(bias + [torch.zeros(-n % 4, device=dev)]), out.codes,
                   out.scales, lins[-1].bias)
        if not _capturing():
            self.__dict__["_int8_made"] = (tag, val, _Made(*val[:5]))
        return val

    def _launch_int8(self, x, d, weights: tuple, p=None):
        """The front end's product of x (B, L, D), a tensor or Int8Rows, into
        d's outputs (coda_project_int8); what has to live until it has been
        enqueued."""
        if len(x.shape) != 3 or x.shape[2] != self.embed_dim:
            raise RuntimeError(f"tokens {tuple(x.shape)} are not (B, L, {self.embed_dim})")
        w, sw, bias = weights[:3]
        if w.device != x.device:
            raise RuntimeError(f"projection weights on {w.device}, input on {x.device}")
        if not isinstance(x, Int8Rows) and x.shape[0] * x.shape[1] > FLOAT_ROWS:
            x = quantize_rows(x)
        xs, d.x_sm, scales = _flat(x) if isinstance(x, Int8Rows) else (*_rows_of(x), None)
        d.x, d.w, d.bias = xs.data_ptr(), w.data_ptr(), bias.data_ptr()
        _call(_hip.lib().coda_project_int8, xs.get_device(), d, _hip.ptr(scales), sw.data_ptr(), w.stride(0), w.shape[1], p)
        return xs, scales

    def _front_int8(self, x, p0: int):
        """q (B,H,L,Dh) before RoPE, k (B,Hkv,L,Dh) roped, v, the gate (B,L)
        float32 (None without one), lambda (B,H,L) and the RoPE tables of
        positions p0 .., of x (B,L,D), a tensor or Int8Rows."""
        B, L = x.shape[:2]
        H, Hkv, Dh, dt, dev = self.num_heads, self.num_kv_heads, self.head_dim, x.dtype, x.device
        cos, sin = self._rope_tables(p0, L, dev, dt)
        Fq, Fk = H * Dh, Hkv * Dh
        q = torch.empty((B, L, H, Dh), dtype=dt, device=dev)
        k = torch.empty((B, L, Hkv, Dh), dtype=dt, device=dev)
        v = torch.empty((B, L, Hkv, Dh), dtype=dt, device=dev)
        lam = torch.empty((B, L, H), dtype=dt, device=dev)
        g = torch.empty((B, L), dtype=torch.float32, device=dev) if self._has_gate() else None
        d = self._proj_desc(x, B * L, L, cos, sin)
        d.q, d.q_sm, d.k, d.k_sm, d.v, d.v_sm = q.data_ptr(), Fq, k.data_ptr(), Fk, v.data_ptr(), Fk
        d.lam, d.lam_sm, d.g = lam.data_ptr(), H, _hip.ptr(g)
        self._launch_int8(x, d, self._int8_weights())
        return (q.permute(0, 2, 1, 3), k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3), g, lam.permute(0, 2, 1), cos, sin)

    def _out_proj(self, heads: torch.Tensor, weights: Optional[tuple] = None) -> torch.Tensor:
        """o_proj of heads (B, L, H*Dh): the module, or in 8 bits (weights:
        _int8_weights() of this call)."""
        if not self.int8_projections:
            return self.o_proj(heads)
        w, sw, bias = (weights or self._int8_weights())[3:]
        return linear_int8(heads, _made(w, sw, heads.shape[-1], heads.dtype), bias)
