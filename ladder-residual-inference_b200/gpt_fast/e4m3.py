"""Projections in 8 bits (e4m3): rows of activations and weights as pairs (codes, scale), and the operators that make and multiply them.

codes [rows, k] (torch.float8_e4m3fn, k a multiple of 8, rows starting at multiples of 16 bytes: see `empty_rows`) and scale [rows] in
fp32 stand for codes * scale; a weight [outputs, k] has a scale for each output.  A row's scale is its largest magnitude / 448.  A row with an infinity or
NaN gets a NaN scale, so that what is computed from it is NaN.  No counterpart in the reference, whose projections are nn.Linear in
16 bits (gpt_fast/utils.py:142-148, 187-198, 258).
"""
import math
from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from ._C import ACT_GLU, ACTIVATIONS, ONE_SM
from .ops import CudaOps

E4M3 = torch.float8_e4m3fn
SWIGLU = (1.0, math.inf, 0.0)
Rows = Tuple[Tensor, Tensor]
_WIDE, _F32 = (torch.bfloat16, torch.float16), torch.float32


def _said(t):
    return f"{t.dtype} {tuple(t.shape)} with strides {t.stride()}"


def empty_rows(rows: int, cols: int, device=None) -> Rows:
    """Room for rows of codes and their scales."""
    codes = torch.empty(rows, -(-cols // 16) * 16, dtype=E4M3, device=device)
    return (codes if codes.shape[1] == cols else codes[:, :cols]), torch.empty(rows, device=device)


def _looked_at(what, rows, cols=None, count=None):
    """Rows, columns and pitch of a pair (codes, scale), which are to be `count` x `cols` if that is given."""
    codes, scale = rows
    shape, strides = codes.shape, codes.stride()
    if len(shape) == 2:
        n, k = shape
        pitch = strides[0] if n != 1 else -(-k // 16) * 16  # (the pitch of a single row may be any number)
        if (codes.dtype is E4M3 and strides[1] == 1 and pitch % 16 == 0 and pitch >= k > 0 and k % 8 == 0 and (cols is None or k == cols and n == count) and
                scale.dtype is _F32 and scale.numel() == n and scale.is_contiguous()):
            return n, k, pitch
    want = "[rows, a multiple of 8]" if cols is None else f"[{count}, {cols}]"
    raise ValueError(f"{what}: float8_e4m3fn codes {want} whose rows start at multiples of 16 bytes (e4m3.empty_rows) and a contiguous fp32 scale for "
                     f"each, not {_said(codes)} and {_said(scale)}")


def _dense(what, t, dtype, shape):
    if not (t.dtype is dtype and t.shape == shape and t.is_contiguous()):
        raise ValueError(f"{what}: contiguous {dtype} {tuple(shape)}, not {_said(t)}")


def _result(out, dtype, rows, n, device):
    if out is None:
        if dtype not in _WIDE:
            raise TypeError(f"results are bfloat16 or float16, not {dtype}")
        return torch.empty(rows, n, dtype=dtype, device=device)
    if out.dtype not in _WIDE:
        raise TypeError(f"results are bfloat16 or float16, not {out.dtype}")
    if not (out.shape == (rows, n) and out.is_contiguous()):
        raise ValueError(f"out: contiguous [{rows}, {n}], not {_said(out)}")
    return out


def _wide_rows(x):
    """Rows, columns and pitch of x, which are what quantize_rows takes."""
    shape, strides = x.shape, x.stride()
    rows, cols = shape if len(shape) == 2 else (-1, 0)
    x_ld = cols if rows == 1 else strides[0] if strides else 0
    if not (rows >= 0 and x.dtype in _WIDE and cols % 8 == 0 and 0 < cols <= 65536 and strides[1] == 1 and x_ld % 8 == 0 and x_ld >= cols):
        raise ValueError(f"x: bfloat16 or float16 rows of a multiple of 8 elements up to 65536 that start at multiples of 16 bytes, not {_said(x)}")
    return rows, cols, x_ld


def quantize_rows(x: Tensor, out: Optional[Rows] = None, early: bool = False) -> Rows:
    """Rows of x [rows, cols] (bfloat16 or float16; rows may lie apart, as parts of a wider buffer) as codes and scales; cols a multiple of 8
    up to 65536.  early: the next kernel may start before these rows are complete, for which it waits by itself."""
    rows, cols, x_ld = _wide_rows(x)
    if out is None:
        out = empty_rows(rows, cols, x.device)
    _, _, codes_ld = _looked_at("out", out, cols, rows)
    CudaOps.quantize_rows_e4m3(x, out[0], out[1], rows, cols, x_ld, codes_ld, early)
    return out


def add_rmsnorm(residual: Tensor, weight: Tensor, eps: float, add1: Optional[Tensor] = None, add2: Optional[Tensor] = None, residual_scale: float = 1.0,
                residual_out: Optional[Tensor] = None, out: Optional[Rows] = None, early: bool = False) -> Rows:
    """round(round(residual * residual_scale) + add1) + add2 to residual_out (None: not kept; may be residual), each sum rounded to the residual's
    type, and RMSNorm of that times weight as codes and scales.  residual, add1, add2 [rows, dim]; dim a multiple of 8 up to 16384.  early: as in
    quantize_rows."""
    shape, dtype = residual.shape, residual.dtype
    rows, dim = shape if len(shape) == 2 else (-1, 0)
    if not (rows >= 0 and dtype in _WIDE and dim % 8 == 0 and 0 < dim <= 16384 and residual.is_contiguous()):
        raise ValueError(f"residual: contiguous bfloat16 or float16 rows of a multiple of 8 elements up to 16384, not {_said(residual)}")
    if not (weight.dtype is dtype and weight.numel() == dim and weight.is_contiguous()):
        _dense("weight", weight, dtype, (dim,))
    for name, t in (("add1", add1), ("add2", add2), ("residual_out", residual_out)):
        if t is not None and not (t.dtype is dtype and t.shape == shape and t.is_contiguous()):
            _dense(name, t, dtype, shape)
    if out is None:
        out = empty_rows(rows, dim, residual.device)
    _, _, codes_ld = _looked_at("out", out, dim, rows)
    CudaOps.add_rmsnorm_e4m3(residual, add1, add2, weight, eps, residual_out, out[0], out[1], rows, dim, codes_ld, residual_scale, early)
    return out


def linear(x: Rows, w: Rows, bias: Optional[Tensor] = None, activation: Optional[str] = None, addend: Optional[Tensor] = None,
           dtype: torch.dtype = torch.bfloat16, out: Optional[Tensor] = None, one_sm: bool = False) -> Tensor:
    """activation(x w^T + bias) + addend, [rows, outputs], summed in fp32 and rounded once.  activation: None, "silu", "gelu" (by the error
    function) or "gelu_tanh"; bias [outputs] and addend [rows, outputs] in the result's type; the addend may be `out`.  dtype: of the result where `out`
    is None.  A w with `ahead` set may be read before the call in front of this one is complete (E4M3Weight).  one_sm: not on pairs of SMs, for a call beside which another stream runs projections or prompt
    attention (a process can keep off them altogether by option gemm_pair = 0)."""
    rows, k, x_ld = _looked_at("x", x)
    n, depth, w_ld = _looked_at("w", w)
    if k != depth:
        raise ValueError(f"rows of {k} codes times weights of {depth}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation={activation!r}: one of {list(ACTIVATIONS)}")
    if out is None or not (out.dtype in _WIDE and out.shape == (rows, n) and out.is_contiguous()):
        out = _result(out, dtype, rows, n, next(iter(x)).device)
    if bias is not None:
        _dense("bias", bias, out.dtype, (n,))
    if addend is not None:
        _dense("addend", addend, out.dtype, (rows, n))
    CudaOps.linear_e4m3(x, w, out, rows, n, k, x_ld, w_ld, bias, addend, ACTIVATIONS[activation],
                        flags=ONE_SM if one_sm else 0)
    return out


def gateup_glu(x: Rows, w1: Rows, glu: Tuple[float, float, float] = SWIGLU, dtype: torch.dtype = torch.bfloat16, out: Optional[Tensor] = None,
               one_sm: bool = False) -> Tensor:
    """The gated unit of x w1^T, w1 [2 inter, k] = [up | gate]: g * sigmoid(alpha g) * (u + offset) with g = min(gate, limit),
    u = clamp(up, -limit, limit), glu = (alpha, limit, offset); SwiGLU by default.  In fp32, rounded once to [rows, inter].
    one_sm: as in linear."""
    rows, k, x_ld = _looked_at("x", x)
    n, depth, w_ld = _looked_at("w1", w1)
    if k != depth or n % 2 or not n:
        raise ValueError(f"rows of {k} codes times [up | gate] weights [{n}, {depth}]")
    if not glu[1] >= 0:
        raise ValueError(f"glu={glu}: the limit is not below 0")
    out = _result(out, dtype, rows, n // 2, next(iter(x)).device)
    CudaOps.linear_e4m3(x, w1, out, rows, n // 2, k, x_ld, w_ld, activation=ACT_GLU, glu=glu, flags=ONE_SM if one_sm else 0)
    return out


class E4M3Weight:
    """Rows of a weight in 8 bits: (codes, scale) = weight.  Slices are rows of the same memory.  ahead: a projection may start on them while the kernel in front of it
    on the stream still runs; for weights that have been complete since before an operation in front of that which begins when all before it is complete
    (a copy, any kernel of torch), or since the host last waited."""
    __slots__ = ("codes", "scale", "ahead")

    def __init__(self, codes: Tensor, scale: Tensor, ahead: bool = False):
        self.codes, self.scale, self.ahead = codes, scale, ahead

    def __iter__(self):
        yield self.codes
        yield self.scale

    def __getitem__(self, rows: slice) -> "E4M3Weight":
        return E4M3Weight(self.codes[rows], self.scale[rows], self.ahead)

    @property
    def shape(self):
        return self.codes.shape


class E4M3Linear(nn.Module):
    """Stands where a model's nn.Linear was: owns the codes and scales of its weight [outputs, k].  `codes` [outputs, k up to a multiple of 16]."""

    @staticmethod
    def check(lin: nn.Linear):
        """Raises where a projection cannot go to 8 bits."""
        if lin.bias is not None:
            raise ValueError("a projection with a bias")
        _wide_rows(lin.weight)
        if lin.weight.data_ptr() % 16:
            raise ValueError("a weight that does not start at a multiple of 16 bytes")

    def __init__(self, weight: Tensor):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.register_buffer("codes", torch.zeros(self.out_features, -(-self.in_features // 16) * 16, dtype=E4M3, device=weight.device))
        self.register_buffer("scale", torch.empty(self.out_features, device=weight.device))
        quantize_rows(weight.detach(), out=(self.codes[:, :self.in_features], self.scale))

    @property
    def weight(self) -> E4M3Weight:
        b = self._buffers
        codes, scale = b["codes"], b["scale"]
        if codes.dtype is not E4M3 or scale.dtype is not _F32:
            raise TypeError("a module that was cast after its weights went to 8 bits holds codes without their meaning")
        return E4M3Weight(codes if codes.shape[1] == self.in_features else codes[:, :self.in_features], scale)

    def forward(self, x: Tensor) -> Tensor:
        rows = x.reshape(-1, self.in_features)
        return linear(quantize_rows(rows, early=True), self.weight, dtype=x.dtype).view(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}"
