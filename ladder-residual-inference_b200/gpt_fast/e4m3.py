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

from ._C import ACT_GLU, ACTIVATIONS
from .ops import CudaOps

E4M3 = torch.float8_e4m3fn
SWIGLU = (1.0, math.inf, 0.0)
Rows = Tuple[Tensor, Tensor]
_WIDE = (torch.bfloat16, torch.float16)


def _said(t):
    return f"{t.dtype} {tuple(t.shape)} with strides {t.stride()}"


def empty_rows(rows: int, cols: int, device=None) -> Rows:
    """Room for rows of codes and their scales."""
    codes = torch.empty(rows, -(-cols // 16) * 16, dtype=E4M3, device=device)
    return (codes if codes.shape[1] == cols else codes[:, :cols]), torch.empty(rows, device=device)


def _check_rows(what, rows, shape=None):
    """The shape of a pair (codes, scale)."""
    codes, scale = rows
    got = codes.shape
    if not (codes.dtype is E4M3 and len(got) == 2 and (shape is None or got == shape) and got[1] % 8 == 0 and got[1] > 0 and
            (got[0] <= 1 or codes.stride(0) % 16 == 0 and codes.stride(0) >= got[1]) and codes.stride(1) == 1):
        raise ValueError(f"{what}: float8_e4m3fn codes {'[rows, a multiple of 8]' if shape is None else tuple(shape)} whose rows start at multiples of 16 bytes "
                         f"(e4m3.empty_rows), not {_said(codes)}")
    if not (scale.dtype is torch.float32 and scale.shape == got[:1] and scale.is_contiguous()):
        raise ValueError(f"{what}: {got[0]} contiguous fp32 scales, not {_said(scale)}")
    return got


def _check_dense(what, t, dtype, shape):
    if not (t.dtype is dtype and t.shape == shape and t.is_contiguous()):
        raise ValueError(f"{what}: contiguous {dtype} {tuple(shape)}, not {_said(t)}")


def quantize_rows(x: Tensor, out: Optional[Rows] = None, early: bool = False) -> Rows:
    """Rows of x [rows, cols] (bfloat16 or float16; rows may lie apart, as parts of a wider buffer) as codes and scales; cols a multiple of 8
    up to 65536.  early: the projection that follows may start on its weights before these rows are complete; not for rows that are themselves its weights."""
    shape = x.shape
    if not (x.dtype in _WIDE and len(shape) == 2 and shape[1] % 8 == 0 and 0 < shape[1] <= 65536 and x.stride(1) == 1 and
            (shape[0] <= 1 or x.stride(0) % 8 == 0 and x.stride(0) >= shape[1])):
        raise ValueError(f"x: bfloat16 or float16 rows of a multiple of 8 elements up to 65536 that start at multiples of 16 bytes, not {_said(x)}")
    if out is None:
        out = empty_rows(*shape, x.device)
    else:
        _check_rows("out", out, shape)
    CudaOps.quantize_rows_e4m3(x, *out, shape, early)
    return out


def add_rmsnorm(residual: Tensor, weight: Tensor, eps: float, add1: Optional[Tensor] = None, add2: Optional[Tensor] = None, residual_scale: float = 1.0,
                residual_out: Optional[Tensor] = None, out: Optional[Rows] = None, early: bool = False) -> Rows:
    """round(round(residual * residual_scale) + add1) + add2 to residual_out (None: not kept; may be residual), each sum rounded to the residual's
    type, and RMSNorm of that times weight as codes and scales.  residual, add1, add2 [rows, dim]; dim a multiple of 8 up to 16384.  early: as in quantize_rows."""
    shape, dtype = residual.shape, residual.dtype
    if not (dtype in _WIDE and len(shape) == 2 and shape[1] % 8 == 0 and 0 < shape[1] <= 16384 and residual.is_contiguous()):
        raise ValueError(f"residual: contiguous bfloat16 or float16 rows of a multiple of 8 elements up to 16384, not {_said(residual)}")
    _check_dense("weight", weight, dtype, shape[1:])
    if add1 is not None:
        _check_dense("add1", add1, dtype, shape)
    if add2 is not None:
        _check_dense("add2", add2, dtype, shape)
    if residual_out is not None:
        _check_dense("residual_out", residual_out, dtype, shape)
    if out is None:
        out = empty_rows(*shape, residual.device)
    else:
        _check_rows("out", out, shape)
    CudaOps.add_rmsnorm_e4m3(residual, add1, add2, weight, eps, residual_out, *out, shape[0], residual_scale, early)
    return out


def linear(x: Rows, w: Rows, bias: Optional[Tensor] = None, activation: Optional[str] = None, addend: Optional[Tensor] = None,
           dtype: torch.dtype = torch.bfloat16, out: Optional[Tensor] = None) -> Tensor:
    """activation(x w^T + bias) + addend, [rows, outputs], summed in fp32 and rounded once.  activation: None, "silu", "gelu" (by the error
    function) or "gelu_tanh"; bias [outputs] and addend [rows, outputs] in the result's type; the addend may be `out`.  dtype: of the result where `out` is None."""
    rows, k = _check_rows("x", x)
    n, depth = _check_rows("w", w)
    if k != depth:
        raise ValueError(f"rows of {k} codes times weights of {depth}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation={activation!r}: one of {list(ACTIVATIONS)}")
    if out is None:
        if dtype not in _WIDE:
            raise TypeError(f"results are bfloat16 or float16, not {dtype}")
        out = torch.empty(rows, n, dtype=dtype, device=x[0].device)
    else:
        dtype = out.dtype
        if dtype not in _WIDE:
            raise TypeError(f"results are bfloat16 or float16, not {dtype}")
        _check_dense("out", out, dtype, (rows, n))
    if bias is not None:
        _check_dense("bias", bias, dtype, (n,))
    if addend is not None:
        _check_dense("addend", addend, dtype, (rows, n))
    CudaOps.linear_e4m3(x, w, out, rows, bias, addend, ACTIVATIONS[activation])
    return out


def gateup_glu(x: Rows, w1: Rows, glu: Tuple[float, float, float] = SWIGLU, dtype: torch.dtype = torch.bfloat16, out: Optional[Tensor] = None) -> Tensor:
    """The gated unit of x w1^T, w1 [2 inter, k] = [up | gate]: g * sigmoid(alpha g) * (u + offset) with g = min(gate, limit),
    u = clamp(up, -limit, limit), glu = (alpha, limit, offset); SwiGLU by default.  In fp32, rounded once to [rows, inter]."""
    rows, k = _check_rows("x", x)
    n, depth = _check_rows("w1", w1)
    if k != depth or n % 2 or not n:
        raise ValueError(f"rows of {k} codes times [up | gate] weights [{n}, {depth}]")
    if not glu[1] >= 0:
        raise ValueError(f"glu={glu}: the limit is not below 0")
    if out is None:
        if dtype not in _WIDE:
            raise TypeError(f"results are bfloat16 or float16, not {dtype}")
        out = torch.empty(rows, n // 2, dtype=dtype, device=x[0].device)
    else:
        if out.dtype not in _WIDE:
            raise TypeError(f"results are bfloat16 or float16, not {out.dtype}")
        _check_dense("out", out, out.dtype, (rows, n // 2))
    CudaOps.linear_e4m3(x, w1, out, rows, activation=ACT_GLU, glu=glu)
    return out
