"""Activations behind projections in 8 bits, at arguments that are known to the last bit: one code of 1 in a row, and a weight's scale as the argument."""
import math

import pytest
import torch

from e4m3_util import E4M3, TINY, U, activation64, half_step
from gpt_fast import _C, e4m3

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]
KERNELS = [("few", 1), ("few", 40), ("pair", 1000)]


def _arguments(dtype):
    """Every part of the activations: their tails down to where the type ends, and far beyond."""
    z = torch.cat([torch.linspace(-14, 9, 5000), torch.linspace(-1, 1, 1001), torch.linspace(-105, -14, 700)])
    return z if dtype is torch.float16 else torch.cat([z, torch.tensor([200.0, -200.0, 1e4, -1e4, 3e12, -3e12, 1e30, -1e30])])


def _projection(rows, z, k):
    """Rows and weights whose sums are the numbers z: sign * 1 * |z| + 0 + .."""
    x = torch.zeros(rows, k)
    x[:, 5] = 1.0
    w = torch.zeros(len(z), k)
    w[:, 5] = torch.where(z < 0, -1.0, 1.0)
    rows8, w8 = e4m3.empty_rows(rows, k, "cuda"), e4m3.empty_rows(len(z), k, "cuda")
    for (codes, scale), v, s in ((rows8, x, torch.ones(rows)), (w8, w, z.abs())):
        codes.copy_(v.to(E4M3))
        scale.copy_(s)
    return rows8, w8


def _slack(name, z, y):
    """The evaluation in fp32 beside the rounding of the result (derived beside the formulas in csrc/e4m3.cuh)."""
    roundings = {"silu": 8 + 1.5 * z.abs(), "gelu": 16 + 1.25 * z * z, "gelu_tanh": 8 + 8 * (2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)).abs()}[name]
    return (roundings * U * y.abs()).nan_to_num(0.0, 0.0, 0.0) + z.abs() * 2.0 ** -126


def _check(got, want, slack, dtype):
    off = slack * (1 + 2 ** -8) + half_step(dtype) * want.abs() * (1 + 2 ** -8) + TINY[dtype]
    far = (got.double() - want).abs() > off
    assert not far.any(), (want[far][:5], got.double()[far][:5], far.sum())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kernel,rows", KERNELS)
@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_activations_to_the_rounding_of_the_result(name, kernel, rows, dtype):
    z = _arguments(dtype)
    k = 520 if kernel == "pair" else 40
    assert (_C.lib.lri_linear_e4m3_plan(0, rows, len(z), k, 0) > 0) == (kernel == "pair")
    x, w = _projection(rows, z, k)
    y = e4m3.linear(x, w, activation=name, dtype=dtype)
    z = z.cuda().double()
    want = activation64(name, z)
    assert (y == y[0]).all()
    _check(y[0], want, _slack(name, z, want), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kernel,rows", KERNELS)
@pytest.mark.parametrize("alpha,up", [(1.0, 1.5), (1.702, -0.75)])
def test_gated_unit_to_the_rounding_of_the_result(kernel, rows, dtype, alpha, up):
    z = _arguments(dtype)
    k = 520 if kernel == "pair" else 40
    assert (_C.lib.lri_linear_e4m3_plan(0, rows, len(z), k, _C.ACT_GLU) > 0) == (kernel == "pair")
    x, w = _projection(rows, torch.cat([torch.full_like(z, up), z]), k)
    y = e4m3.gateup_glu(x, w, (alpha, math.inf, 0.0), dtype=dtype)
    z = z.cuda().double()
    want = z * torch.sigmoid(alpha * z) * up
    assert (y == y[0]).all()
    _check(y[0], want, ((10 + 3 * alpha * z.abs()) * U * want.abs()).nan_to_num(0.0) + z.abs() * abs(up) * 2.0 ** -126, dtype)
