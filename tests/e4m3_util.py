"""Projections in 8 bits for tests: rows of codes with everything around them poisoned, and the operators' definitions in 64 bits."""
import math

import torch

E4M3 = torch.float8_e4m3fn
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half a step of the smallest numbers
U = 2.0 ** -24  # a rounding to fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rows_of(codes, scale, pad=0, device="cuda"):
    """(codes, scale) with rows `pad` * 16 bytes further apart than they need be; what lies between the rows are NaN codes."""
    n, k = codes.shape
    room = torch.full((n, (-(-k // 16) + pad) * 16), 0x7F, dtype=torch.uint8, device=device)
    room[:, :k] = codes.to(device).view(torch.uint8)
    return room.view(E4M3)[:, :k], scale.to(device)


def random_rows(n, k, seed, pad=0, size=1.0, device="cuda"):
    """Codes of all sizes and both signs, scales over a factor of e^2."""
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn(n, k, generator=g) * 60).clamp(-448, 448).to(E4M3)
    return rows_of(codes, torch.exp(0.5 * torch.randn(n, generator=g)) * size / 60, pad, device)


def values(rows):
    return rows[0].double() * rows[1].double().unsqueeze(1)


def quantised(x):
    """Codes and scales of rows by the definition in fp32, which every step of is a single rounding."""
    x = x.float()
    bad = ~torch.isfinite(x).all(-1)
    top = x.abs().amax(-1).clamp(min=2.0 ** -100)
    largest = torch.full_like(top, 448.0)  # (a tensor: torch divides by and into numbers by way of a reciprocal, which rounds twice)
    codes = (x * (largest / top).unsqueeze(-1)).clamp(-448, 448).to(E4M3)
    codes.view(torch.uint8)[bad] = 0
    return codes, torch.where(bad, math.nan, top / largest)


def step(y):
    """The distance of the e4m3 numbers around |y| <= 448."""
    _, e = torch.frexp(y.double().abs())
    return torch.exp2((e.double() - 4).clamp(min=-9))


def activation64(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.erfc(-z / math.sqrt(2)) / 2
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def sums64(x, w):
    """x w^T in 64 bits, and how far a sum in fp32 may be off: within an instruction 32 products and the sum so far are cut to a common exponent, each
    by at most 2^-23 of the sum of magnitudes (33 terms); there are k / 32 instructions, joined in at most 16 parts; then two factors."""
    xv, wv = values(x), values(w)
    z, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    return z, (2 * (x[0].shape[1] / 32 + 33 + 16) + 3) * U * size


def linear64(x, w, bias=None, activation=None, addend=None, dtype=torch.bfloat16):
    """The result in 64 bits and the error that it may have.  Slopes of the activations are below 1.13; their own evaluation in fp32 is good to 16 U of
    |z| (an exponential, a division, erff or tanhf of 2 ulp, three products)."""
    z, off = sums64(x, w)
    if bias is not None:
        z = z + bias.double()
        off = off + U * z.abs()
    y = activation64(activation, z)
    if activation is not None:
        off = 1.13 * off + 16 * U * z.abs()
    if addend is not None:
        y = y + addend.double()
        off = off + U * y.abs()
    return y, off * (1 + 2 ** -8) + half_step(dtype) * y.abs() * (1 + 2 ** -8) + TINY[dtype]


def glu64(x, w1, glu, dtype=torch.bfloat16):
    alpha, limit, offset = glu
    z, off = sums64(x, w1)
    (up, gate), (uo, go) = z.chunk(2, -1), off.chunk(2, -1)
    up, gate = up.clamp(-limit, limit), gate.clamp(max=limit)
    act = gate * torch.sigmoid(alpha * gate)
    y = act * (up + offset)
    # slope of g * sigmoid(alpha g) below 1.13; 16 U of |g| for its evaluation, a rounding of u + offset and one of the product
    err = (1.13 * go + 16 * U * gate.abs()) * ((up + offset).abs() + uo) + act.abs() * (uo + U * (up + offset).abs()) + 2 * U * y.abs()
    return y, err * (1 + 2 ** -8) + half_step(dtype) * y.abs() * (1 + 2 ** -8) + TINY[dtype]


def check(got, want, off):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN elsewhere"
    far = ((got - want).abs() - off)[~torch.isnan(want)]
    if far.numel():
        assert far.max() <= 0, f"{far.max().item()} over the bound, {(far > 0).float().mean().item():.2e} of the results"
